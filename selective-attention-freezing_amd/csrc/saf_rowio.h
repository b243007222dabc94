// Eight consecutive elements of a row as float32, whatever their type and the
// row's alignment, and indices of (row, chunk) units (gfx950).
//
// Global memory instructions take addresses of any alignment, so rows of odd
// widths are read and written with the same 16-byte pieces as aligned ones; only
// a row's last chunk, when it is not whole, goes element by element.
#pragma once
#include "saf_device.h"

namespace saf {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));

template <typename T> struct Row8 {
  static __device__ inline void load(const T* p, float (&f)[8]) {
    const u32x4_any r = *reinterpret_cast<const u32x4_any*>(p);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f[2 * m] = Elem<T>::lo(r[m]);
      f[2 * m + 1] = Elem<T>::hi(r[m]);
    }
  }
  static __device__ inline void store(T* p, const float (&f)[8]) {
    u32x4_any r;
#pragma unroll
    for (int m = 0; m < 4; ++m) r[m] = Elem<T>::pack2(f[2 * m], f[2 * m + 1]);
    *reinterpret_cast<u32x4_any*>(p) = r;
  }
};
template <> struct Row8<float> {
  static __device__ inline void load(const float* p, float (&f)[8]) {
    const f32x4_any a = *reinterpret_cast<const f32x4_any*>(p), b = *reinterpret_cast<const f32x4_any*>(p + 4);
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f[m] = a[m];
      f[m + 4] = b[m];
    }
  }
  static __device__ inline void store(float* p, const float (&f)[8]) {
    f32x4_any a, b;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      a[m] = f[m];
      b[m] = f[m + 4];
    }
    *reinterpret_cast<f32x4_any*>(p) = a;
    *reinterpret_cast<f32x4_any*>(p + 4) = b;
  }
};

// Elements c..c+7 of a row of C; those past it are `past` / not stored.
template <typename T>
__device__ inline void load_row8(const T* row, int c, int C, float (&f)[8], float past = 0.f) {
  if (c + 8 <= C) {
    Row8<T>::load(row + c, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = c + e < C ? (float)row[c + e] : past;
  }
}
template <typename T>
__device__ inline void store_row8(T* row, int c, int C, const float (&f)[8]) {
  if (c + 8 <= C) {
    Row8<T>::store(row + c, f);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < C) row[c + e] = static_cast<T>(f[e]);
  }
}
// The same of a vector of run-time type.
__device__ inline void load_vec8(const void* v, int dtype, int c, int C, float (&f)[8]) {
  if (dtype == 0) load_row8(reinterpret_cast<const float*>(v), c, C, f);
  else if (dtype == 2) load_row8(reinterpret_cast<const __bf16*>(v), c, C, f);
  else load_row8(reinterpret_cast<const _Float16*>(v), c, C, f);
}
__device__ inline void store_elem(void* v, int dtype, int64_t i, float x) {
  if (dtype == 0) reinterpret_cast<float*>(v)[i] = x;
  else if (dtype == 2) reinterpret_cast<__bf16*>(v)[i] = (__bf16)x;
  else reinterpret_cast<_Float16*>(v)[i] = (_Float16)x;
}

// n / d for n < 2^31 and a divisor known on the host, by a multiplication:
// with 2^(s-1) < d <= 2^s and m = floor(2^32 (2^s - d) / d) + 1 the quotient is
// (high word of n m, plus n) >> s.
struct FastDiv {
  uint32_t d, m, s;
  static FastDiv of(uint32_t d) {
    uint32_t s = 0;
    while (s < 32 && (uint64_t(1) << s) < d) ++s;
    return {d, (uint32_t)((((uint64_t(1) << s) - d) << 32) / d + 1), s};
  }
  __device__ inline uint32_t div(uint32_t n) const { return (__umulhi(n, m) + n) >> s; }
};

}  // namespace saf
