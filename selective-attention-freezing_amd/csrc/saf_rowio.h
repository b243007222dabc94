// Eight consecutive elements of a row as float32, whatever their type and the
// row's alignment, and indices of (row, chunk) units (gfx950).
//
// Global memory instructions take addresses of any alignment, so rows of odd
// widths are read and written with the same 16-byte pieces as aligned ones; only
// a row's last chunk, when it is not whole, goes in pieces of four, two and one
// elements, each loaded to its place: what puts them together after the load would
// wait for memory before the next row's load is on its way.
#pragma once
#include "saf_device.h"

namespace saf {

typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));
typedef uint32_t u32x2_e2 __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32_e2 __attribute__((aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x2_any __attribute__((ext_vector_type(2), aligned(4)));

// Eight elements as they lie in memory, and as float32.  Kernels load all the
// pieces that they need before they unpack the first, so that they wait for memory
// once and not once a piece.
template <typename T> struct Row8 {
  u32x4_any raw;
  __device__ inline void unpack(float (&f)[8]) const {
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f[2 * m] = Elem<T>::lo(raw[m]);
      f[2 * m + 1] = Elem<T>::hi(raw[m]);
    }
  }
  static __device__ inline Row8 pack(const float (&f)[8]) {
    Row8 r;
#pragma unroll
    for (int m = 0; m < 4; ++m) r.raw[m] = Elem<T>::pack2(f[2 * m], f[2 * m + 1]);
    return r;
  }
  static __device__ inline Row8 load(const T* p) { return {*reinterpret_cast<const u32x4_any*>(p)}; }
  static __device__ inline Row8 load_once(const T* p) {
    return {__builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p))};
  }
  __device__ inline void store(T* p) const { *reinterpret_cast<u32x4_any*>(p) = raw; }
  __device__ inline void stream(T* p) const { __builtin_nontemporal_store(raw, reinterpret_cast<u32x4_any*>(p)); }
  // its first n < 8 elements, the rest zero
  static __device__ inline Row8 load_part(const T* p, int n) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    Row8 r{};
    if (n & 4) {
      const u32x2_e2 four = *reinterpret_cast<const u32x2_e2*>(h);
      r.raw[0] = four[0];
      r.raw[1] = four[1];
      if (n & 2) r.raw[2] = *reinterpret_cast<const u32_e2*>(h + 4);
      if (n == 7) r.raw[3] = h[6];
      if (n == 5) r.raw[2] = h[4];
    } else {
      if (n & 2) r.raw[0] = *reinterpret_cast<const u32_e2*>(h);
      if (n == 3) r.raw[1] = h[2];
      if (n == 1) r.raw[0] = h[0];
    }
    return r;
  }
  __device__ inline void store_part(T* p, int n) const {
    uint16_t* h = reinterpret_cast<uint16_t*>(p);
    if (n & 4) *reinterpret_cast<u32x2_e2*>(h) = u32x2_e2{raw[0], raw[1]};
    if (n & 2) *reinterpret_cast<u32_e2*>(h + (n & 4)) = n & 4 ? raw[2] : raw[0];
    if (n & 1) h[n & 6] = (uint16_t)(n & 4 ? (n & 2 ? raw[3] : raw[2]) : (n & 2 ? raw[1] : raw[0]));
  }
};
template <> struct Row8<float> {
  f32x4_any raw[2];
  __device__ inline void unpack(float (&f)[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = raw[e / 4][e % 4];
  }
  static __device__ inline Row8 pack(const float (&f)[8]) {
    Row8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r.raw[e / 4][e % 4] = f[e];
    return r;
  }
  static __device__ inline Row8 load(const float* p) {
    return {{*reinterpret_cast<const f32x4_any*>(p), *reinterpret_cast<const f32x4_any*>(p + 4)}};
  }
  static __device__ inline Row8 load_once(const float* p) {
    return {{__builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(p)),
             __builtin_nontemporal_load(reinterpret_cast<const f32x4_any*>(p + 4))}};
  }
  __device__ inline void store(float* p) const {
    *reinterpret_cast<f32x4_any*>(p) = raw[0];
    *reinterpret_cast<f32x4_any*>(p + 4) = raw[1];
  }
  __device__ inline void stream(float* p) const {
    __builtin_nontemporal_store(raw[0], reinterpret_cast<f32x4_any*>(p));
    __builtin_nontemporal_store(raw[1], reinterpret_cast<f32x4_any*>(p + 4));
  }
  static __device__ inline Row8 load_part(const float* p, int n) {
    Row8 r{};
    if (n & 4) {
      r.raw[0] = *reinterpret_cast<const f32x4_any*>(p);
      if (n & 2) {
        const f32x2_any two = *reinterpret_cast<const f32x2_any*>(p + 4);
        r.raw[1][0] = two[0];
        r.raw[1][1] = two[1];
      }
      if (n == 7) r.raw[1][2] = p[6];
      if (n == 5) r.raw[1][0] = p[4];
    } else {
      if (n & 2) {
        const f32x2_any two = *reinterpret_cast<const f32x2_any*>(p);
        r.raw[0][0] = two[0];
        r.raw[0][1] = two[1];
      }
      if (n == 3) r.raw[0][2] = p[2];
      if (n == 1) r.raw[0][0] = p[0];
    }
    return r;
  }
  __device__ inline void store_part(float* p, int n) const {
    if (n & 4) *reinterpret_cast<f32x4_any*>(p) = raw[0];
    if (n & 2) *reinterpret_cast<f32x2_any*>(p + (n & 4)) = n & 4 ? f32x2_any{raw[1][0], raw[1][1]} : f32x2_any{raw[0][0], raw[0][1]};
    if (n & 1) p[n & 6] = n & 4 ? (n & 2 ? raw[1][2] : raw[1][0]) : (n & 2 ? raw[0][2] : raw[0][0]);
  }
};

// Four elements.
template <typename T> struct Row4 {
  u32x2_e2 raw;
  __device__ inline void unpack(float (&f)[4]) const {
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      f[2 * m] = Elem<T>::lo(raw[m]);
      f[2 * m + 1] = Elem<T>::hi(raw[m]);
    }
  }
  static __device__ inline Row4 load(const T* p) { return {*reinterpret_cast<const u32x2_e2*>(p)}; }
  // the first n < 4
  static __device__ inline Row4 load_part(const T* p, int n) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
    Row4 r{};
    if (n & 2) r.raw[0] = *reinterpret_cast<const u32_e2*>(h);
    if (n == 3) r.raw[1] = h[2];
    if (n == 1) r.raw[0] = h[0];
    return r;
  }
  static __device__ inline void store(T* p, const float (&f)[4]) {
    *reinterpret_cast<u32x2_e2*>(p) = u32x2_e2{Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3])};
  }
};
template <> struct Row4<float> {
  f32x4_any raw;
  __device__ inline void unpack(float (&f)[4]) const {
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = raw[e];
  }
  static __device__ inline Row4 load(const float* p) { return {*reinterpret_cast<const f32x4_any*>(p)}; }
  static __device__ inline Row4 load_part(const float* p, int n) {
    Row4 r{};
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) r.raw[e] = p[e];
    return r;
  }
  static __device__ inline void store(float* p, const float (&f)[4]) {
    *reinterpret_cast<f32x4_any*>(p) = f32x4_any{f[0], f[1], f[2], f[3]};
  }
};

// Elements c..c+7 of a row of C; those past it are zero / not stored.  WHOLE: C is a
// multiple of 8 (kernels whose code is large are built for both: what a launch
// reads of it is read anew, and part chunks are most of it).
template <bool WHOLE = false, typename T>
__device__ inline Row8<T> load_raw8(const T* row, int c, int C) {
  Row8<T> r{};
  if (WHOLE ? c < C : c + 8 <= C) r = Row8<T>::load(row + c);
  else if (!WHOLE && c < C) r = Row8<T>::load_part(row + c, C - c);
  return r;
}
// The same, and kEdge for rows of at least 8 elements: a last chunk that is not whole is
// the row's last 8, which edge_unpack moves to their places once they are there; no
// branch then stands between one row's load and the next's.
// ONCE: nothing reads the row again soon, and it takes no other's place in the caches.
enum class RowEnd { kEdge, kAny };
template <RowEnd END, bool ONCE = false, typename T>
__device__ inline Row8<T> edge_raw8(const T* row, int c, int C) {
  Row8<T> r{};
  if constexpr (END == RowEnd::kAny) {
    if (c + 8 <= C) r = ONCE ? Row8<T>::load_once(row + c) : Row8<T>::load(row + c);
    else if (c < C) r = Row8<T>::load_part(row + c, C - c);
  } else {
    const T* p = row + (c + 8 <= C ? c : C - 8);
    if (c < C) r = ONCE ? Row8<T>::load_once(p) : Row8<T>::load(p);
  }
  return r;
}
template <RowEnd END, typename T>
__device__ inline void edge_unpack(const Row8<T>& r, int c, int C, float (&f)[8]) {
  r.unpack(f);
  if (END != RowEnd::kEdge || c + 8 <= C || c >= C) return;
  const int by = c + 8 - C;
#pragma unroll
  for (int s = 4; s > 0; s >>= 1)
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = by & s ? (e + s < 8 ? f[e + s < 8 ? e + s : 0] : 0.f) : f[e];
}
template <bool WHOLE = false, typename T>
__device__ inline void load_row8(const T* row, int c, int C, float (&f)[8]) {
  load_raw8<WHOLE>(row, c, C).unpack(f);
}
template <bool WHOLE = false, typename T>
__device__ inline void store_row8(T* row, int c, int C, const float (&f)[8]) {
  const Row8<T> r = Row8<T>::pack(f);
  if (WHOLE ? c < C : c + 8 <= C) r.store(row + c);
  else if (!WHOLE && c < C) r.store_part(row + c, C - c);
}
// store_row8 of a result that this launch does not read again: past the L2, which
// keeps it for what is read.
template <bool WHOLE = false, typename T>
__device__ inline void stream_row8(T* row, int c, int C, const float (&f)[8]) {
  const Row8<T> r = Row8<T>::pack(f);
  if (WHOLE ? c < C : c + 8 <= C) r.stream(row + c);
  else if (!WHOLE && c < C) r.store_part(row + c, C - c);
}

// N chunks of 8 elements of a vector of C, of a run-time type, at c, c + step, ...
template <typename T, RowEnd END, int N>
__device__ inline void load_vec_of(const void* v, int c, int step, int C, float (&f)[N][8]) {
  Row8<T> r[N];
#pragma unroll
  for (int k = 0; k < N; ++k) r[k] = edge_raw8<END>(reinterpret_cast<const T*>(v), c + step * k, C);
#pragma unroll
  for (int k = 0; k < N; ++k) edge_unpack<END>(r[k], c + step * k, C, f[k]);
}
template <RowEnd END, int N>
__device__ inline void load_vec(const void* v, int dtype, int c, int step, int C, float (&f)[N][8]) {
  if (dtype == 0) load_vec_of<float, END>(v, c, step, C, f);
  else if (dtype == 2) load_vec_of<__bf16, END>(v, c, step, C, f);
  else load_vec_of<_Float16, END>(v, c, step, C, f);
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
