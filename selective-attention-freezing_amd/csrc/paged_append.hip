// New tokens into a paged key / value cache (gfx950): the per-head RMSNorm
// and rotary embedding of q and k at the tokens' positions, and the write of
// k and v into their pages, one pass over the projection output.
//
//   y = w x / sqrt(mean(x^2) + eps)                         (with weights)
//   y[d] cos[s][d] - y[d + rd/2] sin[s][d]   d < rd/2        (with cos / sin,
//   y[d] cos[s][d] + y[d - rd/2] sin[s][d]   d < rd           s the position)
// in fp32, rounded once.  A lane owns one 16-byte piece of a row (8 elements,
// 4 in float32), the lanes of a row are an aligned power-of-two group, and the
// rows of one token (its q, k and v heads) follow each other, so a wave reads
// and writes whole rows.  The bound is HBM for prompts and the launch for
// single tokens.
#include "saf_kernels.h"

namespace saf {

template <typename T> struct Piece {  // 16-bit: 8 elements
  static constexpr int N = 8;
  __device__ static inline void unpack(uint4 r, float (&f)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      f[2 * m] = Elem<T>::lo(w[m]);
      f[2 * m + 1] = Elem<T>::hi(w[m]);
    }
  }
  __device__ static inline uint4 pack(const float (&f)[8]) {
    return make_uint4(Elem<T>::pack2(f[0], f[1]), Elem<T>::pack2(f[2], f[3]), Elem<T>::pack2(f[4], f[5]),
                      Elem<T>::pack2(f[6], f[7]));
  }
};
template <> struct Piece<float> {
  static constexpr int N = 4;
  __device__ static inline void unpack(uint4 r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  __device__ static inline uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// N consecutive elements of a cos / sin row or a norm weight as fp32.
template <int N> __device__ inline void load_f32(const void* p, int dtype, int64_t off, float (&f)[N]) {
#pragma unroll
  for (int m = 0; m < N; ++m) f[m] = load_as_f32(p, off + m, dtype);
}

template <typename T, int LANES>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p) {
  using P = Piece<T>;
  constexpr int N = P::N;
  const int b = blockIdx.y;
  const int NH = p.Uq + p.Uk + p.Hv;
  const int64_t gid = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row = gid / LANES;
  const int ci = (int)(gid & (LANES - 1));
  const int t = (int)(row / NH), hh = (int)(row - (int64_t)t * NH);
  // whole lane groups leave together: the shuffles below stay inside a group
  if (t >= p.T) return;
  const bool is_q = hh < p.Uq, is_v = hh >= p.Uq + p.Uk;
  const int h = is_q ? hh : (is_v ? hh - p.Uq - p.Uk : hh - p.Uq);
  const int d0 = N * ci;
  const bool active = d0 < p.hd;
  const bool kept = p.counts == nullptr || t < p.counts[b];
  T* qo = nullptr;
  if (is_q) qo = reinterpret_cast<T*>(p.q_out) + b * p.qo_sb + h * p.qo_sh + t * p.qo_st;
  if (!kept) {
    if (is_q && active) *reinterpret_cast<uint4*>(qo + d0) = make_uint4(0, 0, 0, 0);
    return;
  }
  const int64_t pos64 = (int64_t)p.positions[b] + t;
  bool ok = pos64 >= 0 && pos64 < p.capacity && (p.cos == nullptr || pos64 < p.cs_rows);
  const int pos = ok ? (int)pos64 : 0;
  int page = 0;
  if (ok) {
    page = p.table[b * p.t_sb + (pos >> p.page_shift)];
    ok = page >= 0 && page < p.n_pages;
  }
  if (!ok) {
    if (is_q && active) {
      float f[N];
#pragma unroll
      for (int m = 0; m < N; ++m) f[m] = __builtin_nanf("");
      *reinterpret_cast<uint4*>(qo + d0) = P::pack(f);
    }
    return;
  }
  const int slot = pos & ((1 << p.page_shift) - 1);
  const T* src;
  T* dst;
  if (is_q) {
    src = reinterpret_cast<const T*>(p.q) + b * p.q_sb + h * p.q_sh + t * p.q_st;
    dst = qo;
  } else if (is_v) {
    src = reinterpret_cast<const T*>(p.v) + b * p.v_sb + h * p.v_sh + t * p.v_st;
    dst = reinterpret_cast<T*>(p.vc) + page * p.vc_sp + h * p.vc_sh + slot * p.vc_st;
  } else {
    src = reinterpret_cast<const T*>(p.k) + b * p.k_sb + h * p.k_sh + t * p.k_st;
    dst = reinterpret_cast<T*>(p.kc) + page * p.kc_sp + h * p.kc_sh + slot * p.kc_st;
  }
  uint4 raw = make_uint4(0, 0, 0, 0);
  if (active) raw = *reinterpret_cast<const uint4*>(src + d0);
  if (is_v) {
    if (active) *reinterpret_cast<uint4*>(dst + d0) = raw;
    return;
  }
  float x[N];
  P::unpack(raw, x);
  const int half = p.rd / 2;
  const bool rot = p.cos != nullptr && d0 < p.rd;
  const int dp = d0 < half ? d0 + half : d0 - half;  // the pair's piece (rot)
  float y[N];
  if (rot && active) P::unpack(*reinterpret_cast<const uint4*>(src + dp), y);
  if (p.q_w != nullptr) {
    float ss = 0.f;
#pragma unroll
    for (int m = 0; m < N; ++m) ss = fmaf(x[m], x[m], ss);
#pragma unroll
    for (int m = 1; m < LANES; m <<= 1) ss += __shfl_xor(ss, m, LANES);
    const float r = rsqrtf(ss / (float)p.hd + p.eps);
    if (active) {
      const void* w = is_q ? p.q_w : p.k_w;
      float f[N];
      load_f32<N>(w, p.w_dtype, d0, f);
#pragma unroll
      for (int m = 0; m < N; ++m) x[m] = x[m] * r * f[m];
      if (rot) {
        load_f32<N>(w, p.w_dtype, dp, f);
#pragma unroll
        for (int m = 0; m < N; ++m) y[m] = y[m] * r * f[m];
      }
    }
  }
  if (!active) return;
  if (rot) {
    float cs[N], sn[N];
    load_f32<N>(p.cos, p.cs_dtype, pos * p.cs_st + d0, cs);
    load_f32<N>(p.sin, p.cs_dtype, pos * p.sn_st + d0, sn);
    const float sign = d0 < half ? -1.f : 1.f;
#pragma unroll
    for (int m = 0; m < N; ++m) x[m] = fmaf(x[m], cs[m], sign * y[m] * sn[m]);
  }
  *reinterpret_cast<uint4*>(dst + d0) = P::pack(x);
}

template <typename T, int LANES>
static hipError_t launch_append_l(const PagedAppendParams& p, hipStream_t s) {
  const int64_t rows = (int64_t)p.T * (p.Uq + p.Uk + p.Hv);
  const dim3 grid((unsigned)((rows * LANES + 255) / 256), (unsigned)p.B);
  hipLaunchKernelGGL((paged_append_kernel<T, LANES>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_append_t(const PagedAppendParams& p, hipStream_t s) {
  int lanes = 1;
  while (lanes * Piece<T>::N < p.hd) lanes <<= 1;
  switch (lanes) {
    case 4: return launch_append_l<T, 4>(p, s);
    case 8: return launch_append_l<T, 8>(p, s);
    case 16: return launch_append_l<T, 16>(p, s);
    case 32: return launch_append_l<T, 32>(p, s);
    case 64: return launch_append_l<T, 64>(p, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_paged_append(const PagedAppendParams& p, int dtype, hipStream_t s) {
  if (dtype == kBF16) return launch_append_t<__bf16>(p, s);
  if (dtype == kF16) return launch_append_t<_Float16>(p, s);
  if (dtype == kF32) return launch_append_t<float>(p, s);
  return hipErrorInvalidValue;
}

}  // namespace saf
