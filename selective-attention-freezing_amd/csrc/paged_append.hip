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
// and writes whole rows.  The bound is HBM for prompts (8 ragged prompts of up
// to 4096 tokens, 9 + 9 + 12 heads of 64: 39 us, 4.6 TB/s read and written) and
// the launch for single tokens (64 tokens, 14 + 2 + 2 heads: 3.9 us replayed as
// a graph, 7.7 us a call).
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

// N consecutive elements of a cos / sin row or a norm weight as fp32, from
// 16-byte aligned rows (vec) or one by one.
template <int N> __device__ inline void load_f32(const void* p, int dtype, int vec, int64_t off, float (&f)[N]) {
  if (!vec) {
#pragma unroll
    for (int m = 0; m < N; ++m) f[m] = load_as_f32(p, off + m, dtype);
  } else if (dtype == kF32) {
#pragma unroll
    for (int m = 0; m < N; m += 4) {
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + off + m);
      f[m] = x.x; f[m + 1] = x.y; f[m + 2] = x.z; f[m + 3] = x.w;
    }
  } else {
    uint32_t w[N / 2];
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + off;
    if constexpr (N == 8) {
      const uint4 x = *reinterpret_cast<const uint4*>(q);
      w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    } else {
      const uint2 x = *reinterpret_cast<const uint2*>(q);
      w[0] = x.x; w[1] = x.y;
    }
#pragma unroll
    for (int m = 0; m < N / 2; ++m) {
      f[2 * m] = dtype == kBF16 ? Elem<__bf16>::lo(w[m]) : Elem<_Float16>::lo(w[m]);
      f[2 * m + 1] = dtype == kBF16 ? Elem<__bf16>::hi(w[m]) : Elem<_Float16>::hi(w[m]);
    }
  }
}

// A thread owns one piece of HPT heads of one kind (q, k or v) of one token:
// the page lookup, the cos / sin piece and the weights serve all of them, and
// their loads are in flight together.  Consecutive lane groups are
// consecutive tokens, so a wave's cache rows lie together.
template <typename T, int LANES, int HPT>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p) {
  using P = Piece<T>;
  constexpr int N = P::N;
  const int b = blockIdx.y;
  const int gq = (p.Uq + HPT - 1) / HPT, gk = (p.Uk + HPT - 1) / HPT, gv = (p.Hv + HPT - 1) / HPT;
  const unsigned row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int ci = threadIdx.x & (LANES - 1);
  const unsigned grp = row / (unsigned)p.T;
  const int t = (int)(row - grp * (unsigned)p.T);
  // whole lane groups leave together: the shuffles below stay inside a group
  if (grp >= (unsigned)(gq + gk + gv)) return;
  const bool is_q = (int)grp < gq, is_v = (int)grp >= gq + gk;
  const int h0 = HPT * (is_q ? (int)grp : (is_v ? (int)grp - gq - gk : (int)grp - gq));
  const int nh = min(HPT, (is_q ? p.Uq : (is_v ? p.Hv : p.Uk)) - h0);
  const int d0 = N * ci;
  const bool active = d0 < p.hd;
  const bool kept = p.counts == nullptr || t < p.counts[b];
  if (!kept && !is_q) return;
  const T* src;
  T* dst;
  int64_t s_sh, d_sh;
  bool ok = kept;
  int pos = 0;
  if (kept) {
    const int64_t pos64 = (int64_t)p.positions[b] + t;
    ok = pos64 >= 0 && pos64 < p.capacity && (p.cos == nullptr || pos64 < p.cs_rows);
    pos = ok ? (int)pos64 : 0;
  }
  int page = 0;
  if (ok) {
    page = p.table[b * p.t_sb + (pos >> p.page_shift)];
    ok = page >= 0 && page < p.n_pages;
  }
  const int slot = pos & ((1 << p.page_shift) - 1);
  if (is_q) {
    src = reinterpret_cast<const T*>(p.q) + b * p.q_sb + h0 * p.q_sh + t * p.q_st;
    s_sh = p.q_sh;
    dst = reinterpret_cast<T*>(p.q_out) + b * p.qo_sb + h0 * p.qo_sh + t * p.qo_st;
    d_sh = p.qo_sh;
  } else if (is_v) {
    src = reinterpret_cast<const T*>(p.v) + b * p.v_sb + h0 * p.v_sh + t * p.v_st;
    s_sh = p.v_sh;
    dst = reinterpret_cast<T*>(p.vc) + page * p.vc_sp + h0 * p.vc_sh + slot * p.vc_st;
    d_sh = p.vc_sh;
  } else {
    src = reinterpret_cast<const T*>(p.k) + b * p.k_sb + h0 * p.k_sh + t * p.k_st;
    s_sh = p.k_sh;
    dst = reinterpret_cast<T*>(p.kc) + page * p.kc_sp + h0 * p.kc_sh + slot * p.kc_st;
    d_sh = p.kc_sh;
  }
  if (!ok) {
    if (is_q && active) {  // padding rows are zero, rows without a slot NaN
      float f[N];
#pragma unroll
      for (int m = 0; m < N; ++m) f[m] = kept ? __builtin_nanf("") : 0.f;
      for (int j = 0; j < nh; ++j) *reinterpret_cast<uint4*>(dst + j * d_sh + d0) = P::pack(f);
    }
    return;
  }
  uint4 raw[HPT], pair[HPT];
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    raw[j] = pair[j] = make_uint4(0, 0, 0, 0);
    if (active && j < nh) raw[j] = *reinterpret_cast<const uint4*>(src + j * s_sh + d0);
  }
  if (is_v) {
#pragma unroll
    for (int j = 0; j < HPT; ++j)
      if (active && j < nh) *reinterpret_cast<uint4*>(dst + j * d_sh + d0) = raw[j];
    return;
  }
  const int half = p.rd / 2;
  const bool rot = active && p.cos != nullptr && d0 < p.rd;
  const int dp = d0 < half ? d0 + half : d0 - half;  // the pair's piece
  float cs[N], sn[N], w[N] = {}, wp[N] = {};
  if (rot) {
#pragma unroll
    for (int j = 0; j < HPT; ++j)
      if (j < nh) pair[j] = *reinterpret_cast<const uint4*>(src + j * s_sh + dp);
    load_f32<N>(p.cos, p.cs_dtype, p.cs_vec, pos * p.cs_st + d0, cs);
    load_f32<N>(p.sin, p.cs_dtype, p.cs_vec, pos * p.sn_st + d0, sn);
    if (d0 < half) {
#pragma unroll
      for (int m = 0; m < N; ++m) sn[m] = -sn[m];
    }
  }
  if (p.q_w != nullptr && active) {
    const void* wt = is_q ? p.q_w : p.k_w;
    load_f32<N>(wt, p.w_dtype, p.w_vec, d0, w);
    if (rot) load_f32<N>(wt, p.w_dtype, p.w_vec, dp, wp);
  }
#pragma unroll
  for (int j = 0; j < HPT; ++j) {
    if (j >= nh) break;  // uniform over the lane group
    float x[N], y[N];
    P::unpack(raw[j], x);
    P::unpack(pair[j], y);
    if (p.q_w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int m = 0; m < N; ++m) ss = fmaf(x[m], x[m], ss);
#pragma unroll
      for (int m = 1; m < LANES; m <<= 1) ss += __shfl_xor(ss, m, LANES);
      const float r = rsqrtf(ss / (float)p.hd + p.eps);
#pragma unroll
      for (int m = 0; m < N; ++m) {
        x[m] = x[m] * r * w[m];
        y[m] = y[m] * r * wp[m];
      }
    }
    if (rot) {
#pragma unroll
      for (int m = 0; m < N; ++m) x[m] = fmaf(x[m], cs[m], y[m] * sn[m]);
    }
    if (active) *reinterpret_cast<uint4*>(dst + j * d_sh + d0) = P::pack(x);
  }
}

template <typename T, int LANES, int HPT>
static hipError_t launch_append_h(const PagedAppendParams& p, hipStream_t s) {
  const int64_t groups = (p.Uq + HPT - 1) / HPT + (p.Uk + HPT - 1) / HPT + (p.Hv + HPT - 1) / HPT;
  const dim3 grid((unsigned)((p.T * groups * LANES + 255) / 256), (unsigned)p.B);
  hipLaunchKernelGGL((paged_append_kernel<T, LANES, HPT>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

// Four heads per thread where that leaves every SIMD work (2^20 pieces are
// 4096 waves of four heads); one where the call is a matter of latency.
template <typename T, int LANES>
static hipError_t launch_append_l(const PagedAppendParams& p, hipStream_t s) {
  const int64_t pieces = (int64_t)p.B * p.T * (p.Uq + p.Uk + p.Hv) * LANES;
  return pieces >= (1 << 20) ? launch_append_h<T, LANES, 4>(p, s) : launch_append_h<T, LANES, 1>(p, s);
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
