// Residual addition and LayerNorm of a training step, forward and backward
// (gfx950).
//
//   r = x + delta (rounded to x's type)      m = mean(r), rstd = 1 / sqrt(var(r) + eps)
//   xh = (r - m) rstd                        y = xh w + b
//   g = dy w
//   dx = dr + rstd (g - mean(g) - xh mean(g xh))
//   dw = sum over rows of dy xh, db = sum over rows of dy
//
// One pass over the rows each way, everything in float32 between the load and
// the one rounding of each result; the variance is the centred sum of squares
// (the row stays in registers, so the second sum costs no second read).  Both
// kernels move bytes and nothing else bounds them.
//
// A row belongs to TPR threads (from eight lanes for 64 channels to sixteen waves for
// 16384), each with NCH chunks of 8 channels, chunk k at channel 8 (TPR k + thread):
// every load and store of the group is one run.  2^25 elements take 40 us forward and
// 52 backward in bf16, 93 and 96 in float32 (6.7 and 5.2, 5.8 and 5.6 TB/s; a copy
// reaches 5.2).  At odd widths a row's last chunk is read as its last 8 channels and
// moved into place in registers (333 channels of bf16: element by element 79 and 98 us,
// so 57 and 68; 2047 of float32 backward 134 and 111).
//
// What nothing reads again goes past the caches: dy and dr (8192 x 2048, float32
// beside bf16, both directions: 105 us through them, 99 past them), r and y (44 and 41
// forward; a training step is the same either way).  delta so read costs rows that fit
// the caches more than it gives (bf16 forward: 41 us, 48), and so do dy and dr whose
// pieces cross lines, which are then fetched twice (rows of 2047: 76 and 91).
//
// Backward: a workgroup walks rows a grid apart and keeps its share of dw and db
// of its threads' channels in registers; at the end it adds its waves in LDS and
// writes one (2, C) float32 partial, and a second kernel adds the partials in
// a fixed order, so the weight gradients are the same in every run.
#include "saf_kernels.h"
#include "saf_rowio.h"

namespace saf {

namespace {

template <int TPR> constexpr int kGroups = TPR > 64 ? 1 : 256 / TPR;  // rows of a workgroup at a time
template <int TPR> constexpr int kThreads = TPR > 64 ? TPR : 256;
// Rows of less than 8 channels are among the narrowest form's only (fwd_width, bwd_width).
template <int TPR, int NCH> constexpr RowEnd kEnd = TPR * NCH == 8 ? RowEnd::kAny : RowEnd::kEdge;

// Sum over the TPR threads of a row, in a fixed order.  `slot` is LDS of the
// reduction's own (one per sum of a row) where several waves share a row.
template <int TPR>
__device__ inline float row_sum(float v, float* slot) {
  if constexpr (TPR <= 32) {
    v = dpp_add<0xb1, 0xf>(v);
    v = dpp_add<0x4e, 0xf>(v);
    v = dpp_add<0x141, 0xf>(v);                   // eight lanes
    if constexpr (TPR > 8) v = dpp_add<0x140, 0xf>(v);
    if constexpr (TPR > 16) v += __shfl_xor(v, 16, 64);
    return v;
  } else {
    v = dpp_wave_sum(v);
    if constexpr (TPR > 64) {
      if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (int i = 0; i < TPR / 64; ++i) v += slot[i];
    }
    return v;
  }
}

template <typename TX, typename TB, int TPR, int NCH>
__global__ __launch_bounds__(kThreads<TPR>) void layernorm_fwd_kernel(const LnTrainParams p) {
  constexpr RowEnd END = kEnd<TPR, NCH>;
  __shared__ float slots[2][TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * kGroups<TPR> + threadIdx.x / TPR;
  // a whole half wave, wave or workgroup leaves together, and sums stay inside it
  if (row >= p.rows) return;
  const int C = p.C;
  const TX* xr = reinterpret_cast<const TX*>(p.x) + row * p.x_rs;
  Row8<TX> x[NCH];
  float v[NCH][8];
#pragma unroll
  for (int k = 0; k < NCH; ++k) x[k] = edge_raw8<END>(xr, 8 * (TPR * k + t), C);
  if (p.delta) {
    const TB* dr = reinterpret_cast<const TB*>(p.delta) + row * p.d_rs;
    TX* rr = reinterpret_cast<TX*>(p.r) + row * C;
    Row8<TB> a[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) a[k] = edge_raw8<END>(dr, 8 * (TPR * k + t), C);
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      float d[8];
      edge_unpack<END>(x[k], 8 * (TPR * k + t), C, v[k]);
      edge_unpack<END>(a[k], 8 * (TPR * k + t), C, d);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[k][e] += d[e];
      stream_row8(rr, 8 * (TPR * k + t), C, v[k]);
      Row8<TX>::pack(v[k]).unpack(v[k]);  // the norm is that of the rounded sum
    }
  } else {
#pragma unroll
    for (int k = 0; k < NCH; ++k) edge_unpack<END>(x[k], 8 * (TPR * k + t), C, v[k]);
  }
  // behind the row, which then needs no registers for its pieces any more, and ahead of
  // the sums that hide them
  float w[NCH][8], b[NCH][8] = {};
  load_vec<END>(p.w, p.wb_dtype, 8 * t, 8 * TPR, C, w);
  if (p.b) load_vec<END>(p.b, p.wb_dtype, 8 * t, 8 * TPR, C, b);
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) s += v[k][e];
  const float mean = row_sum<TPR>(s, slots[0]) / (float)C;
  float q = 0.f;
#pragma unroll
  for (int k = 0; k < NCH; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float d = v[k][e] - mean;
      q = 8 * (TPR * k + t) + e < C ? fmaf(d, d, q) : q;
    }
  const float rstd = 1.f / sqrtf(row_sum<TPR>(q, slots[1]) / (float)C + p.eps);
  if (p.stats && t == 0) {
    p.stats[2 * row] = mean;
    p.stats[2 * row + 1] = rstd;
  }
  TB* yr = reinterpret_cast<TB*>(p.y) + row * C;
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[k][e] = fmaf((v[k][e] - mean) * rstd, w[k][e], b[k][e]);
    stream_row8(yr, 8 * (TPR * k + t), C, w[k]);
  }
}

template <typename TX, typename TB, int TPR, int NCH, bool WHOLE>  // WHOLE: C is a multiple of 8
__global__ __launch_bounds__(kThreads<TPR>) void layernorm_bwd_kernel(const LnTrainBwdParams p) {
  // rows of whole chunks go through the checks of both kinds of chunk all the same: they
  // space a wave's requests out (8192 x 4096 float32: 98 us, 109 with one check; bf16
  // the same either way)
  constexpr RowEnd END = WHOLE ? RowEnd::kAny : kEnd<TPR, NCH>;
  __shared__ float slots[2][TPR > 64 ? TPR / 64 : 1];
  // dw and db of the four waves of a workgroup whose rows are a wave's or less
  constexpr int kCols = 8 * TPR * NCH;
  __shared__ float2 part[TPR > 64 ? 1 : 4][TPR > 64 ? 1 : kCols];
  const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
  const int C = p.C;
  float w[NCH][8], aw[NCH][8] = {}, ab[NCH][8] = {};
  load_vec<END>(p.w, p.w_dtype, 8 * t, 8 * TPR, C, w);
  for (int64_t row = (int64_t)blockIdx.x * kGroups<TPR> + group; row < p.rows;
       row += (int64_t)gridDim.x * kGroups<TPR>) {
    const TX* rr = reinterpret_cast<const TX*>(p.r) + row * p.r_rs;
    const TB* gr = reinterpret_cast<const TB*>(p.dy) + row * p.dy_rs;
    const float mean = p.stats[2 * row], rstd = p.stats[2 * row + 1];
    constexpr bool kTogether = TPR <= 256;  // sixteen waves have no registers for dr as well
    Row8<TX> r[NCH], add[NCH];
    Row8<TB> dy[NCH];
#pragma unroll
    for (int k = 0; k < NCH; ++k) r[k] = edge_raw8<END>(rr, 8 * (TPR * k + t), C);
    if (p.once) {
#pragma unroll
      for (int k = 0; k < NCH; ++k) dy[k] = edge_raw8<END, true>(gr, 8 * (TPR * k + t), C);
    } else {
#pragma unroll
      for (int k = 0; k < NCH; ++k) dy[k] = edge_raw8<END>(gr, 8 * (TPR * k + t), C);
    }
    const TX* er = reinterpret_cast<const TX*>(p.dr) + row * p.dr_rs;
    if (kTogether && p.dr) {
      if (p.once) {
#pragma unroll
        for (int k = 0; k < NCH; ++k) add[k] = edge_raw8<END, true>(er, 8 * (TPR * k + t), C);
      } else {
#pragma unroll
        for (int k = 0; k < NCH; ++k) add[k] = edge_raw8<END>(er, 8 * (TPR * k + t), C);
      }
    }
    float xh[NCH][8], g[NCH][8], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      edge_unpack<END>(r[k], 8 * (TPR * k + t), C, xh[k]);
      edge_unpack<END>(dy[k], 8 * (TPR * k + t), C, g[k]);
    }
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xh[k][e] = (xh[k][e] - mean) * rstd;
        aw[k][e] = fmaf(g[k][e], xh[k][e], aw[k][e]);
        ab[k][e] += g[k][e];
        g[k][e] *= w[k][e];
        s1 += g[k][e];
        s2 = fmaf(g[k][e], xh[k][e], s2);
      }
    // a wave writes a slot again only behind the other sum's barrier, which
    // every wave reaches after it has read this one
    const float c1 = row_sum<TPR>(s1, slots[0]) / (float)C;
    const float c2 = row_sum<TPR>(s2, slots[1]) / (float)C;
    TX* dxr = reinterpret_cast<TX*>(p.dx) + row * C;
#pragma unroll
    for (int k = 0; k < NCH; ++k) {
      const int c = 8 * (TPR * k + t);
      if (c >= C) continue;
      float d[8] = {};
      if (p.dr) {
        if constexpr (!kTogether) add[k] = edge_raw8<END>(er, c, C);
        edge_unpack<END>(add[k], c, C, d);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = fmaf(rstd, g[k][e] - c1 - xh[k][e] * c2, d[e]);
      if (p.dx) store_row8(dxr, c, C, d);
      if (p.ddelta) store_row8(reinterpret_cast<TB*>(p.ddelta) + row * C, c, C, d);
    }
  }
  if (!p.dw && !p.db) return;
  // a workgroup by itself has the sums; the others' parts are added by the next launch
  float* out = p.part + (int64_t)blockIdx.x * 2 * C;
  const bool alone = p.part == nullptr;
  if constexpr (TPR <= 64) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int k = 0; k < NCH; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int o = TPR; o < 32; o <<= 1) {  // the wave's rows
          aw[k][e] += __shfl_xor(aw[k][e], o, 64);
          ab[k][e] += __shfl_xor(ab[k][e], o, 64);
        }
        if constexpr (TPR < 64) {
          aw[k][e] = half_swap_sum(aw[k][e]);
          ab[k][e] = half_swap_sum(ab[k][e]);
        }
        if ((threadIdx.x & 63) < TPR) part[wave][(8 * k + e) * TPR + t] = make_float2(aw[k][e], ab[k][e]);
      }
    __syncthreads();
    for (int i = threadIdx.x; i < kCols; i += 256) {
      const int c = 8 * (i / (8 * TPR) * TPR + i % TPR) + i / TPR % 8;
      if (c >= C) continue;
      const float2 p0 = part[0][i], p1 = part[1][i], p2 = part[2][i], p3 = part[3][i];
      const float sw = (p0.x + p1.x) + (p2.x + p3.x), sb = (p0.y + p1.y) + (p2.y + p3.y);
      if (!alone) {
        out[c] = sw;
        out[C + c] = sb;
      } else {
        if (p.dw) store_elem(p.dw, p.w_dtype, c, sw);
        if (p.db) store_elem(p.db, p.w_dtype, c, sb);
      }
    }
    return;
  }
#pragma unroll
  for (int k = 0; k < NCH; ++k) {
    const int c = 8 * (TPR * k + t);
    if (!alone) {
      store_row8(out, c, C, aw[k]);
      store_row8(out + C, c, C, ab[k]);
      continue;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < C) {
        if (p.dw) store_elem(p.dw, p.w_dtype, c + e, aw[k][e]);
        if (p.db) store_elem(p.db, p.w_dtype, c + e, ab[k][e]);
      }
  }
}

// dw (blockIdx.y 0) and db (1): partials added by 32 lanes a channel, each its
// own residue class in order, then the lanes in order.
__global__ __launch_bounds__(1024) void layernorm_dw_kernel(const LnTrainBwdParams p, int n_part) {
  __shared__ float sums[32][33];
  void* out = blockIdx.y == 0 ? p.dw : p.db;
  if (out == nullptr) return;
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5, c = blockIdx.x * 32 + col, C = p.C;
  float a = 0.f;
  if (c < C) {
    const float* src = p.part + blockIdx.y * C + c;
#pragma unroll 4
    for (int i = lane; i < n_part; i += 32) a += src[(int64_t)i * 2 * C];
  }
  sums[lane][col] = a;
  __syncthreads();
  if (lane != 0 || c >= C) return;
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 32; ++i) s += sums[i][col];
  store_elem(out, p.w_dtype, c, s);
}

// Threads of a row and chunks of a thread for n chunks of 8 channels.  Forward: at
// most two chunks a thread up to 2048 channels, more threads of a row rather than more
// registers of a thread (2^25 float32 elements, rows of 1024: two waves' halves with
// four chunks 116 us, a wave with two 97; rows of 2048 beside bf16 branches: a wave
// with four 71 us, two waves with two 64).  Backward: a thread keeps dw and db of its
// channels over the rows, and rows inside a wave need no barrier: up to four chunks,
// two at odd widths, whose last chunk takes registers of its own (1001 channels of bf16:
// half a wave with four 72 us, a wave with two 55); three for two waves from 2049
// channels on, where four waves with two stood half idle (2560: 77 us, 61).
// Rows of 64 channels by half waves, a quarter of the lanes at work, took 106 and 189
// us where eight lanes a row take 42 and 63.
template <typename TX, typename TB, template <typename, typename, int, int> class F, typename P>
hipError_t fwd_width(int n, const P& p, hipStream_t s) {
  if (n <= 8) return F<TX, TB, 8, 1>::run(p, s);
  if (n <= 16) return F<TX, TB, 16, 1>::run(p, s);
  if (n <= 32) return F<TX, TB, 32, 1>::run(p, s);
  if (n <= 64) return F<TX, TB, 64, 1>::run(p, s);
  if (n <= 128) return F<TX, TB, 64, 2>::run(p, s);
  if (n <= 256) return F<TX, TB, 128, 2>::run(p, s);
  if (n <= 512) return F<TX, TB, 256, 2>::run(p, s);
  if (n <= 768) return F<TX, TB, 256, 3>::run(p, s);
  if (n <= 1024) return F<TX, TB, 256, 4>::run(p, s);
  if (n <= 2048) return F<TX, TB, 1024, 2>::run(p, s);
  return hipErrorInvalidValue;
}
template <typename TX, typename TB, int TPR, int NCH> struct Fwd {
  static hipError_t run(const LnTrainParams& p, hipStream_t s) {
    constexpr int G = kGroups<TPR>;
    const dim3 grid((unsigned)((p.rows + G - 1) / G)), wg(kThreads<TPR>);
    hipLaunchKernelGGL((layernorm_fwd_kernel<TX, TB, TPR, NCH>), grid, wg, 0, s, p);
    return hipGetLastError();
  }
};
template <typename TX, typename TB, int TPR, int NCH, bool WHOLE> struct Bwd {
  static hipError_t run(const LnTrainBwdParams& p, hipStream_t s) {
    const dim3 grid((unsigned)p.n_wg), wg(kThreads<TPR>);
    if (p.n_wg > 0) hipLaunchKernelGGL((layernorm_bwd_kernel<TX, TB, TPR, NCH, WHOLE>), grid, wg, 0, s, p);
    if ((p.dw || p.db) && p.n_wg != 1)
      hipLaunchKernelGGL(layernorm_dw_kernel, dim3((unsigned)((p.C + 31) / 32), 2), dim3(1024), 0, s, p, p.n_wg);
    return hipGetLastError();
  }
};

template <typename TX, typename TB, bool WHOLE>
hipError_t bwd_width(int n, const LnTrainBwdParams& p, hipStream_t s) {
  if (n <= 8) return Bwd<TX, TB, 8, 1, WHOLE>::run(p, s);
  if (n <= 16) return Bwd<TX, TB, 16, 1, WHOLE>::run(p, s);
  if (n <= 32) return Bwd<TX, TB, 32, 1, WHOLE>::run(p, s);
  if (n <= 64) return Bwd<TX, TB, 32, 2, WHOLE>::run(p, s);
  if (n <= 96) return Bwd<TX, TB, 32, 3, WHOLE>::run(p, s);
  if (n <= 128) return Bwd<TX, TB, WHOLE ? 32 : 64, WHOLE ? 4 : 2, WHOLE>::run(p, s);
  if (n <= 192) return Bwd<TX, TB, 64, 3, WHOLE>::run(p, s);
  if (n <= 256) return Bwd<TX, TB, WHOLE ? 64 : 128, WHOLE ? 4 : 2, WHOLE>::run(p, s);
  if (n <= 384) return Bwd<TX, TB, 128, 3, WHOLE>::run(p, s);
  if (n <= 512) return Bwd<TX, TB, 256, 2, WHOLE>::run(p, s);
  if (n <= 768) return Bwd<TX, TB, 256, 3, WHOLE>::run(p, s);
  if (n <= 1024) return Bwd<TX, TB, 256, 4, WHOLE>::run(p, s);
  if (n <= 2048) return Bwd<TX, TB, 1024, 2, WHOLE>::run(p, s);
  return hipErrorInvalidValue;
}

template <typename TX, typename TB>
hipError_t run(const LnTrainParams& p, hipStream_t s) { return fwd_width<TX, TB, Fwd>((p.C + 7) / 8, p, s); }
template <typename TX, typename TB>
hipError_t run(const LnTrainBwdParams& p, hipStream_t s) {
  return p.C % 8 == 0 ? bwd_width<TX, TB, true>(p.C / 8, p, s) : bwd_width<TX, TB, false>((p.C + 7) / 8, p, s);
}

template <typename P>
hipError_t by_types(const P& p, int dtype, int branch, hipStream_t s) {
  if (dtype == kF32) {
    if (branch == kF32) return run<float, float>(p, s);
    return branch == kBF16 ? run<float, __bf16>(p, s) : run<float, _Float16>(p, s);
  }
  return dtype == kBF16 ? run<__bf16, __bf16>(p, s) : run<_Float16, _Float16>(p, s);
}

}  // namespace

// Threads of a row in the forward pass (fwd_width).
int layernorm_row_threads(int C) {
  const int n = (C + 7) / 8;
  return n <= 8 ? 8 : n <= 16 ? 16 : n <= 32 ? 32 : n <= 128 ? 64 : n <= 256 ? 128 : n <= 1024 ? 256 : 1024;
}

// Workgroups of the backward pass: as many as are resident, each with at least one
// round of rows.  One for up to four rounds of rows of a wave or less, which needs no
// second launch (32 x 768: 9 us, 6 + 3 and the gap between in two; 4 x 8192 17 and 9).
int layernorm_bwd_groups(int64_t rows, int C, int n_cu) {
  const int n = (C + 7) / 8;
  const bool whole = C % 8 == 0;
  const int waves = n > 1024 ? 16 : n > 384 ? 4 : n > (whole ? 256 : 192) ? 2 : 1;  // of a row that has several
  const int per = waves > 1 ? 1 : n <= 8 ? 32 : n <= 16 ? 16 : n <= (whole ? 128 : 96) ? 8 : 4;
  const int64_t rounds = (rows + per - 1) / per;
  if (rounds <= (waves > 1 ? 1 : 4)) return 1;
  const int64_t most = (int64_t)n_cu * (waves == 2 ? 4 : waves == 16 ? 1 : 2);
  return (int)(rounds < most ? rounds : most);
}

hipError_t launch_layernorm_train(const LnTrainParams& p, int dtype, int branch, hipStream_t s) {
  return by_types(p, dtype, branch, s);
}
hipError_t launch_layernorm_train_bwd(const LnTrainBwdParams& p, int dtype, int branch, hipStream_t s) {
  return by_types(p, dtype, branch, s);
}

}  // namespace saf
