// Embedding rows by token and the embedding's gradient (gfx950).
//
//   y[n] = scale W[t[n]]                  dW[v] = scale sum over n with t[n] = v of dy[n]
//
// Tokens that are ignored (t = ignore) give zero rows, other tokens outside the
// vocabulary NaN rows; neither has a gradient.
//
// The lookup is a copy: a thread moves 8 channels of a token.
//
// The gradient writes every row of dW, most of them zeros, and reads dy once.
// 1. The positions n are sorted by token, stable, least significant digit first
//    (9 bits at most a pass), while the other workgroups of the same launches
//    clear dW: the sort takes no time of its own as long as it is the shorter.
//    Up to kTile tokens one workgroup sorts in LDS in one launch; more go tile by
//    tile, each pass a launch that counts the digits of every tile and one that
//    places every tile's keys.
// 2. The sorted positions are cut into chunks; a thread sums 8 channels over
//    a chunk and writes the rows whose tokens lie inside it.  A token that crosses
//    chunks leaves float32 partial sums,
// 3. which the third launch adds in order.
// Every sum is in the order of n whatever runs beside it: no atomic touches a
// gradient, and each run gives the same bits.
#include "saf_kernels.h"
#include "saf_rowio.h"

namespace saf {

namespace {

constexpr int kSortThreads = 1024;
constexpr int kWaves = kSortThreads / 64;
constexpr int kKeys = kEmbedTile / kSortThreads;  // keys of a thread
constexpr int kBins = 1 << kEmbedDigit;

__device__ inline int64_t token_at(const void* tokens, int i64, int64_t st, int64_t n) {
  return i64 ? reinterpret_cast<const int64_t*>(tokens)[n * st] : (int64_t)reinterpret_cast<const int32_t*>(tokens)[n * st];
}

template <typename TW, typename TY>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const EmbedParams p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.units) return;
  const uint32_t n = p.per_row.div(i);
  const int c = 8 * (int)(i - n * p.per_row.d), C = p.C;
  const int64_t tok = token_at(p.tokens, p.tok_i64, p.tok_st, n);
  float f[8];
  if (tok >= 0 && tok < p.V && tok != p.ignore) {
    load_row8(reinterpret_cast<const TW*>(p.w) + tok * p.w_rs, c, C, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= p.scale;
  } else {
    const float x = tok == p.ignore ? 0.f : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = x;
  }
  store_row8(reinterpret_cast<TY*>(p.y) + (int64_t)n * C, c, C, f);
}

// ---- sorting -----------------------------------------------------------------

// Key of a token: itself, or V (behind every word) where it has no gradient.
__device__ inline uint32_t key_of(const EmbedBwdParams& p, int64_t n) {
  const int64_t t = token_at(p.tokens, p.tok_i64, p.tok_st, n);
  return t >= 0 && t < p.V && t != p.ignore ? (uint32_t)t : (uint32_t)p.V;
}

// Zeros over this workgroup's part of bytes lo..hi of dW (16-byte aligned).
__device__ inline void clear_part(const EmbedBwdParams& p, int64_t lo, int64_t hi, int wg, int n_wg) {
  char* base = reinterpret_cast<char*>(p.dw);
  const int64_t whole = lo + (hi - lo) / 16 * 16;
  for (int64_t o = lo + 16 * ((int64_t)wg * kSortThreads + threadIdx.x); o < whole; o += 16 * (int64_t)n_wg * kSortThreads)
    *reinterpret_cast<uint4*>(base + o) = make_uint4(0, 0, 0, 0);
  // the last bytes of dW, of which 16-bit types leave an even number
  const int64_t o = whole + 2 * threadIdx.x;
  if (wg == 0 && o < hi) *reinterpret_cast<uint16_t*>(base + o) = 0;
}

// Positions of a tile's keys among equal digits.  Wave w has keys
// (w iters + i) 64 + lane in the order of i and lane; the lanes of one digit find
// each other by a ballot per bit, and the first of them adds their number to the
// digit's count in count[w], which afterwards holds the wave's keys per digit.
__device__ inline void rank_keys(const uint32_t (&key)[kKeys], uint32_t (&rank)[kKeys], int iters, int valid, int shift,
                                 int bits, uint32_t (*count)[kBins]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b = threadIdx.x; b < kWaves * kBins; b += kSortThreads) (&count[0][0])[b] = 0;
  __syncthreads();
  const uint64_t before = (uint64_t(1) << lane) - 1;
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    if (i >= iters) break;
    const bool on = (wave * iters + i) * 64 + lane < valid;
    const uint32_t d = (key[i] >> shift) & ((1u << bits) - 1);
    uint64_t same = __ballot(on);
    for (int b = 0; b < bits; ++b) {
      const uint64_t m = __ballot((d >> b) & 1);
      same &= (d >> b) & 1 ? m : ~m;
    }
    const bool first = on && (same & before) == 0;
    uint32_t at = 0;
    if (first) at = atomicAdd(&count[wave][d], (uint32_t)__popcll(same));
    // lanes without a key take any lane's
    rank[i] = __shfl(at, on ? __ffsll((unsigned long long)same) - 1 : lane, 64) + (uint32_t)__popcll(same & before);
  }
  __syncthreads();
}

// Exclusive sums over bins and waves: count[w][d] becomes the first place of wave
// w's keys of digit d, from the start start(d, total of the tile) on, or
// from the running sum of the tile alone (start == null).
__device__ inline void place_bins(uint32_t (*count)[kBins], uint32_t* total, const uint32_t* start) {
  const int d = threadIdx.x;
  if (d < kBins) {
    uint32_t s = 0;
    for (int w = 0; w < kWaves; ++w) {
      const uint32_t n = count[w][d];
      count[w][d] = s;
      s += n;
    }
    total[d] = s;
  }
  __syncthreads();
  if (start == nullptr) {
    // running sum over the bins, doubling the reach each round
    for (int o = 1; o < kBins; o <<= 1) {
      const uint32_t v = d < kBins && d >= o ? total[d - o] : 0;
      __syncthreads();
      if (d < kBins) total[d] += v;
      __syncthreads();
    }
  }
  if (d < kBins) {
    const uint32_t first = start ? start[d] : (d ? total[d - 1] : 0);
    for (int w = 0; w < kWaves; ++w) count[w][d] += first;
  }
  __syncthreads();
}

// Workgroup 0: all passes over up to kEmbedTile tokens in LDS.  The others clear dW.
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(const EmbedBwdParams p) {
  __shared__ uint32_t count[kWaves][kBins];
  __shared__ uint32_t total[kBins];
  __shared__ uint2 held[kEmbedTile];
  if (blockIdx.x > 0) {
    clear_part(p, 0, p.dw_bytes, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, N = (int)p.N;
  const int iters = (N + kSortThreads - 1) / kSortThreads;
  uint32_t key[kKeys], pos[kKeys], rank[kKeys];
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const int at = (wave * iters + i) * 64 + lane;
    pos[i] = at;
    key[i] = i < iters && at < N ? key_of(p, at) : 0;
  }
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    rank_keys(key, rank, iters, N, shift, p.bits, count);
    place_bins(count, total, nullptr);
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
      if (i < iters && (wave * iters + i) * 64 + lane < N)
        held[count[wave][(key[i] >> shift) & ((1u << p.bits) - 1)] + rank[i]] = make_uint2(key[i], pos[i]);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      const int at = (wave * iters + i) * 64 + lane;
      if (i < iters && at < N) {
        const uint2 h = held[at];
        key[i] = h.x;
        pos[i] = h.y;
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const int at = (wave * iters + i) * 64 + lane;
    if (i < iters && at < N) p.sorted[at] = make_uint2(key[i], pos[i]);
  }
}

// The tile's keys of one pass, from the tokens in the first.
__device__ inline uint2 tile_key(const EmbedBwdParams& p, const uint2* from, int64_t n) {
  return from ? from[n] : make_uint2(key_of(p, n), (uint32_t)n);
}

// Digit counts of every tile; workgroups behind the tiles clear their part.
__global__ __launch_bounds__(kSortThreads) void embed_count_kernel(const EmbedBwdParams p, const uint2* from, int shift,
                                                                   int64_t lo, int64_t hi) {
  __shared__ uint32_t count[kBins];
  if ((int)blockIdx.x >= p.n_tiles) {
    clear_part(p, lo, hi, blockIdx.x - p.n_tiles, gridDim.x - p.n_tiles);
    return;
  }
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) count[b] = 0;
  __syncthreads();
  const int64_t n0 = (int64_t)blockIdx.x * kEmbedTile;
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const int64_t n = n0 + i * kSortThreads + threadIdx.x;
    if (n < p.N) atomicAdd(&count[(tile_key(p, from, n).x >> shift) & ((1u << p.bits) - 1)], 1u);
  }
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) p.counts[(int64_t)blockIdx.x * kBins + b] = count[b];
}

// Every tile's keys to their places of this pass.
__global__ __launch_bounds__(kSortThreads) void embed_place_kernel(const EmbedBwdParams p, const uint2* from, uint2* to,
                                                                   int shift, int64_t lo, int64_t hi) {
  __shared__ uint32_t count[kWaves][kBins];
  __shared__ uint32_t total[kBins], start[kBins];
  if ((int)blockIdx.x >= p.n_tiles) {
    clear_part(p, lo, hi, blockIdx.x - p.n_tiles, gridDim.x - p.n_tiles);
    return;
  }
  // first place of each digit for this tile: all smaller digits, and this
  // digit in the tiles before
  const int d = threadIdx.x;
  uint32_t mine = 0, all = 0;
  if (d < kBins) {
    for (int t = 0; t < p.n_tiles; ++t) {
      const uint32_t n = p.counts[(int64_t)t * kBins + d];
      if (t < (int)blockIdx.x) mine += n;
      all += n;
    }
    total[d] = all;
  }
  __syncthreads();
  for (int o = 1; o < kBins; o <<= 1) {
    const uint32_t v = d < kBins && d >= o ? total[d - o] : 0;
    __syncthreads();
    if (d < kBins) total[d] += v;
    __syncthreads();
  }
  if (d < kBins) start[d] = total[d] - all + mine;
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * kEmbedTile;
  const int valid = (int)(p.N - n0 < kEmbedTile ? p.N - n0 : kEmbedTile);
  uint32_t key[kKeys], pos[kKeys], rank[kKeys];
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const int at = (wave * kKeys + i) * 64 + lane;
    const uint2 k = at < valid ? tile_key(p, from, n0 + at) : make_uint2(0, 0);
    key[i] = k.x;
    pos[i] = k.y;
  }
  rank_keys(key, rank, kKeys, valid, shift, p.bits, count);
  place_bins(count, total, start);
#pragma unroll
  for (int i = 0; i < kKeys; ++i)
    if ((wave * kKeys + i) * 64 + lane < valid)
      to[count[wave][(key[i] >> shift) & ((1u << p.bits) - 1)] + rank[i]] = make_uint2(key[i], pos[i]);
}

// ---- sums --------------------------------------------------------------------

template <typename TW, typename TY>
__global__ __launch_bounds__(256) void embed_sum_kernel(const EmbedBwdParams p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.units) return;
  const uint32_t chunk = p.per_row.div(i);
  const int c = 8 * (int)(i - chunk * p.per_row.d), C = p.C;
  const int64_t lo = (int64_t)chunk * p.chunk, hi = lo + p.chunk < p.N ? lo + p.chunk : p.N;
  uint32_t word = p.sorted[lo].x;
  if (word == (uint32_t)p.V) return;
  // the chunk's first word may have begun before it
  bool head = lo > 0 && p.sorted[lo - 1].x == word;
  const TY* dy = reinterpret_cast<const TY*>(p.dy);
  TW* dw = reinterpret_cast<TW*>(p.dw);
  float acc[8] = {};
  auto finish = [&](bool open) {  // open: the word goes on in the next chunk
    if (head) {
      store_row8(p.head + (int64_t)chunk * C, c, C, acc);
    } else if (open) {
      store_row8(p.tail + (int64_t)chunk * C, c, C, acc);
    } else {
      float o[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = acc[e] * p.scale;
      store_row8(dw + (int64_t)word * C, c, C, o);
    }
  };
  for (int64_t n = lo; n < hi; ++n) {
    const uint2 k = p.sorted[n];
    if (k.x != word) {
      finish(false);
      head = false;
      word = k.x;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] = 0.f;
      if (word == (uint32_t)p.V) return;
    }
    float f[8];
    load_row8(dy + (int64_t)k.y * p.dy_rs, c, C, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += f[e];
  }
  finish(hi < p.N && p.sorted[hi].x == word);
}

// Words that cross chunks: the chunk where one begins adds its partials.
template <typename TW>
__global__ __launch_bounds__(256) void embed_join_kernel(const EmbedBwdParams p) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= p.units) return;
  const uint32_t chunk = p.per_row.div(i);
  const int c = 8 * (int)(i - chunk * p.per_row.d), C = p.C;
  const int64_t lo = (int64_t)chunk * p.chunk, hi = lo + p.chunk;
  if (hi >= p.N) return;
  const uint32_t word = p.sorted[hi - 1].x;
  if (word == (uint32_t)p.V || p.sorted[hi].x != word) return;
  if (lo > 0 && p.sorted[lo - 1].x == word) return;  // begun in an earlier chunk
  float acc[8];
  load_row8(p.tail + (int64_t)chunk * C, c, C, acc);
  for (int64_t k = chunk + 1; k * p.chunk < p.N && p.sorted[k * p.chunk].x == word; ++k) {
    float f[8];
    load_row8(p.head + k * C, c, C, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] += f[e];
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) acc[e] *= p.scale;
  store_row8(reinterpret_cast<TW*>(p.dw) + (int64_t)word * C, c, C, acc);
}

template <typename TW>
hipError_t bwd_t(const EmbedBwdParams& p, int dtype, hipStream_t s) {
  const dim3 sort_wg(kSortThreads);
  if (p.n_tiles == 0) {  // nothing but zeros
    hipLaunchKernelGGL(embed_count_kernel, dim3((unsigned)p.n_clear), sort_wg, 0, s, p, (const uint2*)nullptr, 0, (int64_t)0,
                       p.dw_bytes);
    return hipGetLastError();
  }
  if (p.n_tiles == 1) {
    hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)(1 + p.n_clear)), sort_wg, 0, s, p);
  } else {
    // an equal part of the zeros beside each of the 2 x passes launches; the
    // pass that comes last writes `sorted`
    const int64_t step = (p.dw_bytes / (2 * p.passes) + 15) / 16 * 16;
    const uint2* from = nullptr;
    for (int i = 0; i < p.passes; ++i) {
      uint2* to = (p.passes - 1 - i) & 1 ? p.sorted2 : p.sorted;
      for (int half = 0; half < 2; ++half) {
        const int64_t lo = (2 * i + half) * step;
        int64_t hi = 2 * i + half == 2 * p.passes - 1 ? p.dw_bytes : lo + step;
        if (hi > p.dw_bytes) hi = p.dw_bytes;
        const dim3 grid((unsigned)(p.n_tiles + (lo < hi ? p.n_clear : 0)));
        if (half == 0)
          hipLaunchKernelGGL(embed_count_kernel, grid, sort_wg, 0, s, p, from, i * p.bits, lo, hi);
        else
          hipLaunchKernelGGL(embed_place_kernel, grid, sort_wg, 0, s, p, from, to, i * p.bits, lo, hi);
      }
      from = to;
    }
  }
  const dim3 grid((p.units + 255) / 256), wg(256);
  if (dtype == kF32) hipLaunchKernelGGL((embed_sum_kernel<TW, float>), grid, wg, 0, s, p);
  else if (dtype == kBF16) hipLaunchKernelGGL((embed_sum_kernel<TW, __bf16>), grid, wg, 0, s, p);
  else hipLaunchKernelGGL((embed_sum_kernel<TW, _Float16>), grid, wg, 0, s, p);
  if (p.N > p.chunk) hipLaunchKernelGGL((embed_join_kernel<TW>), grid, wg, 0, s, p);
  return hipGetLastError();
}

template <typename TW>
hipError_t fwd_t(const EmbedParams& p, int dtype, hipStream_t s) {
  const dim3 grid((p.units + 255) / 256), wg(256);
  if (dtype == kF32) hipLaunchKernelGGL((embed_fwd_kernel<TW, float>), grid, wg, 0, s, p);
  else if (dtype == kBF16) hipLaunchKernelGGL((embed_fwd_kernel<TW, __bf16>), grid, wg, 0, s, p);
  else hipLaunchKernelGGL((embed_fwd_kernel<TW, _Float16>), grid, wg, 0, s, p);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_embed(const EmbedParams& p, int w_dtype, int y_dtype, hipStream_t s) {
  if (w_dtype == kF32) return fwd_t<float>(p, y_dtype, s);
  if (w_dtype == kBF16) return fwd_t<__bf16>(p, y_dtype, s);
  return fwd_t<_Float16>(p, y_dtype, s);
}
hipError_t launch_embed_bwd(const EmbedBwdParams& p, int w_dtype, int y_dtype, hipStream_t s) {
  if (w_dtype == kF32) return bwd_t<float>(p, y_dtype, s);
  if (w_dtype == kBF16) return bwd_t<__bf16>(p, y_dtype, s);
  return bwd_t<_Float16>(p, y_dtype, s);
}

}  // namespace saf
