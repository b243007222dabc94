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
//    Up to kEmbedFew tokens nothing is sorted: each workgroup looks for the words of its
//    rows in the list of tokens.  Up to kEmbedOnce tokens one workgroup sorts in LDS in
//    one launch.  More go tile by tile, a launch a pass that places every tile's keys;
//    each workgroup counts the digits of all keys for itself, from kEmbedCounted tokens
//    on a launch before it counts them once, and past kEmbedScanned tiles another sums
//    the counts up.
// 2. The sorted positions are cut into chunks; a wave sums 256 channels over a chunk
//    and writes the rows whose tokens lie inside it.  A token that crosses chunks
//    leaves float32 partial sums,
// 3. which the third launch adds: every kLanes-th of them in one run of their order,
//    the part of the token's first chunk ahead of the first run, then the runs in order.
// The order is fixed by N and C, which decide the chunks, and by the positions of the
// token, whatever runs beside it: no atomic touches a gradient, and each run gives the
// same bits.  It is the order of n inside a chunk only (up to kEmbedFew tokens: in all).
#include "saf_kernels.h"
#include "saf_rowio.h"

namespace saf {

namespace {

constexpr int kSortThreads = 1024;
constexpr int kWaves = kSortThreads / 64;
constexpr int kBins = 1 << kEmbedDigit;
// Units from which a thread of the lookup has two: 131072 tokens of 896 bf16 channels 44 us
// against 46, 4096 the same 6.7 either way.
constexpr uint32_t kWideUnits = 1 << 19;

// U units a thread, 256 apart; their tokens are read together, then their rows.
template <typename TW, typename TY, int U, bool WHOLE>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const EmbedParams p) {
  const uint32_t first = blockIdx.x * (256 * U) + threadIdx.x;
  const int C = p.C;
  uint32_t n[U];
  int c[U];
  int64_t tok[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t i = first + 256 * u;
    n[u] = p.per_row.div(i);
    c[u] = i < p.units ? 8 * (int)(i - n[u] * p.per_row.d) : C;  // C: nothing to move
    if (i >= p.units) n[u] = 0;
  }
  if (p.tok_i64) {
#pragma unroll
    for (int u = 0; u < U; ++u) tok[u] = reinterpret_cast<const int64_t*>(p.tokens)[n[u] * p.tok_st];
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) tok[u] = reinterpret_cast<const int32_t*>(p.tokens)[n[u] * p.tok_st];
  }
  Row8<TW> w[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const bool word = tok[u] >= 0 && tok[u] < p.V;
    w[u] = load_raw8<WHOLE>(reinterpret_cast<const TW*>(p.w) + (word ? tok[u] * p.w_rs : 0), c[u], C);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float f[8];
    w[u].unpack(f);
    const bool word = tok[u] >= 0 && tok[u] < p.V && tok[u] != p.ignore;
    const float other = tok[u] == p.ignore ? 0.f : __uint_as_float(0x7fc00000u);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = word ? f[e] * p.scale : other;
    stream_row8<WHOLE>(reinterpret_cast<TY*>(p.y) + (int64_t)n[u] * C, c[u], C, f);
  }
}

// ---- sorting -----------------------------------------------------------------

// Keys of positions at(0), at(1), ...: the token itself, or V (behind every word)
// where it has no gradient; some value at and past `end`.  Every token is read
// before the first is looked at.
template <int KEYS, typename At>
__device__ inline void keys_of(const EmbedBwdParams& p, int64_t end, At at, uint32_t (&key)[KEYS]) {
  int64_t t[KEYS];
  if (p.tok_i64) {
#pragma unroll
    for (int i = 0; i < KEYS; ++i) t[i] = at(i) < end ? reinterpret_cast<const int64_t*>(p.tokens)[at(i) * p.tok_st] : 0;
  } else {
    int32_t t32[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) t32[i] = at(i) < end ? reinterpret_cast<const int32_t*>(p.tokens)[at(i) * p.tok_st] : 0;
#pragma unroll
    for (int i = 0; i < KEYS; ++i) t[i] = t32[i];
  }
#pragma unroll
  for (int i = 0; i < KEYS; ++i) key[i] = t[i] >= 0 && t[i] < p.V && t[i] != p.ignore ? (uint32_t)t[i] : (uint32_t)p.V;
}

// Zeros over this workgroup's part of bytes lo..hi of dW (16-byte aligned), past the
// caches: dW is mostly zeros that nothing reads soon, and would take the place of dy
// and of the embedding there (32768 tokens, 151936 x 896 bf16: the kernels of both
// directions together 107 us through the caches, 90 past them; 65536 tokens, 50304 x 768
// float32: 120 and 99; 16384: 60 and 62).
__device__ inline void clear_part(const EmbedBwdParams& p, int64_t lo, int64_t hi, int wg, int n_wg) {
  char* base = reinterpret_cast<char*>(p.dw);
  const int64_t whole = lo + (hi - lo) / 16 * 16;
  for (int64_t o = lo + 16 * ((int64_t)wg * kSortThreads + threadIdx.x); o < whole; o += 16 * (int64_t)n_wg * kSortThreads)
    __builtin_nontemporal_store(u32x4_any{0, 0, 0, 0}, reinterpret_cast<u32x4_any*>(base + o));
  // the last bytes of dW, of which 16-bit types leave an even number
  const int64_t o = whole + 2 * threadIdx.x;
  if (wg == 0 && o < hi) *reinterpret_cast<uint16_t*>(base + o) = 0;
}

// A workgroup places up to kEmbedOnce keys stably by a digit.  Each wave owns a run of
// them; counts[w] first receives the number of wave w's keys of each digit, then
// the place of the first of them, and a key takes its digit's place and moves it on
// by one.  Places and numbers have 16 bits, two digits a word.
typedef uint32_t Counts[kWaves][kBins / 2];

__device__ inline void clear_counts(Counts& counts) {
  for (int b = threadIdx.x; b < kWaves * kBins / 2; b += kSortThreads) (&counts[0][0])[b] = 0;
  __syncthreads();
}

__device__ inline void count_key(Counts& counts, uint32_t d) {
  atomicAdd(&counts[threadIdx.x >> 6][d >> 1], 1u << (16 * (d & 1)));
}

// Sum of v over the threads up to this one; `sums` is LDS of one value a wave.
__device__ inline uint32_t running_sum(uint32_t v, uint32_t* sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  if (lane == 63) sums[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += sums[w];
  return v;
}

// Numbers into places, in the order of digits, then waves.
__device__ inline void places(Counts& counts, uint32_t* sums) {
  __syncthreads();
  const int d = threadIdx.x;  // a pair of digits
  uint32_t n[kWaves] = {}, all = 0;
  if (d < kBins / 2) {
#pragma unroll
    for (int w = 0; w < kWaves; ++w) n[w] = counts[w][d];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += n[w];  // either half is kEmbedOnce at most: no carry
  }
  const uint32_t both = (all & 0xffff) + (all >> 16);
  const uint32_t low = running_sum(both, sums) - both;
  if (d < kBins / 2) {
    uint32_t at = low | (low + (all & 0xffff)) << 16;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      counts[w][d] = at;
      at += n[w];
    }
  }
  __syncthreads();
}

// The place of this lane's key of digit d, for the lanes that have one: lanes of
// one digit find each other by a ballot per bit, and the first of them takes places
// for all, which they fill in the order of lanes.
__device__ inline uint32_t take_place(Counts& counts, uint32_t d, bool on) {
  // other: the lanes whose digit differs in some bit, or that have none
  const uint64_t some = __ballot(on);
  uint32_t lo = ~(uint32_t)some, hi = ~(uint32_t)(some >> 32);
#pragma unroll
  for (int b = 0; b < kEmbedDigit; ++b) {  // a shorter digit's upper bits are zeros of all lanes
    const uint32_t bit = (uint32_t)((int32_t)(d << (31 - b)) >> 31);
    const uint64_t m = __ballot(bit != 0);
    lo |= (uint32_t)m ^ bit;
    hi |= (uint32_t)(m >> 32) ^ bit;
  }
  lo = ~lo;
  hi = ~hi;
  const uint32_t before = __builtin_amdgcn_mbcnt_hi(hi, __builtin_amdgcn_mbcnt_lo(lo, 0));
  uint32_t at = 0;
  if (on && before == 0) {
    const uint32_t n = (uint32_t)(__popc(lo) + __popc(hi));
    at = atomicAdd(&counts[threadIdx.x >> 6][d >> 1], n << (16 * (d & 1))) >> (16 * (d & 1)) & 0xffff;
  }
  const int first = lo ? __ffs((int)lo) - 1 : 31 + __ffs((int)hi);
  return __shfl(at, on ? first : (int)(threadIdx.x & 63), 64) + before;
}

// Workgroup 0: all passes over up to kEmbedOnce tokens in LDS, the keys at their
// positions and the positions in the order so far.  The others clear dW.
__global__ __launch_bounds__(kSortThreads) void embed_sort_kernel(const EmbedBwdParams p) {
  __shared__ Counts counts;
  __shared__ uint32_t sums[kWaves];
  __shared__ uint32_t keys[kEmbedOnce];
  __shared__ uint16_t order[2][kEmbedOnce];
  if (blockIdx.x > 0) {
    clear_part(p, 0, p.dw_bytes, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, N = (int)p.N;
  for (int n0 = threadIdx.x; n0 < N; n0 += 4 * kSortThreads) {
    const auto at = [&](int i) { return n0 + i * kSortThreads; };
    uint32_t key[4];
    keys_of(p, N, at, key);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at(i) < N) {
        keys[at(i)] = key[i];
        order[0][at(i)] = (uint16_t)at(i);
      }
  }
  const int run = (N + kSortThreads - 1) / kSortThreads * 64, lo = wave * run;
  const uint32_t mask = (1u << p.bits) - 1;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * p.bits;
    const uint16_t* from = order[pass & 1];
    uint16_t* to = order[~pass & 1];
    clear_counts(counts);
    for (int at = lo + lane; at < lo + run; at += 64)
      if (at < N) count_key(counts, keys[from[at]] >> shift & mask);
    places(counts, sums);
    for (int at = lo + lane; at < lo + run; at += 64) {
      const bool on = at < N;
      const uint32_t pos = on ? from[at] : 0;
      const uint32_t place = take_place(counts, keys[pos] >> shift & mask, on);
      if (on) to[place] = (uint16_t)pos;
    }
    __syncthreads();
  }
  for (int at = threadIdx.x; at < N; at += kSortThreads) {
    const uint32_t pos = order[p.passes & 1][at];
    p.sorted[at] = make_uint2(keys[pos], pos);
  }
}

// Keys and positions at(0), at(1), ..., from the tokens in the first pass.
constexpr int kKeys = kEmbedTile / kSortThreads;
template <int KEYS, typename At>
__device__ inline void tile_keys(const EmbedBwdParams& p, const uint2* from, At at, uint32_t (&key)[KEYS],
                                 uint32_t (&pos)[KEYS]) {
  if (from) {
    uint2 k[KEYS];
#pragma unroll
    for (int i = 0; i < KEYS; ++i) k[i] = at(i) < p.N ? from[at(i)] : make_uint2(0, 0);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) {
      key[i] = k[i].x;
      pos[i] = k[i].y;
    }
  } else {
    keys_of(p, p.N, at, key);
#pragma unroll
    for (int i = 0; i < KEYS; ++i) pos[i] = (uint32_t)at(i);
  }
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
  const auto at = [&](int i) { return n0 + i * kSortThreads + threadIdx.x; };
  uint32_t key[kKeys], pos[kKeys];
  tile_keys(p, from, at, key, pos);
#pragma unroll
  for (int i = 0; i < kKeys; ++i)
    if (at(i) < p.N) atomicAdd(&count[key[i] >> shift & ((1u << p.bits) - 1)], 1u);
  __syncthreads();
  for (int b = threadIdx.x; b < kBins; b += kSortThreads) p.counts[(int64_t)blockIdx.x * kBins + b] = count[b];
}

// Counts of very many tiles summed up, once: a tile's become those of the tiles before
// it, the row behind the last the totals.  Workgroups of 64 digits, each of their waves
// with a run of tiles.
__global__ __launch_bounds__(1024) void embed_scan_kernel(const EmbedBwdParams p) {
  __shared__ uint32_t sums[16][64];
  const int col = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t* of = p.counts + blockIdx.x * 64 + col;
  const int run = (p.n_tiles + 15) / 16, lo = wave * run, hi = lo + run < p.n_tiles ? lo + run : p.n_tiles;
  uint32_t s = 0;
#pragma unroll 16
  for (int t = lo; t < hi; ++t) s += of[(int64_t)t * kBins];
  sums[wave][col] = s;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += sums[w][col];
#pragma unroll 16
  for (int t = lo; t < hi; ++t) {
    const uint32_t n = of[(int64_t)t * kBins];
    of[(int64_t)t * kBins] = before;
    before += n;
  }
  if (wave == 15) of[(int64_t)p.n_tiles * kBins] = before;
}

// Every tile's keys to their places of this pass.
__global__ __launch_bounds__(kSortThreads) void embed_place_kernel(const EmbedBwdParams p, const uint2* from, uint2* to,
                                                                   int shift, int64_t lo, int64_t hi) {
  __shared__ Counts counts;
  __shared__ uint32_t sums[2][kWaves], part[2][kBins], base[kBins];
  if ((int)blockIdx.x >= p.n_tiles) {
    clear_part(p, lo, hi, blockIdx.x - p.n_tiles, gridDim.x - p.n_tiles);
    return;
  }
  const int64_t n0 = (int64_t)blockIdx.x * kEmbedTile;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const auto at = [&](int i) { return n0 + (wave * kKeys + i) * 64 + lane; };
  const uint32_t mask = (1u << p.bits) - 1;
  uint32_t key[kKeys], pos[kKeys];
  tile_keys(p, from, at, key, pos);
  clear_counts(counts);
#pragma unroll
  for (int i = 0; i < kKeys; ++i)
    if (at(i) < p.N) count_key(counts, key[i] >> shift & mask);
  // of each digit: the keys in the tiles before, and in all
  const int d = threadIdx.x;
  uint32_t before = 0, all = 0;
  if (p.counts == nullptr) {
    for (int b = d; b < 2 * kBins; b += kSortThreads) (&part[0][0])[b] = 0;
    __syncthreads();
    for (int64_t first = 0; first < p.N; first += 8 * kSortThreads) {
      const auto any = [&](int i) { return first + i * kSortThreads + threadIdx.x; };
      uint32_t other[8], unused[8];
      tile_keys(p, from, any, other, unused);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (any(i) < p.N) atomicAdd(&part[any(i) < n0][other[i] >> shift & mask], 1u);
    }
    __syncthreads();
    if (d < kBins) {
      before = part[1][d];
      all = before + part[0][d];
    }
  } else if (d < kBins && p.n_tiles > kEmbedScanned) {
    before = p.counts[(int64_t)blockIdx.x * kBins + d];
    all = p.counts[(int64_t)p.n_tiles * kBins + d];
  } else if (d < kBins) {
    const uint32_t* of = p.counts + d;
#pragma unroll 16
    for (int t = 0; t < p.n_tiles; ++t) {
      const uint32_t n = of[(int64_t)t * kBins];
      before += t < (int)blockIdx.x ? n : 0;
      all += n;
    }
  }
  const uint32_t smaller = running_sum(all, sums[0]) - all;
  places(counts, sums[1]);
  // from a place among the tile's keys to one among all keys
  if (d < kBins) base[d] = smaller + before - (counts[0][d >> 1] >> (16 * (d & 1)) & 0xffff);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const uint32_t digit = key[i] >> shift & mask;
    const uint32_t place = take_place(counts, digit, at(i) < p.N);
    if (at(i) < p.N) to[base[digit] + place] = make_uint2(key[i], pos[i]);
  }
}

// ---- sums --------------------------------------------------------------------

// A wave sums 256 channels of a chunk, four a lane.  Its lanes read the chunk's
// positions in one piece; which word a row belongs to is the same for all of them,
// so the rows' addresses and the branches at a word's end are scalar, and kRows rows
// at a time are on their way before the first is added.
constexpr int kRows = 16;

template <bool WHOLE, typename T>
__device__ inline void store4(T* p, const float (&f)[4], int n) {
  if (n == 4) {
    Row4<T>::store(p, f);
  } else if (!WHOLE) {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) p[e] = static_cast<T>(f[e]);
  }
}

template <typename TW, typename TY, bool WHOLE>  // WHOLE: C is a multiple of 4
__global__ __launch_bounds__(256) void embed_sum_kernel(const EmbedBwdParams p) {
  const uint32_t i = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
  if (i >= p.units) return;
  const uint32_t chunk = p.per_row.div(i);
  const int lane = threadIdx.x & 63, C = p.C;
  const int c = 256 * (int)(i - chunk * p.per_row.d) + 4 * lane;
  // a lane behind the row's end reads its beginning and stores nothing
  const int at = c < C ? c : 0, have = C - at < 4 ? C - at : 4, put = c < C ? have : 0;
  const int64_t lo = (int64_t)chunk * p.chunk;
  const int n = (int)(p.N - lo < p.chunk ? p.N - lo : p.chunk);
  const uint32_t V = (uint32_t)p.V;
  const uint2 mine = lane < n ? p.sorted[lo + lane] : make_uint2(V, 0);
  const uint32_t left = lo > 0 ? p.sorted[lo - 1].x : V, right = lo + n < p.N ? p.sorted[lo + n].x : V;
  const TY* dy = reinterpret_cast<const TY*>(p.dy);
  TW* dw = reinterpret_cast<TW*>(p.dw);
  const int live = __popcll(__ballot(mine.x != V));  // words come first
  uint32_t word = V;  // none yet
  bool head = false;  // the chunk's first word has begun before it
  float acc[4] = {};
  auto finish = [&](bool open) {  // open: the word goes on in the next chunk
    if (head || open) {
      store4<WHOLE>((head ? p.head : p.tail) + (int64_t)chunk * C + c, acc, put);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= p.scale;
      store4<WHOLE>(dw + (int64_t)word * C + c, acc, put);
    }
  };
  for (int j0 = 0; j0 < live; j0 += kRows) {
    Row4<TY> rows[kRows];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const uint32_t row = __builtin_amdgcn_readlane(mine.y, j0 + j < live ? j0 + j : 0);
      const TY* from = dy + (int64_t)row * p.dy_rs + at;
      if (WHOLE || have == 4) rows[j] = Row4<TY>::load(from);
      else rows[j] = Row4<TY>::load_part(from, have);
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      if (j0 + j >= live) break;
      const uint32_t w = __builtin_amdgcn_readlane(mine.x, j0 + j);
      if (w != word) {
        if (j0 + j == 0) head = w == __builtin_amdgcn_readfirstlane(left);
        else finish(false), head = false;
        word = w;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = 0.f;
      }
      float f[4];
      rows[j].unpack(f);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += f[e];
    }
  }
  if (word != V) finish(word == __builtin_amdgcn_readfirstlane(right));
}

// Up to kEmbedFew tokens, as many as a wave has lanes: a workgroup owns a run of rows
// of dW, clears them, finds the words among them in the list of all tokens, and sums
// their rows of dy, a wave 256 channels of a word.  One launch, no workspace.
constexpr int kFewThreads = 512;

template <typename TW, typename TY>
__global__ __launch_bounds__(kFewThreads) void embed_few_kernel(const EmbedBwdParams p) {
  static_assert(kEmbedFew == 64, "a lane a token");
  const int N = (int)p.N, C = p.C, t = threadIdx.x, lane = t & 63;
  const int64_t per = (p.V + gridDim.x - 1) / gridDim.x, v0 = blockIdx.x * per;
  if (v0 >= p.V) return;
  const int64_t v1 = v0 + per < p.V ? v0 + per : p.V;
  uint32_t key[1];  // every wave has all of them
  keys_of(p, N, [&](int) { return lane; }, key);
  // rows as bytes: whole pieces of 16, and what is left before and behind them
  char* base = reinterpret_cast<char*>(p.dw);
  const int64_t lo = v0 * C * (int64_t)sizeof(TW), hi = v1 * C * (int64_t)sizeof(TW);
  const int64_t a = (lo + 15) / 16 * 16 < hi ? (lo + 15) / 16 * 16 : hi, b = hi / 16 * 16 > a ? hi / 16 * 16 : a;
  for (int64_t o = a + 16 * t; o < b; o += 16 * kFewThreads)
    __builtin_nontemporal_store(u32x4_any{0, 0, 0, 0}, reinterpret_cast<u32x4_any*>(base + o));
  if (lo + 2 * t < a) *reinterpret_cast<uint16_t*>(base + lo + 2 * t) = 0;
  if (b + 2 * t < hi) *reinterpret_cast<uint16_t*>(base + b + 2 * t) = 0;
  __builtin_amdgcn_s_waitcnt(0);  // a row's zeros are written before another wave writes its sums
  __syncthreads();
  const TY* dy = reinterpret_cast<const TY*>(p.dy);
  const int blocks = (C + 255) / 256;
  // the words of these rows one after the other, their channels dealt out to the waves
  uint64_t left = __ballot(lane < N && key[0] >= (uint32_t)v0 && key[0] < (uint32_t)v1);
  for (int unit = 0; left; unit += blocks) {
    const uint32_t word = __builtin_amdgcn_readlane(key[0], __builtin_ctzll(left));
    const uint64_t all = __ballot(lane < N && key[0] == word);
    left &= ~all;
    for (int block = 0; block < blocks; ++block) {
      if ((unit + block) % (kFewThreads / 64) != t >> 6) continue;
      const int c = 256 * block + 4 * lane;
      const int at = c < C ? c : 0, have = C - at < 4 ? C - at : 4, put = c < C ? have : 0;
      float acc[4] = {};
      for (uint64_t is = all; is;) {
        // eight rows on their way before the first is added; behind the last a repeat of it
        constexpr int G = 8;
        const int live = __popcll(is);
        int n[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
          n[j] = is ? __builtin_ctzll(is) : n[j ? j - 1 : 0];
          is &= is - 1;
        }
        Row4<TY> rows[G];
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const TY* from = dy + (int64_t)n[j] * p.dy_rs + at;
          if (have == 4) rows[j] = Row4<TY>::load(from);
          else rows[j] = Row4<TY>::load_part(from, have);
        }
#pragma unroll
        for (int j = 0; j < G; ++j) {
          float f[4];
          rows[j].unpack(f);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[e] = j < live ? acc[e] + f[e] : acc[e];
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= p.scale;
      store4<false>(reinterpret_cast<TW*>(p.dw) + (int64_t)word * C + c, acc, put);
    }
  }
}

// Words that cross chunks: the workgroups of the chunk where one begins add its
// partials, kLanes of them at a time for 32 groups of 8 channels, each lane's in
// order (every kLanes-th, the first lane's behind the first chunk's) and then the lanes
// in order.
constexpr int kLanes = 16;

template <typename TW>
__global__ __launch_bounds__(32 * kLanes) void embed_join_kernel(const EmbedBwdParams p) {
  __shared__ float sums[kLanes][8][33];
  const int64_t chunk = blockIdx.x, lo = chunk * p.chunk, hi = lo + p.chunk;
  const uint32_t word = p.sorted[hi - 1].x;  // the grid has no workgroup of the last chunk
  if (word == (uint32_t)p.V || p.sorted[hi].x != word) return;
  if (lo > 0 && p.sorted[lo - 1].x == word) return;  // begun in an earlier chunk
  // the last chunk whose first word it is, 64 candidates a step: near ones, then
  // ones 64 times as far apart as long as all are, and back
  const int64_t n_chunks = (p.N + p.chunk - 1) / p.chunk;
  int64_t in = chunk + 1, step = 1;
  for (bool out = true;;) {
    const int64_t k = in + step * (1 + (threadIdx.x & 63));
    const uint64_t is = __ballot(k < n_chunks && p.sorted[k < n_chunks ? k * p.chunk : 0].x == word);
    const int more = ~is ? __builtin_ctzll(~is) : 64;
    in += step * more;
    if (out && more == 64) {
      step *= 64;
    } else if (step == 1) {
      break;
    } else {
      out = false;
      step /= 64;
    }
  }
  const int col = threadIdx.x & 31, lane = threadIdx.x >> 5;
  const int c = 8 * (int)(blockIdx.y * 32 + col), C = p.C;
  float acc[8] = {};
  if (c < C) {
    if (lane == 0) load_row8(p.tail + chunk * C, c, C, acc);
#pragma unroll 4
    for (int64_t k = chunk + 1 + lane; k <= in; k += kLanes) {
      float f[8];
      load_row8(p.head + k * C, c, C, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += f[e];
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) sums[lane][e][col] = acc[e];
  __syncthreads();
  if (lane != 0 || c >= C) return;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    float x = acc[e];
    for (int l = 1; l < kLanes; ++l) x += sums[l][e][col];
    acc[e] = x * p.scale;
  }
  store_row8(reinterpret_cast<TW*>(p.dw) + (int64_t)word * C, c, C, acc);
}

template <typename TW, typename TY>
void sum(const EmbedBwdParams& p, hipStream_t s) {
  const dim3 grid((p.units + 3) / 4), wg(256);
  if (p.C % 4 == 0) hipLaunchKernelGGL((embed_sum_kernel<TW, TY, true>), grid, wg, 0, s, p);
  else hipLaunchKernelGGL((embed_sum_kernel<TW, TY, false>), grid, wg, 0, s, p);
}
template <typename TW, typename TY>
void few(const EmbedBwdParams& p, hipStream_t s) {
  hipLaunchKernelGGL((embed_few_kernel<TW, TY>), dim3((unsigned)p.n_clear), dim3(kFewThreads), 0, s, p);
}
template <typename TW, typename TY>
void few_or_sum(const EmbedBwdParams& p, hipStream_t s) {
  if (p.N <= kEmbedFew) few<TW, TY>(p, s);
  else sum<TW, TY>(p, s);
}
// bf16 and fp16 do not meet (the C entry refuses them).
template <typename TW>
void few_or_sum(const EmbedBwdParams& p, int dtype, hipStream_t s) {
  if constexpr (sizeof(TW) == 4) {
    if (dtype == kF32) few_or_sum<float, float>(p, s);
    else if (dtype == kBF16) few_or_sum<float, __bf16>(p, s);
    else few_or_sum<float, _Float16>(p, s);
  } else {
    if (dtype == kF32) few_or_sum<TW, float>(p, s);
    else few_or_sum<TW, TW>(p, s);
  }
}

template <typename TW>
hipError_t bwd_t(const EmbedBwdParams& p, int dtype, hipStream_t s) {
  const dim3 sort_wg(kSortThreads);
  if (p.N <= kEmbedFew) {
    few_or_sum<TW>(p, dtype, s);
    return hipGetLastError();
  }
  if (p.N <= kEmbedOnce) {
    hipLaunchKernelGGL(embed_sort_kernel, dim3((unsigned)(1 + p.n_clear)), sort_wg, 0, s, p);
  } else {
    // an equal part of the zeros beside each of the launches; the pass that comes
    // last writes `sorted`
    const int launches = (p.counts ? 2 : 1) * p.passes;
    const int64_t step = (p.dw_bytes / launches + 15) / 16 * 16;
    const uint2* from = nullptr;
    for (int i = 0; i < launches; ++i) {
      const int64_t lo = i * step < p.dw_bytes ? i * step : p.dw_bytes;
      const int64_t hi = i + 1 < launches && lo + step < p.dw_bytes ? lo + step : p.dw_bytes;
      const dim3 grid((unsigned)(p.n_tiles + (lo < hi ? p.n_clear : 0)));
      const int pass = p.counts ? i / 2 : i;
      if (p.counts && i % 2 == 0) {
        hipLaunchKernelGGL(embed_count_kernel, grid, sort_wg, 0, s, p, from, pass * p.bits, lo, hi);
        if (p.n_tiles > kEmbedScanned) hipLaunchKernelGGL(embed_scan_kernel, dim3(kBins / 64), sort_wg, 0, s, p);
        continue;
      }
      uint2* to = (p.passes - 1 - pass) & 1 ? p.sorted2 : p.sorted;
      hipLaunchKernelGGL(embed_place_kernel, grid, sort_wg, 0, s, p, from, to, pass * p.bits, lo, hi);
      from = to;
    }
  }
  few_or_sum<TW>(p, dtype, s);
  const int64_t n_chunks = (p.N + p.chunk - 1) / p.chunk;
  if (n_chunks > 1)
    hipLaunchKernelGGL((embed_join_kernel<TW>), dim3((unsigned)(n_chunks - 1), (unsigned)((p.C + 255) / 256)), dim3(32 * kLanes),
                       0, s, p);
  return hipGetLastError();
}

template <typename TW, typename TY, bool WHOLE>
hipError_t fwd_tt(const EmbedParams& p, hipStream_t s) {
  if (p.units < kWideUnits)
    hipLaunchKernelGGL((embed_fwd_kernel<TW, TY, 1, WHOLE>), dim3((p.units + 255) / 256), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((embed_fwd_kernel<TW, TY, 2, WHOLE>), dim3((p.units + 511) / 512), dim3(256), 0, s, p);
  return hipGetLastError();
}
template <typename TW, typename TY>
hipError_t fwd_tt(const EmbedParams& p, hipStream_t s) {
  return p.C % 8 == 0 ? fwd_tt<TW, TY, true>(p, s) : fwd_tt<TW, TY, false>(p, s);
}
template <typename TW>
hipError_t fwd_t(const EmbedParams& p, int dtype, hipStream_t s) {
  if constexpr (sizeof(TW) == 4) {
    if (dtype == kF32) return fwd_tt<float, float>(p, s);
    return dtype == kBF16 ? fwd_tt<float, __bf16>(p, s) : fwd_tt<float, _Float16>(p, s);
  } else {
    return dtype == kF32 ? fwd_tt<TW, float>(p, s) : fwd_tt<TW, TW>(p, s);
  }
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
