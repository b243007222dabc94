// Log probabilities of given tokens with the entropy and the top alternatives
// of each row of logits, and their gradient (gfx950).
//
// With x = scale * logits, m its maximum, and exponents in base 2
// (x' = x log2 e, M = m log2 e):
//   S = sum 2^(x' - M),  logp = x_t - m - ln 2 log2 S
//   H = ln 2 (log2 S - sum 2^(x' - M) (x' - M) / S)
// in one pass over the row: each thread keeps its own running maximum and
// sums, corrected when the maximum moves, and the block merges them.  The
// bound is one read of the logits.
//
// The top k come out of the same pass.  Each thread's largest element has a
// key (value, first index of its 16-byte piece); the k-th largest of these
// thread keys, tau, is a lower bound of the k-th largest element, and only
// the k threads at or above tau own elements that can reach it.  So k / NT of
// the row is read again, the few elements at or above tau are collected, and
// each finds its rank by counting the larger ones (value, then lower index:
// a strict order, so the result does not depend on the collection's order).
//
// Few long rows are cut into segments, one workgroup each; a second kernel
// joins the segments' sums and merges their sorted top lists.
//
// Measured: 8192 x 50304 bf16 133 us replayed on one input, partly from the
// Infinity Cache, and 170 us (4.9 TB/s) behind its gradient, which takes 271 us
// (6.1 TB/s read and written); with entropy and 10 alternatives 157 us a call
// (5.3 TB/s).  511 x 50257 fp32, entropy and 20 alternatives, 31 us, 26 us from
// the cache; 4 x 151936, 5 alternatives, 10.3 us with the join.
#include "saf_kernels.h"

namespace saf {

constexpr float kLn2 = 0.6931471805599453f;
// collected elements; more (adversarial rows) take the slow selection
constexpr int cand_room(int nt) { return nt == 64 ? 256 : 1024; }

template <typename T> struct Chunk {
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
template <> struct Chunk<float> {
  static constexpr int N = 4;
  __device__ static inline void unpack(uint4 r, float (&f)[4]) {
    f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
  }
  __device__ static inline uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

// Order of the alternatives: larger value first (NaN as -inf, -0 as +0), then
// the lower position.  Larger keys come first; no element has key 0.
__device__ inline uint32_t value_key(float v) {
  v = v == v ? v + 0.f : -INFINITY;
  const uint32_t b = __float_as_uint(v);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ inline uint64_t order_key(float v, uint32_t pos) { return (uint64_t)value_key(v) << 32 | (uint32_t)~pos; }

// The value of lane ^ M, by moves inside the vector unit (an LDS shuffle takes
// several times as long, and the sorts below are chains of them).
template <int CTRL> __device__ __forceinline__ uint32_t dpp_u32(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)x, (int)x, CTRL, 0xf, 0xf, false);
}
template <int M> __device__ __forceinline__ uint32_t lane_xor(uint32_t x, int lane) {
  if constexpr (M == 1) return dpp_u32<0xb1>(x);                  // quad_perm [1, 0, 3, 2]
  if constexpr (M == 2) return dpp_u32<0x4e>(x);                  // quad_perm [2, 3, 0, 1]
  if constexpr (M == 4) return dpp_u32<0x1b>(dpp_u32<0x141>(x));  // row_half_mirror, quad_perm [3, 2, 1, 0]
  if constexpr (M == 8) return dpp_u32<0x128>(x);                 // row_ror:8
  if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return lane & 16 ? r[0] : r[1];
  }
  if constexpr (M == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return lane & 32 ? r[0] : r[1];
  }
}
template <int M> __device__ __forceinline__ uint64_t lane_xor64(uint64_t x, int lane) {
  return (uint64_t)lane_xor<M>((uint32_t)(x >> 32), lane) << 32 | lane_xor<M>((uint32_t)x, lane);
}
// One exchange of a bitonic sort: the lane keeps the larger key where want_max.
template <int M> __device__ __forceinline__ uint64_t exchange(uint64_t x, int lane, bool want_max) {
  const uint64_t y = lane_xor64<M>(x, lane);
  return (y > x) == want_max ? y : x;
}
// Descending (ascending where !down) order of bitonic runs of 2 M keys.
template <int M> __device__ __forceinline__ uint64_t merge_runs(uint64_t x, int lane, bool down) {
  x = exchange<M>(x, lane, ((lane & M) == 0) == down);
  if constexpr (M > 1) x = merge_runs<M / 2>(x, lane, down);
  return x;
}
template <int M> __device__ __forceinline__ uint64_t wave_max64_step(uint64_t x, int lane) {
  x = exchange<M>(x, lane, true);
  if constexpr (M > 1) x = wave_max64_step<M / 2>(x, lane);
  return x;
}
__device__ inline uint64_t wave_max64(uint64_t x, int lane) { return wave_max64_step<32>(x, lane); }

// Descending order of a bitonic sequence over the lanes, and of any keys.
__device__ inline uint64_t wave_merge_desc(uint64_t x, int lane) { return merge_runs<32>(x, lane, true); }
__device__ inline uint64_t wave_sort_desc(uint64_t x, int lane) {
  x = merge_runs<1>(x, lane, (lane & 2) == 0);
  x = merge_runs<2>(x, lane, (lane & 4) == 0);
  x = merge_runs<4>(x, lane, (lane & 8) == 0);
  x = merge_runs<8>(x, lane, (lane & 16) == 0);
  x = merge_runs<16>(x, lane, (lane & 32) == 0);
  return merge_runs<32>(x, lane, true);
}

// Exponents x' - M of one row or thread, M = m log2 e scale.  Below 2^24 they are
// one FMA against the rounded M: every term of a sum then carries the same offset
// m sl2 - round(m sl2), at most a half there, which delta() gives back.  Beyond
// (a thread or row that holds nothing but a mask's value, say -1e10) the offset
// would overflow 2^offset, and the difference is formed first.
struct Anchor {
  float m, ref, sl2;
  bool wide;
  // m of a row with nothing above -inf: 0, so that no inf - inf arises
  __device__ inline Anchor(float m_, float sl2_) : sl2(sl2_) {
    m = m_ == -INFINITY ? 0.f : m_;
    ref = m * sl2;
    wide = !(fabsf(ref) < 16777216.f);
  }
  __device__ inline float exponent(float x) const { return wide ? (x - m) * sl2 : fmaf(x, sl2, -ref); }
  __device__ inline float delta() const { return wide ? 0.f : fmaf(m, sl2, -ref); }
};

// Running softmax sums in base 2 relative to the anchor of m.
struct Sums {
  float m = -INFINITY, s = 0.f, t = 0.f;  // raw maximum, sum e, sum e (x' - M)
  template <bool ENT> __device__ inline void raise(float m_new, float sl2) {
    const Anchor a(m, sl2), b(m_new, sl2);
    const bool none = m == -INFINITY;
    // not a.ref - b.ref, which the compiler may form as fma(a.m, sl2, -b.ref)
    const float d = none ? 0.f : fmaxf(fmaf(a.m - b.m, sl2, b.delta() - a.delta()), -1000.f);
    const float f = none ? 0.f : fast_exp2(d);  // times 0 keeps a NaN
    if (ENT) t = f * fmaf(s, d, t);
    s *= f;
    m = m_new;
  }
  // one element that does not exceed m, with its exponent
  template <bool ENT> __device__ inline void add(float v) {
    const float e = fast_exp2(v);
    s += e;
    if (ENT) t = fmaf(e, fmaxf(v, -1000.f), t);  // e = 0 far below: no 0 * inf
  }
  template <bool ENT, int N> __device__ inline void add_all(const float (&x)[N], float sl2) {
    const Anchor a(m, sl2);
    if (a.wide) {
#pragma unroll
      for (int e = 0; e < N; ++e) add<ENT>((x[e] - a.m) * sl2);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) add<ENT>(fmaf(x[e], sl2, -a.ref));
    }
  }
};
// The sums of a whole wave: one common maximum, then plain sums.
template <bool ENT> __device__ inline void wave_merge(Sums& a, float sl2) {
  a.raise<ENT>(wave_max(a.m), sl2);
  a.s = dpp_wave_sum(a.s);
  if (ENT) a.t = dpp_wave_sum(a.t);
}

__device__ inline int64_t token_of(const LogprobParams& p, int64_t r) {
  return p.tok_i64 ? reinterpret_cast<const int64_t*>(p.tokens)[r * p.tok_st]
                   : (int64_t)reinterpret_cast<const int32_t*>(p.tokens)[r * p.tok_st];
}
template <typename T> __device__ inline float elem_f32(const T* p) {
  if constexpr (sizeof(T) == 4) return *p;
  else return Elem<T>::lo((uint32_t)*reinterpret_cast<const uint16_t*>(p));
}

// Log probability (nats) of a logit x: the difference in the logits' units,
// which does not overflow where x' - M in base 2 would.
__device__ inline float log_prob(float x, const Anchor& a, float lg, float scale) {
  return fmaf(x - a.m, scale, -kLn2 * (lg - a.delta()));
}
// One row's outputs from its sums (one thread).  A row with nothing above -inf
// has S = 0 and gets NaN.
template <typename T>
__device__ inline void write_row(const LogprobParams& p, int64_t row, const Sums& a, float sl2) {
  const Anchor c(a.m, sl2);
  const float lg = a.s > 0.f ? log2f(a.s) : __builtin_nanf("");
  if (p.stats) {
    p.stats[2 * row] = c.m;
    p.stats[2 * row + 1] = lg;
  }
  const int64_t tok = token_of(p, row);
  float lp = 0.f;
  if (tok != p.ignore) {
    lp = __builtin_nanf("");
    if (tok >= 0 && tok < p.V)
      lp = log_prob(elem_f32(reinterpret_cast<const T*>(p.logits) + row * p.x_rs + tok), c, lg, p.scale);
  }
  p.logp[row] = lp;
  if (p.entropy) p.entropy[row] = (lg - a.t / a.s) * kLn2;
}
__device__ inline void write_top(const LogprobParams& p, int64_t row, int rank, uint64_t key, const Sums& a, float sl2) {
  const int64_t at = row * p.top + rank;
  const float lg = a.s > 0.f ? log2f(a.s) : __builtin_nanf("");
  p.top_index[at] = (int64_t)(uint32_t)~(uint32_t)key;
  p.top_logp[at] = log_prob(key_value((uint32_t)(key >> 32)), Anchor(a.m, sl2), lg, p.scale);
}

template <typename T, int NT, bool TOP, bool ENT>
__global__ __launch_bounds__(NT) void logprob_kernel(const LogprobParams p) {
  using C = Chunk<T>;
  constexpr int N = C::N, W = NT / 64, U = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / (unsigned)p.n_seg;
  const int seg = blockIdx.x - (int)row * p.n_seg;
  const int v0 = seg * p.seg_len, n = min(p.seg_len, p.V - v0);
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.x_rs + v0;
  const float sl2 = p.scale * kLog2e;
  // 16-byte pieces from the first aligned element on; the elements before and
  // after them one by one (thread i the i-th)
  const int head = min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
  const int nv = (n - head) / N, tail0 = head + nv * N;
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);

  Sums a;
  uint32_t best = 0xffffffffu;  // position (within the segment) of the piece that holds a.m
  auto single = [&](int i) {
    const float f = elem_f32(x + i);
    if (TOP && best == 0xffffffffu) best = i;
    if (f > a.m) {
      a.raise<ENT>(f, sl2);
      if (TOP) best = i;
    }
    a.add<ENT>(Anchor(a.m, sl2).exponent(f));
  };
  if (tid < head) single(tid);
  // groups of U pieces per thread, the next group's loads in flight while one is
  // summed; pieces past the end are -inf (no weight, never a new maximum)
  auto load = [&](uint4 (&r)[U], int k) {
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = xv[min(k + u * NT, nv - 1)];
  };
  auto sum = [&](const uint4 (&r)[U], int k) {
    float f[U][N], cm[U], gm = -INFINITY;
    const bool whole = k - tid + U * NT <= nv;  // the whole block's group
#pragma unroll
    for (int u = 0; u < U; ++u) {
      cm[u] = -INFINITY;
      if (k - tid + u * NT >= nv) break;  // nothing left for any thread
      C::unpack(r[u], f[u]);
      if (!whole && k + u * NT >= nv) {
#pragma unroll
        for (int e = 0; e < N; ++e) f[u][e] = -INFINITY;
      }
      cm[u] = f[u][0];
#pragma unroll
      for (int e = 1; e < N; ++e) cm[u] = fmaxf(cm[u], f[u][e]);
      gm = fmaxf(gm, cm[u]);
    }
    if (TOP && best == 0xffffffffu && k < nv) best = head + k * N;
    if (gm > a.m) {
      a.raise<ENT>(gm, sl2);
      if (TOP) {
#pragma unroll
        for (int u = U - 1; u >= 0; --u)
          if (cm[u] == gm) best = head + (k + u * NT) * N;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (k - tid + u * NT < nv) a.add_all<ENT>(f[u], sl2);
  };
  if (nv > 0) {
    uint4 ra[U], rb[U];
    load(ra, tid);
    for (int k = tid;;) {
      load(rb, k + U * NT);
      sum(ra, k);
      k += U * NT;
      if (k - tid >= nv) break;
      load(ra, k + U * NT);
      sum(rb, k);
      k += U * NT;
      if (k - tid >= nv) break;
    }
  }
  if (tail0 + tid < n) single(tail0 + tid);
  const uint64_t mykey = TOP && best != 0xffffffffu ? order_key(a.m, best) : 0;

  // the block's sums (with TOP in every thread)
  __shared__ float sm_a[W][3];
  wave_merge<ENT>(a, sl2);
  if constexpr (W > 1) {
    if (lane == 0) {
      sm_a[wave][0] = a.m;
      sm_a[wave][1] = a.s;
      sm_a[wave][2] = a.t;
    }
    __syncthreads();
    if (!TOP && wave != 0) return;
    a = Sums{};
    if (lane < W) a = Sums{sm_a[lane][0], sm_a[lane][1], sm_a[lane][2]};
    wave_merge<ENT>(a, sl2);
  }
  const int64_t part = row * p.n_seg + seg;
  if (tid == 0) {
    if (p.n_seg > 1) {
      p.part[4 * part] = a.m;
      p.part[4 * part + 1] = a.s;
      p.part[4 * part + 2] = a.t;
    } else {
      write_row<T>(p, row, a, sl2);
    }
  }
  if constexpr (!TOP) return;

  constexpr int kCand = cand_room(NT);
  __shared__ uint64_t sm_cand[kCand];
  __shared__ int sm_win[32];
  __shared__ int sm_nwin, sm_ncand;
  const int K = p.top;
  if (tid == 0) sm_nwin = sm_ncand = 0;
  // tau, the K-th largest thread key (0: fewer than K threads hold elements)
  uint64_t keys = wave_sort_desc(mykey, lane);
  if constexpr (W > 1) {
    __shared__ uint64_t sm_key[W][32];
    __shared__ uint64_t sm_tau;
    if (lane < 32) sm_key[wave][lane] = keys;
    __syncthreads();
    if (wave == 0) {
      // the waves' lists one after the other behind the largest 32 so far, in
      // reverse: a bitonic sequence
      for (int w = 1; w < W; ++w) {
        if (lane >= 32) keys = sm_key[w][63 - lane];
        keys = wave_merge_desc(keys, lane);
      }
      if (lane == K - 1) sm_tau = keys;
    }
    __syncthreads();
    keys = sm_tau;
  } else {
    __syncthreads();
    keys = (uint64_t)__shfl((uint32_t)(keys >> 32), K - 1, 64) << 32 | __shfl((uint32_t)keys, K - 1, 64);
  }
  const uint64_t tau = keys;
  const bool win = mykey != 0 && mykey >= tau;
  // with tau = 0 (short segments) every element is collected below
  if (win && tau != 0) sm_win[atomicAdd(&sm_nwin, 1)] = tid;
  __syncthreads();
  auto collect = [&](float f, uint32_t piece, uint32_t i) {
    if (order_key(f, piece) >= tau) {
      const int at = atomicAdd(&sm_ncand, 1);
      if (at < kCand) sm_cand[at] = order_key(f, v0 + i);
    }
  };
  if (tid < head) collect(elem_f32(x + tid), tid, tid);
  if (tail0 + tid < n) collect(elem_f32(x + tail0 + tid), tail0 + tid, tail0 + tid);
  {
    const int per = (nv + NT - 1) / NT;  // pieces of one thread
    const int total = tau != 0 ? sm_nwin * per : nv;
    for (int w = tid; w < total; w += NT) {
      const int kk = tau != 0 ? sm_win[w / per] + (w % per) * NT : w;
      if (kk < nv) {
        float f[N];
        C::unpack(xv[kk], f);
#pragma unroll
        for (int e = 0; e < N; ++e) collect(f[e], head + kk * N, head + kk * N + e);
      }
    }
  }
  __syncthreads();
  const int nc = sm_ncand;
  auto put = [&](int rank, uint64_t key) {
    if (p.n_seg > 1) p.part_top[part * K + rank] = key;
    else write_top(p, row, rank, key, a, sl2);
  };
  if (nc <= kCand) {
    for (int i = tid; i < nc; i += NT) {
      const uint64_t mine = sm_cand[i];
      int rank = 0;
      for (int j = 0; j < nc; ++j) rank += sm_cand[j] > mine;
      if (rank < K) put(rank, mine);
    }
    // a segment shorter than K
    for (int i = nc + tid; i < K; i += NT)
      if (p.n_seg > 1) p.part_top[part * K + i] = 0;
  } else {
    // too many: the next largest key below the last one, K times over the row
    uint64_t last = ~(uint64_t)0;
    for (int i = 0; i < K; ++i) {
      uint64_t bk = 0;
      for (int j = tid; j < n; j += NT) {
        const uint64_t key = order_key(elem_f32(x + j), v0 + j);
        if (key < last && key > bk) bk = key;
      }
      bk = wave_max64(bk, lane);
      __syncthreads();
      if (lane == 0) sm_cand[wave] = bk;
      __syncthreads();
      for (int w = 0; w < W; ++w) bk = sm_cand[w] > bk ? sm_cand[w] : bk;
      last = bk;
      if (tid == 0) put(i, bk);
    }
  }
}

// Join of a row's segments: one wave per row, lane s the segment s.
template <typename T, bool ENT>
__global__ __launch_bounds__(64) void logprob_join_kernel(const LogprobParams p) {
  const int lane = threadIdx.x;
  const int64_t row = blockIdx.x;
  const float sl2 = p.scale * kLog2e;
  const int64_t part = row * p.n_seg + lane;
  Sums a;
  if (lane < p.n_seg) {
    a.m = p.part[4 * part];
    a.s = p.part[4 * part + 1];
    a.t = p.part[4 * part + 2];
  }
  wave_merge<ENT>(a, sl2);
  if (lane == 0) write_row<T>(p, row, a, sl2);
  int at = 0;
  uint64_t head = p.top > 0 && lane < p.n_seg ? p.part_top[part * p.top] : 0;
  for (int i = 0; i < p.top; ++i) {
    const uint64_t best = wave_max64(head, lane);
    if (head == best && best != 0) {
      write_top(p, row, i, best, a, sl2);
      ++at;
      head = at < p.top ? p.part_top[part * p.top + at] : 0;
    }
  }
}

// Gradient: each workgroup a run of kBwdPieces pieces per thread of one row.
constexpr int kBwdPieces = 4;
template <typename T, bool ENT>
__global__ __launch_bounds__(256) void logprob_bwd_kernel(const LogprobBwdParams p) {
  using C = Chunk<T>;
  constexpr int N = C::N, RUN = 256 * N * kBwdPieces;
  const int n_run = (p.V + RUN - 1) / RUN;
  const int64_t row = blockIdx.x / (unsigned)n_run;
  const int v0 = (int)(blockIdx.x - (unsigned)row * n_run) * RUN, n = min(RUN, p.V - v0);
  const T* x = reinterpret_cast<const T*>(p.logits) + row * p.x_rs + v0;
  T* dx = reinterpret_cast<T*>(p.dx) + row * p.d_rs + v0;
  const float sl2 = p.scale * kLog2e;
  const Anchor c(p.stats[2 * row], sl2);
  const float lg = p.stats[2 * row + 1];
  const int64_t tok64 = p.tok_i64 ? reinterpret_cast<const int64_t*>(p.tokens)[row * p.tok_st]
                                  : (int64_t)reinterpret_cast<const int32_t*>(p.tokens)[row * p.tok_st];
  const bool skip = tok64 == p.ignore;
  const bool inside = tok64 >= 0 && tok64 < p.V;
  const int tok = skip || !inside ? -1 : (int)tok64 - v0;
  float g = skip ? 0.f : (inside ? p.dlogp[row * p.g_st] : __builtin_nanf(""));
  float ge = 0.f, H = 0.f;
  if (ENT) {
    ge = p.dent[row * p.ge_st];
    H = p.entropy[row];
  }
  // a row that takes no part has a zero gradient whatever it holds
  const bool zero = skip && (!ENT || ge == 0.f);
  auto grad = [&](float f, int i) {
    if (zero) return 0.f;
    const float v = c.exponent(f) - lg, q = fast_exp2(v);
    float d = -g * q;
    if (ENT) d = fmaf(-ge * q, fmaf(fmaxf(v, -1000.f), kLn2, H), d);
    if (i == tok) d += g;
    return d * p.scale;
  };
  // pieces where logits and gradient rows have the same alignment, else one by one
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
  const int head = same ? min(n, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T)) : n;
  const int nv = (n - head) / N, tail0 = head + nv * N;
  auto put = [&](int i) {
    const float d = grad(elem_f32(x + i), i);
    if constexpr (sizeof(T) == 4) dx[i] = d;
    else *reinterpret_cast<uint16_t*>(dx + i) = (uint16_t)Elem<T>::pack2(d, 0.f);
  };
  for (int i = threadIdx.x; i < head; i += 256) put(i);
  const uint4* xv = reinterpret_cast<const uint4*>(x + head);
  uint4* dv = reinterpret_cast<uint4*>(dx + head);
  uint4 r[kBwdPieces];
#pragma unroll
  for (int u = 0; u < kBwdPieces; ++u)
    if ((int)threadIdx.x + 256 * u < nv) r[u] = xv[threadIdx.x + 256 * u];
#pragma unroll
  for (int u = 0; u < kBwdPieces; ++u) {
    const int k = threadIdx.x + 256 * u;
    if (k < nv) {
      float f[N];
      C::unpack(r[u], f);
#pragma unroll
      for (int e = 0; e < N; ++e) f[e] = grad(f[e], head + k * N + e);
      dv[k] = C::pack(f);
    }
  }
  if (tail0 + (int)threadIdx.x < n) put(tail0 + threadIdx.x);
}

template <typename T, int NT>
static hipError_t launch_logprob_nt(const LogprobParams& p, hipStream_t s) {
  const dim3 grid((unsigned)(p.R * p.n_seg));
  if (p.top > 0) {
    if (p.entropy) hipLaunchKernelGGL((logprob_kernel<T, NT, true, true>), grid, dim3(NT), 0, s, p);
    else hipLaunchKernelGGL((logprob_kernel<T, NT, true, false>), grid, dim3(NT), 0, s, p);
  } else {
    if (p.entropy) hipLaunchKernelGGL((logprob_kernel<T, NT, false, true>), grid, dim3(NT), 0, s, p);
    else hipLaunchKernelGGL((logprob_kernel<T, NT, false, false>), grid, dim3(NT), 0, s, p);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.n_seg == 1) return e;
  if (p.entropy) hipLaunchKernelGGL((logprob_join_kernel<T, true>), dim3((unsigned)p.R), dim3(64), 0, s, p);
  else hipLaunchKernelGGL((logprob_join_kernel<T, false>), dim3((unsigned)p.R), dim3(64), 0, s, p);
  return hipGetLastError();
}

// Threads per row (or segment): one wave where a row is at most eight pieces per
// lane (4096 rows of 4000, top 10: 12 us against 21 with 256 threads, whose
// barriers cost more than the row); 512 for long rows without alternatives (8192
// rows of 50304: 130 us against 137 with 256, 6.3 TB/s) and where a row has a CU
// to itself (200 rows of 151936, top 5: 18 us against 22); else 256 (8192 rows of
// 50304, top 10: 158 us against 209 with 512, whose sorts and barriers leave the
// CU idle; with one wave the second look at the top threads' pieces is a long
// chain, 243).
template <typename T> static hipError_t launch_logprob_t(const LogprobParams& p, hipStream_t s) {
  const int pieces = p.seg_len / Chunk<T>::N;
  if (pieces <= 512) return launch_logprob_nt<T, 64>(p, s);
  if (pieces >= 4096 && (p.top == 0 || p.R * p.n_seg <= p.n_cu)) return launch_logprob_nt<T, 512>(p, s);
  return launch_logprob_nt<T, 256>(p, s);
}

hipError_t launch_token_logprobs(const LogprobParams& p, int dtype, hipStream_t s) {
  if (dtype == kBF16) return launch_logprob_t<__bf16>(p, s);
  if (dtype == kF16) return launch_logprob_t<_Float16>(p, s);
  if (dtype == kF32) return launch_logprob_t<float>(p, s);
  return hipErrorInvalidValue;
}

template <typename T> static hipError_t launch_bwd_t(const LogprobBwdParams& p, hipStream_t s) {
  constexpr int RUN = 256 * Chunk<T>::N * kBwdPieces;
  const dim3 grid((unsigned)(p.R * ((p.V + RUN - 1) / RUN)));
  if (p.dent) hipLaunchKernelGGL((logprob_bwd_kernel<T, true>), grid, dim3(256), 0, s, p);
  else hipLaunchKernelGGL((logprob_bwd_kernel<T, false>), grid, dim3(256), 0, s, p);
  return hipGetLastError();
}

hipError_t launch_token_logprobs_bwd(const LogprobBwdParams& p, int dtype, hipStream_t s) {
  if (dtype == kBF16) return launch_bwd_t<__bf16>(p, s);
  if (dtype == kF16) return launch_bwd_t<_Float16>(p, s);
  if (dtype == kF32) return launch_bwd_t<float>(p, s);
  return hipErrorInvalidValue;
}

}  // namespace saf
