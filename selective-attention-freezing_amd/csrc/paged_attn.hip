// Attention of one new token per sequence over a paged key / value cache
// (gfx950): live, dense-frozen and decomposed-frozen heads in one launch.
//
// For sequence b with n cached tokens (the new one, i = n - 1, included):
//   live         o = sum_j softmax_j(q . k_j scale) v_j
//   dense        o = sum_j patt[i, j] v_j
//   decomposed   o = sum_j exp(alpha_j + rho_{i-j} - z_i) v_j
// Every key and value is read once and used for at most a handful of queries,
// so the bound is HBM: the layout serves wide loads in flight, and the matrix
// pipe (which a single query column leaves almost idle) does the arithmetic
// without LDS traffic.
//
// Unit: the query heads (columns, at most 16) that share one K and one V
// head: a KV group with kvidx, a single head without.  A wave takes steps of
// 32 keys:
//   S^T[key][col] = K . Q^T      (A = K rows straight from memory)
//   O^T[d][col]  += V^T . P^T    (B = P in the registers that S^T left it in)
// with 16x16 MFMA tiles: lane (c = l % 16, g = l / 16) of an S^T tile holds
// column c, keys 4g..4g+3, and with the key order {4g + r, 16 + 4g + r} the
// eight weights of a lane over the step's two tiles are its B operand of the
// P.V product as they stand.  The A operand of P.V needs eight keys of one d
// per lane: lane (c, g) loads E consecutive d of the eight keys of its group
// and transposes them in registers (one v_perm_b32 per two elements), with
// output row 4g + r of tile e standing for d = E (4g + r) + e.
//
// P is rounded to 16 bits for the product as two terms, P = hi + lo, so the
// rounding of the result is the output's own; fp16 weights are scaled by 2^8
// first (their small ones would be subnormal: weights above 255 overflow).
//
// Measured: 128 ragged sequences of up to 8192 keys, 8 KV heads of 128, 2.3 GB:
// 423 us, 5.5 TB/s; one sequence of 65537 keys, fp16 at hd 128: 90 us with the
// join, 5.2 TB/s; 64 ragged sequences of up to 4096 keys, 12 heads of 64: 80 us,
// 4.7 TB/s; one sequence of 1024 keys: 9.1 us.  (Graph replays on one input;
// the Infinity Cache serves the last one and a part of the two before it.)
#include "saf_kernels.h"

namespace saf {

typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3_a4_t __attribute__((ext_vector_type(3), aligned(4)));

__device__ inline f32x4_t zero4() { return f32x4_t{0.f, 0.f, 0.f, 0.f}; }

// Maximum / sum over the four lanes c, c + 16, c + 32, c + 48.
__device__ inline float column_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_swap_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}
__device__ inline float column_sum(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return half_swap_sum(__uint_as_float(r[0]) + __uint_as_float(r[1]));
}

// Inclusive sum over the lanes up to this one (GFX9 DPP moves; every lane
// active): shifts inside 16-lane rows, then lane 15 of rows 0 and 2 and lane 31
// into the rows behind them.
template <int CTRL, int ROWMASK> __device__ __forceinline__ int dpp_add_i32(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWMASK, 0xf, false);
}
__device__ inline int wave_scan(int x) {
  x = dpp_add_i32<0x111, 0xf>(x);  // row_shr:1
  x = dpp_add_i32<0x112, 0xf>(x);  // row_shr:2
  x = dpp_add_i32<0x114, 0xf>(x);  // row_shr:4
  x = dpp_add_i32<0x118, 0xf>(x);  // row_shr:8
  x = dpp_add_i32<0x142, 0xa>(x);  // row_bcast:15, rows 1 and 3
  return dpp_add_i32<0x143, 0xc>(x);  // row_bcast:31, rows 2 and 3
}

__device__ inline f32x4_t mfma16(__bf16, uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}
__device__ inline f32x4_t mfma16(_Float16, uint4 a, uint4 b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0,
                                                0);
}

// One step's K and V in registers and its products, 16-bit storage.
template <typename T, int HD> struct PagedTile {
  static constexpr int E = HD <= 128 ? HD / 16 : 8;  // consecutive d per lane
  static constexpr int NBLK = HD / (16 * E);
  static constexpr int KS = HD / 32;
  static constexpr float kShift = Elem<T>::is_bf16 ? 0.f : 8.f;  // log2 of the scale of P
  typedef uint4 Query[KS];
  uint4 k[2][KS];
  uint32_t v[NBLK][2][4][E / 2];

  __device__ static inline void load_q(Query& q, const T* row, bool live, int g) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      q[ks] = live ? *reinterpret_cast<const uint4*>(row + 32 * ks + 8 * g) : make_uint4(0, 0, 0, 0);
  }
  // byte offsets of a lane within a row
  __device__ static inline uint32_t k_lane(int g) { return 16 * g; }
  __device__ static inline uint32_t v_lane(int c) { return 2 * E * c; }
  __device__ inline void load_k(const char* page, uint32_t off, int t) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k[t][ks] = *reinterpret_cast<const uint4*>(page + off + 64 * ks);
  }
  __device__ inline void load_v(const char* page, uint32_t off, int t, int r) {
#pragma unroll
    for (int b = 0; b < NBLK; ++b) {
      const char* p = page + off + 32 * E * b;
      uint32_t(&w)[E / 2] = v[b][t][r];
      if constexpr (E == 2) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
      } else if constexpr (E == 4) {
        const u32x2_t x = *reinterpret_cast<const u32x2_t*>(p);
        w[0] = x[0]; w[1] = x[1];
      } else if constexpr (E == 6) {
        const u32x3_a4_t x = *reinterpret_cast<const u32x3_a4_t*>(p);
        w[0] = x[0]; w[1] = x[1]; w[2] = x[2];
      } else {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
      }
    }
  }
  __device__ inline f32x4_t scores(const Query& q, int t) const {
    f32x4_t s = zero4();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) s = mfma16(T{}, k[t][ks], q[ks], s);
    return s;
  }
  __device__ inline void pv(f32x4_t (&o)[NBLK][E], const float (&p)[2][4]) const {
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float a = p[t][2 * h], b = p[t][2 * h + 1];
        const uint32_t w = Elem<T>::pack2(a, b);
        hi[2 * t + h] = w;
        lo[2 * t + h] = Elem<T>::pack2(a - Elem<T>::lo(w), b - Elem<T>::hi(w));
      }
    const uint4 ph = make_uint4(hi[0], hi[1], hi[2], hi[3]), pl = make_uint4(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
    for (int b = 0; b < NBLK; ++b)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
        uint32_t a[4];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            a[2 * t + h] = __builtin_amdgcn_perm(v[b][t][2 * h + 1][e / 2], v[b][t][2 * h][e / 2], sel);
        const uint4 av = make_uint4(a[0], a[1], a[2], a[3]);
        o[b][e] = mfma16(T{}, av, ph, o[b][e]);
        o[b][e] = mfma16(T{}, av, pl, o[b][e]);
      }
  }
};

// float32: v_mfma_f32_16x16x4_f32 (one key or d per lane and operand), the
// same tiles with K's 16 d of a slice in the order 4g + e and P.V one key per
// lane group and product.
template <int HD> struct PagedTile<float, HD> {
  static constexpr int E = HD % 64 == 0 ? 4 : 2;
  static constexpr int NBLK = HD / (16 * E);
  static constexpr int KS = HD / 16;
  static constexpr float kShift = 0.f;
  typedef float4 Query[KS];
  float4 k[2][KS];
  float v[NBLK][2][4][E];

  __device__ static inline void load_q(Query& q, const float* row, bool live, int g) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
      q[ks] = live ? *reinterpret_cast<const float4*>(row + 16 * ks + 4 * g) : make_float4(0.f, 0.f, 0.f, 0.f);
  }
  __device__ static inline uint32_t k_lane(int g) { return 16 * g; }
  __device__ static inline uint32_t v_lane(int c) { return 4 * E * c; }
  __device__ inline void load_k(const char* page, uint32_t off, int t) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) k[t][ks] = *reinterpret_cast<const float4*>(page + off + 64 * ks);
  }
  __device__ inline void load_v(const char* page, uint32_t off, int t, int r) {
#pragma unroll
    for (int b = 0; b < NBLK; ++b) {
      const char* p = page + off + 64 * E * b;
      if constexpr (E == 4) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[b][t][r][0] = x.x; v[b][t][r][1] = x.y; v[b][t][r][2] = x.z; v[b][t][r][3] = x.w;
      } else {
        const float2 x = *reinterpret_cast<const float2*>(p);
        v[b][t][r][0] = x.x; v[b][t][r][1] = x.y;
      }
    }
  }
  __device__ inline f32x4_t scores(const Query& q, int t) const {
    f32x4_t s = zero4();
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][ks].x, q[ks].x, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][ks].y, q[ks].y, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][ks].z, q[ks].z, s, 0, 0, 0);
      s = __builtin_amdgcn_mfma_f32_16x16x4f32(k[t][ks].w, q[ks].w, s, 0, 0, 0);
    }
    return s;
  }
  __device__ inline void pv(f32x4_t (&o)[NBLK][E], const float (&p)[2][4]) const {
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int b = 0; b < NBLK; ++b)
#pragma unroll
          for (int e = 0; e < E; ++e)
            o[b][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[b][t][r][e], p[t][r], o[b][e], 0, 0, 0);
  }
};

template <typename T> __device__ inline void store4(T* p, float4 x) {
  *reinterpret_cast<uint2*>(p) = make_uint2(Elem<T>::pack2(x.x, x.y), Elem<T>::pack2(x.z, x.w));
}
template <> __device__ inline void store4<float>(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }

template <typename T> __device__ inline float4 load4(const T* p) {
  const uint2 w = *reinterpret_cast<const uint2*>(p);
  return make_float4(Elem<T>::lo(w.x), Elem<T>::hi(w.x), Elem<T>::lo(w.y), Elem<T>::hi(w.y));
}
template <> __device__ inline float4 load4<float>(const float* p) { return *reinterpret_cast<const float4*>(p); }

constexpr int kOPad = 4;  // floats after each column's HD partial sums

// What one wave keeps of its unit while it walks the keys.
template <typename T, int HD> struct PagedWave {
  using Tile = PagedTile<T, HD>;
  static constexpr int E = Tile::E, NBLK = Tile::NBLK;
  typename Tile::Query q;
  f32x4_t o[NBLK][E];
  float m, l;
  bool bad;
};

// exp(alpha + rho - z).  Where the weight matters z is close to the sum and their
// difference exact: the sum's own rounding (TwoSum) is all that large logits lose.
__device__ inline float decomposed_weight(float a, float d, float z) {
  const float sum = a + d, back = sum - a;
  const float lost = sum == -INFINITY ? 0.f : (a - (sum - back)) + (d - back);
  return fast_exp2(((sum - z) + lost) * kLog2e);
}

// Weights of the frozen columns for the keys kb0..kb1-1, into w[f][key - kb0]
// (f = column - nl), before the walk: the waves take runs of 256 keys of one
// column in turn, four keys per lane, whose loads are in flight together.
// Whole steps are written: weight 0 behind the last key.
__device__ inline void frozen_weights(const PagedAttnParams& p, float* w, int pitch, int c0, int nl, int nc, int n, int kb0,
                                      int kb1, int wave, int W, int lane, float scale) {
  const int F = nc - nl, end = kb0 + ((kb1 - kb0 + 31) & ~31);
  const int items = F * ((kb1 - kb0 + 255) >> 8);
  for (int item = wave; item < items; item += W) {
    const int run = item / F, f = item - run * F;
    const int64_t word = p.col[c0 + nl + f];
    const int state = col_state(word), row = col_pat(word);
    const bool fits = n <= (state == 1 ? p.p_S : p.d_S);  // else the row is NaN
    const int key0 = kb0 + 256 * run + lane;
    float x[4];
    if (!fits) {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = __builtin_nanf("");
    } else if (state == 1) {
      uint32_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k)
        v[k] = load_bits(p.patt, row * p.p_sh + (n - 1) * p.p_si + min(key0 + 64 * k, kb1 - 1) * p.p_sj, p.patt_dtype);
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = bits_to_f32(v[k], p.patt_dtype) * scale;
    } else {
      uint32_t a[4], d[4];
      const uint32_t z = load_bits(p.z, row * p.z_sh + (n - 1) * p.z_ss, p.z_dtype);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int key = min(key0 + 64 * k, kb1 - 1);
        a[k] = load_bits(p.alpha, row * p.a_sh + key * p.a_ss, p.a_dtype);
        d[k] = load_bits(p.rho, row * p.r_sh + (n - 1 - key) * p.r_ss, p.r_dtype);
      }
      const float zf = bits_to_f32(z, p.z_dtype);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        x[k] = decomposed_weight(bits_to_f32(a[k], p.a_dtype), bits_to_f32(d[k], p.r_dtype), zf) * scale;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int key = key0 + 64 * k;
      if (key < end) w[f * pitch + key - kb0] = key < kb1 ? x[k] : 0.f;
    }
  }
}

// The keys kb0..kb1-1 of one workgroup, steps of 32 dealt to its waves in
// turn.  LIVE: the unit has live columns (K is read); FROZEN: it has frozen
// ones (weights in w, kb0-based).
template <typename T, int HD, bool LIVE, bool FROZEN>
__device__ inline void walk(const PagedAttnParams& p, PagedWave<T, HD>& st, const char* kc, const char* vc,
                            const int32_t* table, float* w, int pitch, int c0, int nl, int nc, int n, int kb0, int kb1,
                            int wave, int W, int lane) {
  using Tile = PagedTile<T, HD>;
  constexpr int E = Tile::E, NBLK = Tile::NBLK;
  const int c = lane & 15, g = lane >> 4;
  const bool live_col = c < nl;
  const int page_mask = (1 << p.page_shift) - 1;
  const uint32_t k_row = (uint32_t)p.k_st * sizeof(T), v_row = (uint32_t)p.v_st * sizeof(T);
  const uint32_t k_lane = Tile::k_lane(g), v_lane = Tile::v_lane(c);
  const uint32_t k_full = c * k_row + k_lane, v_full = 4 * g * v_row + v_lane;
  const int64_t k_page = p.k_sp * (int64_t)sizeof(T), v_page = p.v_sp * (int64_t)sizeof(T);
  const int n_it = kb1 - kb0 > 32 * wave ? (kb1 - kb0 - 32 * wave + 32 * W - 1) / (32 * W) : 0;

  // page ids of the wave's next 32 steps, two 16-key tiles each (a page holds
  // whole tiles), in one load; a step whose second tile lies past the end uses
  // its first tile's page and rows twice, with weight 0
  int ids = 0;
  auto load = [&](Tile& tile, int it) {
    const int key0 = kb0 + 32 * (wave + it * W);
    if ((it & 31) == 0) {
      const int kk = key0 + 32 * W * (lane >> 1);
      ids = 0;
      if (kk < kb1) {
        const int kt = (lane & 1) && kk + 16 < kb1 ? kk + 16 : kk;
        ids = table[kt >> p.page_shift];
        if (ids < 0 || ids >= p.n_pages) {
          st.bad = true;
          ids = 0;
        }
      }
    }
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int page = __builtin_amdgcn_readlane(ids, 2 * (it & 31) + t);
      const int kt = t && key0 + 16 < kb1 ? key0 + 16 : key0;
      const int row0 = kt & page_mask, last = min(16, kb1 - kt) - 1;
      uint32_t k_off = k_full, v_off[4] = {v_full, v_full + v_row, v_full + 2 * v_row, v_full + 3 * v_row};
      if (last < 15) {  // rows past the end repeat the last one
        k_off = min(c, last) * k_row + k_lane;
#pragma unroll
        for (int r = 0; r < 4; ++r) v_off[r] = min(4 * g + r, last) * v_row + v_lane;
      }
      if (LIVE) tile.load_k(kc + page * k_page + row0 * k_row, k_off, t);
      const char* vp = vc + page * v_page + row0 * v_row;
#pragma unroll
      for (int r = 0; r < 4; ++r) tile.load_v(vp, v_off[r], t, r);
    }
  };
  auto compute = [&](const Tile& tile, int it) {
    const int key0 = kb0 + 32 * (wave + it * W);
    float x[2][4];
    if (LIVE) {
      f32x4_t sc[2];
#pragma unroll
      for (int t = 0; t < 2; ++t) sc[t] = tile.scores(st.q, t);
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[t][r] = sc[t][r] * p.scale_log2;
      if (key0 + 32 > kb1) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (key0 + 16 * t + 4 * g + r >= kb1) x[t][r] = -INFINITY;
      }
      float mx = x[0][0];
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, x[t][r]);
      const float m_new = fmaxf(st.m, column_max(mx));
      const float mu = m_new == -INFINITY ? 0.f : m_new;  // nothing above -inf yet: weights 0
      float corr = fast_exp2(st.m - mu);
      float sum = 0.f;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[t][r] = fast_exp2(x[t][r] - (mu - Tile::kShift));
          sum += x[t][r];
        }
      if (!FROZEN || live_col) {
        st.l = st.l * corr + sum;
        st.m = m_new;
      } else {
        corr = 1.f;
      }
      if (__any(corr != 1.f)) {
#pragma unroll
        for (int k = 0; k < NBLK; ++k)
#pragma unroll
          for (int e = 0; e < E; ++e) st.o[k][e] *= corr;
      }
    }
    if (FROZEN && !live_col) {
      // columns past the unit's repeat its last one (never written)
      const float* wr = w + (min(c, nc - 1) - nl) * pitch + (key0 - kb0) + 4 * g;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const float4 f = *reinterpret_cast<const float4*>(wr + 16 * t);
        x[t][0] = f.x; x[t][1] = f.y; x[t][2] = f.z; x[t][3] = f.w;
      }
    }
    tile.pv(st.o, x);
  };
  // the frozen weights behind the first tile's loads, unless that keeps too many
  // registers alive; the first barrier also ends the last block's reads
  constexpr bool kEarly = sizeof(Tile) < 512;
  Tile ta;
  if (kEarly && n_it > 0) load(ta, 0);
  if (FROZEN) {
    __syncthreads();
    frozen_weights(p, w, pitch, c0, nl, nc, n, kb0, kb1, wave, W, lane, Tile::kShift != 0.f ? 256.f : 1.f);
    __syncthreads();
  }
  if (n_it == 0) return;
  if (!kEarly) load(ta, 0);
  if constexpr (sizeof(Tile) <= 512) {
    // two tiles in registers: the next step's loads are in flight while a step
    // is computed.  They are issued without a condition (past the end the last
    // step again), so that the wait for a tile leaves the next one's loads out.
    Tile tb;
    for (int it = 0;;) {
      load(tb, min(it + 1, n_it - 1));
      compute(ta, it);
      if (++it >= n_it) break;
      load(ta, min(it + 1, n_it - 1));
      compute(tb, it);
      if (++it >= n_it) break;
    }
  } else {
    // float32 at hd 256: one tile is half of the registers
    for (int it = 0;;) {
      compute(ta, it);
      if (++it >= n_it) break;
      load(ta, it);
    }
  }
}

// Cut sequences.  The launch has n_ranges workgroups per unit, and the
// sequences' keys are dealt to them in ranges of `runs` runs of 128 keys (at
// least p.chunk keys): as even a share of all cached tokens as whole ranges
// allow, whatever the sequences' lengths and the page table's width are.  Every
// wave works this out from the lengths for itself (n_ranges >= 2 B).
struct Ranges {
  int runs;   // runs of 128 keys per range
  int n0;     // this lane's sequence among the first 64, in runs
  __device__ static inline int len(const PagedAttnParams& p, int b) {  // in runs, at most 2^23
    return b < p.B ? (min(max(p.lengths[b], 0), p.capacity) + 127) >> 7 : 0;
  }
  // ceil(n / runs): the reciprocal's estimate is off by at most one
  __device__ inline int count(int n) const {
    const int x = n + runs - 1;
    int q = (int)((float)x * __builtin_amdgcn_rcpf((float)runs));
    q -= q * runs > x;
    q += (q + 1) * runs <= x;
    return q;
  }

  __device__ inline Ranges(const PagedAttnParams& p, int lane) {
    n0 = len(p, lane);
    float total = (float)n0;
    for (int b = lane + 64; b < p.B; b += 64) total += (float)len(p, b);
    // about half a range per sequence is lost to whole ranges
    const float share = dpp_wave_sum(total) * __builtin_amdgcn_rcpf((float)p.n_ranges - 0.5f * (float)p.B);
    runs = max((int)share + 1, p.chunk >> 7);
    for (;;) {  // ends at the latest where every sequence is one range
      int n = count(n0);
      for (int b = lane + 64; b < p.B; b += 64) n += count(len(p, b));
      if ((int)dpp_wave_sum((float)n) <= p.n_ranges) break;
      runs += (runs >> 3) + 1;
    }
    runs = __builtin_amdgcn_readfirstlane(runs);
  }
  // Sequence and place in it of range j (b = -1: there is none), or, with
  // want >= 0, the first range of sequence `want` in `first`.
  __device__ inline void find(const PagedAttnParams& p, int lane, int j, int want, int& b, int& place, int& first) const {
    int base = 0;
    b = -1;
    for (int b0 = 0; b0 < p.B; b0 += 64) {
      const int r = count(b0 == 0 ? n0 : len(p, b0 + lane));
      const int incl = wave_scan(r), excl = base + incl - r;
      if (want >= b0 && want < b0 + 64) first = __builtin_amdgcn_readlane(excl, want - b0);
      const uint64_t hit = __ballot(j >= excl && j < excl + r);
      if (hit != 0) {
        const int at = __builtin_ctzll(hit);
        b = b0 + at;
        place = j - __builtin_amdgcn_readlane(excl, at);
      }
      base += __builtin_amdgcn_readlane(incl, 63);
    }
  }
};

// Four d of one column's sum over the keys j0..j1-1, where the products of the
// walk gave NaN: an infinite value times the two terms of its weight (0 inf,
// inf - inf), or times the weight 0 of a row that a step repeats past the end.
// Once more then, each value that is not finite times its whole weight (what is
// finite does not change the sum).  A sum without such a value stays NaN.
template <typename T, int HD>
__device__ __forceinline__ float4 sum_of_unfinite(const PagedAttnParams& p, float4 acc, int u, int b, int col, int j0, int j1,
                                                  float mu, int d) {
  const int n = p.lengths[b];
  if (n > p.capacity) return acc;
  const PagedUnit un = p.unit[u];
  const int64_t word = p.col[un.c0 + col];
  const int state = col_state(word), row = col_pat(word);
  const bool fits = state == 0 || n <= (state == 1 ? p.p_S : p.d_S);
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + col_q(word) * p.q_sh;
  const T* kc = reinterpret_cast<const T*>(p.kc) + un.k * p.k_sh;
  const T* vc = reinterpret_cast<const T*>(p.vc) + un.v * p.v_sh;
  const int32_t* table = p.table + b * p.t_sb;
  float r[4] = {0.f, 0.f, 0.f, 0.f}, a[4] = {acc.x, acc.y, acc.z, acc.w};
  int found = 0;  // bit e: a[e] has one
  for (int j = j0; j < j1; ++j) {
    const int page = table[j >> p.page_shift], slot = j & ((1 << p.page_shift) - 1);
    if (page < 0 || page >= p.n_pages) return acc;
    const float4 v4 = load4(vc + page * p.v_sp + (int64_t)slot * p.v_st + d);
    const float v[4] = {v4.x, v4.y, v4.z, v4.w};
    bool any = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) any |= !(fabsf(v[e]) < INFINITY);
    float w = __builtin_nanf("");
    if (state == 0) {  // a weight that is not finite makes the column's sum of weights NaN
      if (!any) continue;
      const T* k = kc + page * p.k_sp + (int64_t)slot * p.k_st;
      float s = 0.f;
      for (int c = 0; c < HD; c += 4) {
        const float4 x = load4(q + c), y = load4(k + c);
        s = fmaf(x.x, y.x, fmaf(x.y, y.y, fmaf(x.z, y.z, fmaf(x.w, y.w, s))));
      }
      w = fast_exp2(s * p.scale_log2 - mu);
    } else if (!fits) {
    } else if (state == 1) {
      w = load_as_f32(p.patt, row * p.p_sh + (n - 1) * p.p_si + j * p.p_sj, p.patt_dtype);
    } else {
      w = decomposed_weight(load_as_f32(p.alpha, row * p.a_sh + j * p.a_ss, p.a_dtype),
                            load_as_f32(p.rho, row * p.r_sh + (n - 1 - j) * p.r_ss, p.r_dtype),
                            load_as_f32(p.z, row * p.z_sh + (n - 1) * p.z_ss, p.z_dtype));
    }
    const bool all = !(fabsf(w) < INFINITY);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (all || !(fabsf(v[e]) < INFINITY)) {
        r[e] += w * v[e];
        found |= 1 << e;
      }
    bool open = false;  // a NaN stays one
#pragma unroll
    for (int e = 0; e < 4; ++e) open |= a[e] != a[e] && r[e] == r[e];
    if (!open) break;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (a[e] != a[e] && (found >> e & 1)) a[e] = r[e];
  return make_float4(a[0], a[1], a[2], a[3]);
}

// Grid: one workgroup per (unit, range), units fastest; uncut: per (unit,
// sequence).
template <typename T, int HD, bool CUT>
__global__ __launch_bounds__(64 * paged_max_waves(sizeof(T), HD), paged_simd_waves(sizeof(T), HD)) void paged_attn_kernel(
    const PagedAttnParams p) {
  using Tile = PagedTile<T, HD>;
  constexpr int E = Tile::E, NBLK = Tile::NBLK;
  const int lane = threadIdx.x & 63, W = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int u = blockIdx.x % p.n_units, item = blockIdx.x / p.n_units;
  int b = item, chunk = p.chunk, place = 0, unused;
  if constexpr (CUT) {
    const Ranges ranges(p, lane);
    ranges.find(p, lane, item, -1, b, place, unused);
    chunk = 128 * ranges.runs;
    b = __builtin_amdgcn_readfirstlane(b);
    place = __builtin_amdgcn_readfirstlane(place);
    if (b < 0) return;
  }
  const PagedUnit un = p.unit[u];
  const int c0 = un.c0, nc = un.cols, nl = un.live;

  const int n_in = p.lengths[b];
  const int n = n_in < 0 ? 0 : (n_in > p.capacity ? p.capacity : n_in);
  const int j0 = place * chunk, j1 = min(n, j0 + chunk);

  extern __shared__ __align__(16) float lds[];
  float* sm_ml = lds;           // [W][16][2]
  float* sm_o = lds + W * 32;   // [W][nc][HD + kOPad], before it the frozen weights

  const bool live_col = c < nl;
  PagedWave<T, HD> st;
  {
    const T* qrow = reinterpret_cast<const T*>(p.q);
    if (live_col) qrow += b * p.q_sb + col_q(p.col[c0 + c]) * p.q_sh;
    Tile::load_q(st.q, qrow, live_col, g);
  }
#pragma unroll
  for (int k = 0; k < NBLK; ++k)
#pragma unroll
    for (int e = 0; e < E; ++e) st.o[k][e] = zero4();
  st.m = live_col || c >= nc ? -INFINITY : 0.f;
  st.l = 0.f;
  st.bad = n_in > p.capacity;

  const char* kc = reinterpret_cast<const char*>(p.kc) + un.k * p.k_sh * (int64_t)sizeof(T);
  const char* vc = reinterpret_cast<const char*>(p.vc) + un.v * p.v_sh * (int64_t)sizeof(T);
  const int32_t* table = p.table + b * p.t_sb;
  if (nl == nc) {
    walk<T, HD, true, false>(p, st, kc, vc, table, nullptr, 0, c0, nl, nc, n, j0, j1, wave, W, lane);
  } else {
    // frozen weights in LDS, for as many keys at a time as fit
    const int pitch = min(p.w_floats / (nc - nl), chunk) & ~31;
    for (int kb0 = j0; kb0 < j1; kb0 += pitch) {
      const int kb1 = min(j1, kb0 + pitch);
      if (nl > 0) walk<T, HD, true, true>(p, st, kc, vc, table, sm_o, pitch, c0, nl, nc, n, kb0, kb1, wave, W, lane);
      else walk<T, HD, false, true>(p, st, kc, vc, table, sm_o, pitch, c0, nl, nc, n, kb0, kb1, wave, W, lane);
    }
    __syncthreads();
  }

  // merge of the workgroup's waves: every wave's column maxima and sums and
  // its partial O in LDS, then each thread four d of one column
  st.l = column_sum(st.l);
  if (__any(st.bad)) {
    st.l = __builtin_nanf("");
#pragma unroll
    for (int k = 0; k < NBLK; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e)
        st.o[k][e] = f32x4_t{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
  }
  if (g == 0) {
    sm_ml[(wave * 16 + c) * 2] = st.m;
    sm_ml[(wave * 16 + c) * 2 + 1] = st.l;
  }
  if (c < nc) {
    float* dst = sm_o + (wave * nc + c) * (HD + kOPad);
#pragma unroll
    for (int k = 0; k < NBLK; ++k)
#pragma unroll
      for (int x = 0; x < E; ++x) {  // elements 4x..4x+3 of the lane's 4E consecutive d
        float4 f;
        f.x = st.o[k][(4 * x + 0) % E][(4 * x + 0) / E];
        f.y = st.o[k][(4 * x + 1) % E][(4 * x + 1) / E];
        f.z = st.o[k][(4 * x + 2) % E][(4 * x + 2) / E];
        f.w = st.o[k][(4 * x + 3) % E][(4 * x + 3) / E];
        *reinterpret_cast<float4*>(dst + 16 * E * k + 4 * E * g + 4 * x) = f;
      }
  }
  __syncthreads();
  for (int idx = threadIdx.x; idx < nc * (HD / 4); idx += blockDim.x) {
    const int col = idx / (HD / 4), d = 4 * (idx % (HD / 4));
    float mm = -INFINITY;
    for (int w = 0; w < W; ++w) mm = fmaxf(mm, sm_ml[(w * 16 + col) * 2]);
    const float mu = mm == -INFINITY ? 0.f : mm;
    float ll = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = 0; w < W; ++w) {
      const float f = fast_exp2(sm_ml[(w * 16 + col) * 2] - mu);
      const float4 x = *reinterpret_cast<const float4*>(sm_o + (w * nc + col) * (HD + kOPad) + d);
      ll += f * sm_ml[(w * 16 + col) * 2 + 1];
      acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    }
    const float any = (acc.x + acc.y) + (acc.z + acc.w);  // NaN also of +inf and -inf: each is looked at
    if (any != any && ll == ll) {  // a NaN sum of weights makes the column NaN as it is
      // the arguments read again, by an address that the compiler does not see
      // through, so that none of this is kept in registers during the walk
      // (the kernel has one argument, the start of its segment)
      uint64_t segment = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
      asm volatile("" : "+v"(segment));
      acc = sum_of_unfinite<T, HD>(*reinterpret_cast<const PagedAttnParams*>(segment), acc, u, b, col, j0, j1, mu, d);
    }
    if constexpr (CUT) {
      const int64_t slot = (int64_t)item * p.n_heads + c0 + col;
      *reinterpret_cast<float4*>(p.part_o + slot * HD + d) = acc;
      if (d == 0) {
        p.part_ml[2 * slot] = mm;
        p.part_ml[2 * slot + 1] = ll;
      }
      continue;
    }
    const int h = col_head(p.col[c0 + col]);
    const bool empty = n_in <= 0;
    const float inv = empty ? 0.f : (col < nl ? 1.f / ll : (Tile::kShift != 0.f ? 1.f / 256.f : 1.f));
    acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
    store4(reinterpret_cast<T*>(p.out) + b * p.o_sb + h * p.o_sh + d, acc);
    if (p.lse && d == 0 && col < nl) p.lse[b * p.l_sb + h * p.l_sh] = empty ? -INFINITY : mm + log2f(ll) - Tile::kShift;
  }
}

// Join of the key ranges of one (sequence, column): 256 threads, HD / 4
// lanes per range, ranges in a fixed order.
template <typename T, int HD>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedAttnParams p) {
  constexpr int L = HD / 4, G = 256 / L;  // hd 96: 10 groups of 24, the rest idle
  __shared__ float4 sm[G][L];
  const int col = blockIdx.x % p.n_heads, b = blockIdx.x / p.n_heads;
  const int64_t word = p.col[col];
  const int h = col_head(word);
  const bool live = col_state(word) == 0;
  const int n_in = p.lengths[b];
  const bool bad = n_in > p.capacity;
  const int n = n_in < 0 ? 0 : (bad ? p.capacity : n_in);
  const int lane = threadIdx.x & 63;
  const Ranges ranges(p, lane);
  int first = 0, unused_b, unused_place;
  ranges.find(p, lane, -1, b, unused_b, unused_place, first);
  const int ns = ranges.count((n + 127) >> 7);
  const int64_t slot = (int64_t)first * p.n_heads + col;  // of range 0; the next ones n_heads further
  const float* ml = p.part_ml + 2 * slot;
  const int step = 2 * p.n_heads;
  float mm = -INFINITY;
  for (int s = lane; s < ns; s += 64) mm = fmaxf(mm, ml[s * step]);
  mm = wave_max(mm);
  const float mu = mm == -INFINITY ? 0.f : mm;
  float ll = 0.f;
  for (int s = lane; s < ns; s += 64) ll += fast_exp2(ml[s * step] - mu) * ml[s * step + 1];
  ll = dpp_wave_sum(ll);
  const int grp = threadIdx.x / L, d4 = threadIdx.x % L;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (grp < G) {
    for (int s = grp; s < ns; s += G) {
      const float f = fast_exp2(ml[s * step] - mu);
      const float4 x = *reinterpret_cast<const float4*>(p.part_o + (slot + (int64_t)s * p.n_heads) * HD + 4 * d4);
      acc.x += f * x.x; acc.y += f * x.y; acc.z += f * x.z; acc.w += f * x.w;
    }
    sm[grp][d4] = acc;
  }
  __syncthreads();
  if (threadIdx.x >= L) return;
  acc = sm[0][d4];
  for (int k = 1; k < G; ++k) {
    const float4 x = sm[k][d4];
    acc.x += x.x; acc.y += x.y; acc.z += x.z; acc.w += x.w;
  }
  constexpr float shift = PagedTile<T, HD>::kShift;
  float inv = live ? 1.f / ll : (shift != 0.f ? 1.f / 256.f : 1.f);
  if (n == 0) inv = 0.f;
  if (bad) inv = __builtin_nanf("");
  acc.x *= inv; acc.y *= inv; acc.z *= inv; acc.w *= inv;
  store4(reinterpret_cast<T*>(p.out) + b * p.o_sb + h * p.o_sh + 4 * d4, acc);
  if (p.lse && d4 == 0 && live)
    p.lse[b * p.l_sb + h * p.l_sh] = bad ? __builtin_nanf("") : (n == 0 ? -INFINITY : mm + log2f(ll) - shift);
}

template <typename T, int HD>
static hipError_t launch_paged_t(const PagedAttnParams& p, hipStream_t s) {
  const size_t o_floats = (size_t)p.waves * p.max_cols * (HD + kOPad);
  const size_t lds = sizeof(float) * (p.waves * 32 + (o_floats > (size_t)p.w_floats ? o_floats : (size_t)p.w_floats));
  const dim3 block(64 * p.waves);
  if (p.n_ranges == 1) {
    hipLaunchKernelGGL((paged_attn_kernel<T, HD, false>), dim3((unsigned)((int64_t)p.B * p.n_units)), block, lds, s, p);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((paged_attn_kernel<T, HD, true>), dim3((unsigned)(p.n_ranges * p.n_units)), block, lds, s, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL((paged_join_kernel<T, HD>), dim3((unsigned)(p.B * p.n_heads)), dim3(256), 0, s, p);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_paged_dt(const PagedAttnParams& p, int hd, hipStream_t s) {
  switch (hd) {
    case 32: return launch_paged_t<T, 32>(p, s);
    case 64: return launch_paged_t<T, 64>(p, s);
    case 96: return launch_paged_t<T, 96>(p, s);
    case 128: return launch_paged_t<T, 128>(p, s);
    case 256: return launch_paged_t<T, 256>(p, s);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_paged_attn(const PagedAttnParams& p, int dtype, int hd, hipStream_t s) {
  if (dtype == kBF16) return launch_paged_dt<__bf16>(p, hd, s);
  if (dtype == kF16) return launch_paged_dt<_Float16>(p, hd, s);
  if (dtype == kF32) return launch_paged_dt<float>(p, hd, s);
  return hipErrorInvalidValue;
}

}  // namespace saf
