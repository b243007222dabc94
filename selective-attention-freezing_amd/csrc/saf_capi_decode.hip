// Host side of the operators behind the prefill: the paged cache's append and
// single-token attention, and the log probabilities of tokens.  Argument
// checks and launches of the C-ABI in include/saf_attn.h; nothing here
// allocates or throws.
#include <cmath>

#include "saf_host.h"

using namespace saf;

namespace {

constexpr int64_t kMaxGrid = 0x7fffffff;

bool act_dtype(int d) { return d == SAF_BF16 || d == SAF_F16 || d == SAF_F32; }

// (B, U, T, HD) rows or cache pages (P, U, PS, HD): 16-byte aligned rows with
// a unit last stride.
int check_rows(const saf_tensor_t& t, const char* name, int dtype) {
  if (t.ndim != 4) return fail(SAF_EINVAL, "%s must be 4-D (got %d-D)", name, t.ndim);
  if (t.dtype != dtype) return fail(SAF_EINVAL, "%s must share v's dtype (got %s)", name, dtype_name(t.dtype));
  if (t.stride[3] != 1 && t.size[3] != 1)
    return fail(SAF_EALIGN, "%s must have a contiguous last dimension (stride %lld)", name, (long long)t.stride[3]);
  const int es = elem_size(dtype);
  if (reinterpret_cast<uintptr_t>(t.data) % 16 != 0) return fail(SAF_EALIGN, "%s data pointer is not 16-byte aligned", name);
  for (int i = 0; i < 3; ++i)
    if (t.size[i] > 1 && (t.stride[i] * es) % 16 != 0)
      return fail(SAF_EALIGN, "%s stride %d (%lld elements) is not a multiple of 16 bytes", name, i, (long long)t.stride[i]);
  return SAF_OK;
}

// A cache: its pages' slots are addressed with 32-bit offsets within a page.
int check_cache(const saf_tensor_t& t, const char* name, int dtype) {
  if (int rc = check_rows(t, name, dtype)) return rc;
  if (t.size[0] < 1) return fail(SAF_EINVAL, "%s has no pages", name);
  if (t.size[0] > kMaxGrid || t.size[1] > 32767) return fail(SAF_EUNSUPPORTED, "%s has too many pages or heads", name);
  const int64_t ps = t.size[2];
  if (ps < 16 || ps > (1 << 20) || (ps & (ps - 1)) != 0)
    return fail(SAF_EUNSUPPORTED, "%s: page size %lld is not a power of two from 16 to 2^20", name, (long long)ps);
  const int64_t row = t.stride[2] * elem_size(dtype);
  if (row < 0 || row * ps >= kMaxGrid) return fail(SAF_EUNSUPPORTED, "%s: a page must span less than 2 GiB", name);
  if (t.stride[2] < t.size[3]) return fail(SAF_EINVAL, "%s slots overlap (stride %lld)", name, (long long)t.stride[2]);
  return SAF_OK;
}

int check_i32(const saf_tensor_t& t, const char* name, int ndim, int64_t n) {
  if (!present(t) || t.dtype != SAF_I32 || t.ndim != ndim || t.size[0] != n)
    return fail(SAF_EINVAL, "%s must be int32 with %d dimension(s) and %lld rows", name, ndim, (long long)n);
  if (t.size[ndim - 1] > 1 && t.stride[ndim - 1] != 1) return fail(SAF_EALIGN, "%s must have a unit last stride", name);
  return SAF_OK;
}

int page_shift_of(int64_t ps) {
  int s = 0;
  while ((int64_t(1) << s) < ps) ++s;
  return s;
}

// Table columns x page size, the positions a sequence can have.
int check_capacity(const saf_tensor_t& table, int64_t ps, int& capacity) {
  const int64_t cap = table.size[1] * ps;
  if (cap > (int64_t(1) << 30)) return fail(SAF_EUNSUPPORTED, "page_table covers more than 2^30 positions");
  capacity = (int)cap;
  return SAF_OK;
}

int check_vec(const saf_tensor_t& t, const char* name, int64_t n) {
  if (t.ndim != 1 || t.size[0] != n || !act_dtype(t.dtype) || (n > 1 && t.stride[0] != 1))
    return fail(SAF_EINVAL, "%s must be a contiguous (%lld,) floating vector", name, (long long)n);
  return SAF_OK;
}

// ---- paged attention ----------------------------------------------------------

// Key ranges.  Sequences are cut only where whole ones would leave half of the
// resident workgroups idle, into as many ranges together as fill them once
// (whole rounds cost more than a ragged tail: 64 sequences of up to 4096 keys,
// 768 units for 768 workgroups, took 86 us whole, 94 us in two ranges each,
// 106 us in eight), of at least kMinKeys keys, and only where a unit's keys and
// values reach kSplitBytes (one CU reads about 55 GB/s): below, the second
// launch costs what the shorter walk saves.  As calls the two meet between 448 and
// 512 KB whatever the type and head dim (12 heads of 64, bf16, whole and cut: 9.8
// and 13.2 us at 256 KB, 13.8 and 13.4 at 448, 15.8 and 11.8 at 512; 32 heads on 8
// KV heads of 128: 9.9 and 13.0, 12.9 and 12.7, 14.1 and 13.0; float32: 10.3 and
// 14.9, 14.1 and 13.7, 15.3 and 15.0), replayed as a graph, without the host's
// part, between 320 and 448 KB.  Ranges dealt over all
// sequences instead of an equal number to each: 16 ragged sequences in two KV
// groups 25 us against 29, 8 at hd 256 69 against 73.  Uncut sequences from
// kWideFrom positions on run eight waves where the registers allow (64 x 4096
// keys: 80 us against 86; 128 x 8192 keys at hd 128: 422 against 442); short
// ones four (64 x 128 keys: 7.4 us against 12.6, idle waves cost their launch).
constexpr int kMinKeys = 256, kWideFrom = 2048;
constexpr int64_t kSplitBytes = 512 << 10;
constexpr int kWeightFloats = 6144;  // 24 KB: five workgroups of a CU fit its LDS with their partial sums

int plan_paged(const saf_paged_attn_args* a, PagedAttnParams& p, int& dtype, int& hd) {
  if (a == nullptr) return fail(SAF_EINVAL, "args is NULL");
  const saf_tensor_t &vc = a->v_cache, &o = a->out;
  if (!present(vc) || !present(o)) return fail(SAF_EINVAL, "v_cache and out are required");
  if (!act_dtype(vc.dtype)) return fail(SAF_EUNSUPPORTED, "unsupported v_cache dtype %s", dtype_name(vc.dtype));
  dtype = vc.dtype;
  if (int rc = check_cache(vc, "v_cache", dtype)) return rc;
  hd = (int)vc.size[3];
  if (!supported_hd(vc.size[3]))
    return fail(SAF_EUNSUPPORTED, "head_dim %lld is not supported (32, 64, 96, 128, 256)", (long long)vc.size[3]);
  const int H = a->n_heads;
  if (H <= 0 || H > SAF_MAX_HEADS) return fail(SAF_EUNSUPPORTED, "n_heads %d outside 1..%d", H, SAF_MAX_HEADS);
  if (a->frozen == nullptr) return fail(SAF_EINVAL, "frozen (host head-state table) is required");
  const int64_t HV = vc.size[1];
  if (a->kvidx == nullptr && HV != H) return fail(SAF_EINVAL, "v_cache must hold one head per output head (or pass kvidx)");
  if (int rc = check_rows(o, "out", dtype)) return rc;
  const int64_t B = o.size[0];
  if (o.size[1] != H || o.size[2] != 1 || o.size[3] != hd)
    return fail(SAF_EINVAL, "out must have shape (B, H, 1, HD) = (%lld, %d, 1, %d)", (long long)B, H, hd);
  if (int rc = check_i32(a->page_table, "page_table", 2, B)) return rc;
  if (int rc = check_i32(a->lengths, "lengths", 1, B)) return rc;
  if (int rc = check_capacity(a->page_table, vc.size[2], p.capacity)) return rc;
  if (!std::isfinite(a->sm_scale)) return fail(SAF_EINVAL, "sm_scale must be finite");
  bool any_live = false, any_dense = false, any_dec = false;
  for (int h = 0; h < H; ++h) {
    const int st = a->frozen[h];
    if (st < 0 || st > 2) return fail(SAF_EINVAL, "frozen[%d] = %d is not a head state (0, 1, 2)", h, st);
    if (a->kvidx && (a->kvidx[h] < 0 || a->kvidx[h] >= HV))
      return fail(SAF_EINVAL, "kvidx must index the HKV heads of the caches (kvidx[%d] = %d)", h, a->kvidx[h]);
    any_live |= st == 0;
    any_dense |= st == 1;
    any_dec |= st == 2;
  }
  if (any_live) {
    const saf_tensor_t &q = a->q, &kc = a->k_cache;
    if (!present(q) || !present(kc)) return fail(SAF_EINVAL, "live heads require q and k_cache");
    if (int rc = check_rows(q, "q", dtype)) return rc;
    if (q.size[0] != B || q.size[2] != 1 || q.size[3] != hd || q.size[1] > 32767)
      return fail(SAF_EINVAL, "q must have shape (B, U, 1, HD)");
    if (int rc = check_cache(kc, "k_cache", dtype)) return rc;
    if (kc.size[0] != vc.size[0] || kc.size[2] != vc.size[2] || kc.size[3] != hd)
      return fail(SAF_EINVAL, "k_cache and v_cache must have the same pages, page size and head dimension");
    if (kc.size[1] != (a->kvidx ? HV : q.size[1]))
      return fail(SAF_EINVAL, "k_cache must hold one head per live slot of q (with kvidx: the HKV heads of v_cache)");
    for (int h = 0; h < H; ++h) {
      const int slot = a->hidx ? a->hidx[h] : h;
      if (a->frozen[h] == 0 && (slot < 0 || slot >= q.size[1]))
        return fail(SAF_EINVAL, "hidx[%d] = %d does not index the %lld compact q heads", h, slot, (long long)q.size[1]);
    }
    p.q = q.data; p.q_sb = q.stride[0]; p.q_sh = q.stride[1];
    p.kc = kc.data; p.k_sp = kc.stride[0]; p.k_sh = kc.stride[1]; p.k_st = (int)kc.stride[2];
  }
  if (any_dense) {
    const saf_tensor_t& t = a->patt;
    if (!present(t)) return fail(SAF_EINVAL, "dense-frozen heads require patt");
    if (t.ndim != 3 || t.size[1] != t.size[2] || t.size[0] > 32767 || t.size[1] > kMaxGrid)
      return fail(SAF_EINVAL, "patt must have shape (P, S, S)");
    if (!act_dtype(t.dtype)) return fail(SAF_EUNSUPPORTED, "unsupported patt dtype %s", dtype_name(t.dtype));
    for (int h = 0; h < H; ++h) {
      const int row = a->pidx ? a->pidx[h] : h;
      if (a->frozen[h] == 1 && (row < 0 || row >= t.size[0]))
        return fail(SAF_EINVAL, "pidx for dense-frozen heads must index patt (head %d: row %d of %lld)", h, row,
                    (long long)t.size[0]);
    }
    p.patt = t.data; p.patt_dtype = t.dtype; p.p_S = (int)t.size[1];
    p.p_sh = t.stride[0]; p.p_si = t.stride[1]; p.p_sj = t.stride[2];
  }
  if (any_dec) {
    const saf_tensor_t* t[3] = {&a->alpha, &a->rho, &a->z};
    const char* names[3] = {"alpha", "rho", "z"};
    for (int i = 0; i < 3; ++i) {
      if (!present(*t[i])) return fail(SAF_EINVAL, "decomposed-frozen heads require alpha/rho/z");
      if (t[i]->ndim != 2 || t[i]->size[0] != H || t[i]->size[1] != t[0]->size[1] || t[i]->size[1] > kMaxGrid)
        return fail(SAF_EINVAL, "alpha, rho and z must have matching (H, S) shapes (%s)", names[i]);
      if (!act_dtype(t[i]->dtype)) return fail(SAF_EUNSUPPORTED, "unsupported %s dtype %s", names[i], dtype_name(t[i]->dtype));
    }
    p.alpha = t[0]->data; p.a_dtype = t[0]->dtype; p.a_sh = t[0]->stride[0]; p.a_ss = t[0]->stride[1];
    p.rho = t[1]->data; p.r_dtype = t[1]->dtype; p.r_sh = t[1]->stride[0]; p.r_ss = t[1]->stride[1];
    p.z = t[2]->data; p.z_dtype = t[2]->dtype; p.z_sh = t[2]->stride[0]; p.z_ss = t[2]->stride[1];
    p.d_S = (int)t[0]->size[1];
  }
  if (present(a->lse)) {
    const saf_tensor_t& t = a->lse;
    if (t.dtype != SAF_F32 || t.ndim != 3 || t.size[0] != B || t.size[1] != H || t.size[2] != 1)
      return fail(SAF_EINVAL, "lse must be fp32 (B, H, 1)");
    p.lse = reinterpret_cast<float*>(t.data); p.l_sb = t.stride[0]; p.l_sh = t.stride[1];
  }
  p.vc = vc.data; p.v_sp = vc.stride[0]; p.v_sh = vc.stride[1]; p.v_st = (int)vc.stride[2];
  p.out = o.data; p.o_sb = o.stride[0]; p.o_sh = o.stride[1];
  p.table = reinterpret_cast<const int32_t*>(a->page_table.data); p.t_sb = a->page_table.stride[0];
  p.lengths = reinterpret_cast<const int32_t*>(a->lengths.data);
  p.page_shift = page_shift_of(vc.size[2]);
  p.n_pages = (int)vc.size[0];
  p.n_heads = H;
  p.scale_log2 = a->sm_scale * kLog2e;

  // units: without kvidx one head each; with it a KV head's query heads, live
  // ones first, at most 16 columns per unit
  int nu = 0, col = 0, max_frozen = 0;
  p.max_cols = 1;
  auto add = [&](int h, bool open, int k, int v) {
    if (open) p.unit[nu++] = PagedUnit{(int16_t)k, (int16_t)v, (uint8_t)col, 0, 0, 0};
    PagedUnit& u = p.unit[nu - 1];
    const int st = a->frozen[h];
    ++u.cols;
    u.live += st == 0;
    if (u.cols > p.max_cols) p.max_cols = u.cols;
    if (u.cols - u.live > max_frozen) max_frozen = u.cols - u.live;
    p.col[col++] = col_word(h, st, st == 0 ? (a->hidx ? a->hidx[h] : h) : 0, st == 1 && a->pidx ? a->pidx[h] : h);
  };
  if (a->kvidx == nullptr) {
    for (int h = 0; h < H; ++h) add(h, true, a->frozen[h] == 0 ? (a->hidx ? a->hidx[h] : h) : 0, h);
  } else {
    bool done[SAF_MAX_HEADS] = {};
    for (int h0 = 0; h0 < H; ++h0) {
      if (done[h0]) continue;
      const int kv = a->kvidx[h0];
      bool open = true;
      for (int pass = 0; pass < 2; ++pass)  // live heads, then frozen ones
        for (int h = h0; h < H; ++h) {
          if (a->kvidx[h] != kv || (a->frozen[h] == 0) != (pass == 0)) continue;
          done[h] = true;
          add(h, open, kv, kv);
          open = p.unit[nu - 1].cols == 16;
        }
    }
  }
  p.n_units = nu;

  if (B > kMaxGrid / SAF_MAX_HEADS / 64) return fail(SAF_EUNSUPPORTED, "batch %lld is too large", (long long)B);
  p.B = (int)B;
  // ranges: as many as the resident workgroups leave for each unit
  const int64_t slots = (int64_t)cu_count() * paged_simd_waves(elem_size(dtype), hd);
  int64_t ranges = slots / nu;
  const int64_t most = ((int64_t)p.capacity + kMinKeys - 1) / kMinKeys * B;
  if (ranges > most) ranges = most;
  const int64_t unit_bytes = (int64_t)p.capacity * hd * elem_size(dtype) * 2;
  p.n_ranges = ranges >= 2 * B && B > 0 && unit_bytes >= kSplitBytes ? (int)ranges : 1;
  p.chunk = p.n_ranges > 1 ? kMinKeys : (p.capacity + 31) / 32 * 32;
  if (p.chunk < 32) p.chunk = 32;
  p.waves = p.n_ranges == 1 && p.capacity >= kWideFrom ? paged_max_waves(elem_size(dtype), hd) : 4;
  // LDS of the frozen columns' weights: the whole capacity where that is within
  // kWeightFloats, at least one step per column
  if (max_frozen > 0) {
    int64_t keys = kWeightFloats / max_frozen / 32 * 32;
    if (keys > (p.capacity + 31) / 32 * 32) keys = (p.capacity + 31) / 32 * 32;
    if (keys < 32) keys = 32;
    p.w_floats = (int)keys * max_frozen;
  }
  return SAF_OK;
}

int64_t paged_slots(const PagedAttnParams& p) { return p.n_ranges > 1 ? (int64_t)p.n_heads * p.n_ranges : 0; }

// ---- log probabilities -----------------------------------------------------------

int plan_logprobs(const saf_token_logprobs_args* a, LogprobParams& p, bool outputs) {
  if (a == nullptr) return fail(SAF_EINVAL, "args is NULL");
  const saf_tensor_t &x = a->logits, &t = a->tokens, &st = a->stats;
  if (x.ndim != 2) return fail(SAF_EINVAL, "logits must be 2-D (rows, vocabulary)");
  const int64_t R = x.size[0], V = x.size[1];
  if (!act_dtype(x.dtype)) return fail(SAF_EUNSUPPORTED, "unsupported logits dtype %s", dtype_name(x.dtype));
  if (V < 1 || V > (int64_t(1) << 30)) return fail(SAF_EUNSUPPORTED, "vocabulary %lld outside 1..2^30", (long long)V);
  if (R > 0 && !present(x)) return fail(SAF_EINVAL, "logits are required");
  if (V > 1 && x.stride[1] != 1) return fail(SAF_EALIGN, "logits need a unit column stride");
  if (t.ndim != 1 || t.size[0] != R || (t.dtype != SAF_I32 && t.dtype != SAF_I64) || (R > 0 && !present(t)))
    return fail(SAF_EINVAL, "tokens must be int32 or int64 with one entry per row");
  if (R > 0 && !outputs && !present(st)) return fail(SAF_EINVAL, "the forward's stats are required");
  if (present(st) && (st.ndim != 2 || st.size[0] != R || st.size[1] != 2 || st.dtype != SAF_F32 || st.stride[1] != 1 ||
                      (R > 1 && st.stride[0] != 2)))
    return fail(SAF_EINVAL, "stats must be contiguous fp32 (R, 2)");
  if (!(a->scale > 0.f) || !std::isfinite(a->scale)) return fail(SAF_EINVAL, "scale must be positive and finite");
  if (a->top < 0 || a->top > 32 || a->top > V)
    return fail(SAF_EUNSUPPORTED, "top = %d outside 0..32 or above the vocabulary", a->top);
  auto f32_rows = [&](const saf_tensor_t& o, const char* name) {
    if (o.dtype != SAF_F32 || o.ndim != 1 || o.size[0] != R || (R > 1 && o.stride[0] != 1))
      return fail(SAF_EINVAL, "%s must be a contiguous fp32 (R,) vector", name);
    return (int)SAF_OK;
  };
  if (present(a->entropy))
    if (int rc = f32_rows(a->entropy, "entropy")) return rc;
  if (outputs) {
    if (R > 0 && !present(a->logp)) return fail(SAF_EINVAL, "logp is required");
    if (int rc = f32_rows(a->logp, "logp")) return rc;
    if (a->top > 0 && R > 0) {
      const saf_tensor_t* o[2] = {&a->top_index, &a->top_logp};
      for (int i = 0; i < 2; ++i)
        if (!present(*o[i]) || o[i]->ndim != 2 || o[i]->size[0] != R || o[i]->size[1] != a->top ||
            o[i]->dtype != (i == 0 ? SAF_I64 : SAF_F32) || (a->top > 1 && o[i]->stride[1] != 1) ||
            (R > 1 && o[i]->stride[0] != a->top))
          return fail(SAF_EINVAL, "top_index (int64) and top_logp (fp32) must be contiguous (R, top)");
    }
  }
  p.logits = x.data; p.x_rs = x.stride[0]; p.R = R; p.V = (int)V;
  p.tokens = t.data; p.tok_i64 = t.dtype == SAF_I64; p.tok_st = t.stride[0];
  p.ignore = a->ignore_index;
  p.scale = a->scale;
  p.logp = reinterpret_cast<float*>(a->logp.data);
  p.entropy = reinterpret_cast<float*>(a->entropy.data);
  p.stats = reinterpret_cast<float*>(st.data);
  p.top = a->top;
  p.top_index = reinterpret_cast<int64_t*>(a->top_index.data);
  p.top_logp = reinterpret_cast<float*>(a->top_logp.data);
  p.n_cu = cu_count();
  // few long rows (256 KB and more) are cut into segments of at least 16 KB, one
  // workgroup each: one CU reads about 55 GB/s (4 rows of 151936: 10 us with the
  // join, 16 us whole; shorter rows do not pay for the second launch)
  const int64_t row_bytes = V * elem_size(x.dtype);
  int64_t seg = 1;
  if (R > 0 && R <= p.n_cu / 4 && row_bytes >= (256 << 10)) {
    seg = 2 * (int64_t)p.n_cu / R;
    if (seg > row_bytes >> 14) seg = row_bytes >> 14;
    if (seg > 64) seg = 64;
  }
  const int64_t len = ((V + seg - 1) / seg + 63) / 64 * 64;
  p.seg_len = (int)(seg == 1 ? V : len);
  p.n_seg = seg == 1 ? 1 : (int)((V + len - 1) / len);
  if (R > kMaxGrid / (p.n_seg > 1 ? p.n_seg : 1)) return fail(SAF_EUNSUPPORTED, "too many rows (%lld)", (long long)R);
  return SAF_OK;
}

int64_t logprob_ws(const LogprobParams& p) { return p.n_seg > 1 ? p.R * p.n_seg * (16 + 8 * (int64_t)p.top) : 0; }

}  // namespace

extern "C" {

int64_t saf_paged_attn_workspace_bytes(const saf_paged_attn_args* args) {
  PagedAttnParams p{};
  int dtype, hd;
  if (plan_paged(args, p, dtype, hd) != SAF_OK) return -1;
  return paged_slots(p) * (hd + 2) * 4;
}

int saf_paged_attn_fwd(const saf_paged_attn_args* args, void* stream) {
  PagedAttnParams p{};
  int dtype, hd;
  if (int rc = plan_paged(args, p, dtype, hd)) return rc;
  if (p.B == 0) return SAF_OK;
  const int64_t slots = paged_slots(p), need = slots * (hd + 2) * 4;
  if (need > 0) {
    if (args->workspace == nullptr || args->workspace_bytes < need)
      return fail(SAF_EWORKSPACE, "paged attention needs a %lld-byte workspace (got %lld)", (long long)need,
                  (long long)args->workspace_bytes);
    if (reinterpret_cast<uintptr_t>(args->workspace) % 16 != 0) return fail(SAF_EALIGN, "workspace must be 16-byte aligned");
    p.part_o = reinterpret_cast<float*>(args->workspace);
    p.part_ml = p.part_o + slots * hd;
  }
  return launched(launch_paged_attn(p, dtype, hd, reinterpret_cast<hipStream_t>(stream)), "paged_attn");
}

int saf_paged_append(const saf_paged_append_args* a, void* stream) {
  if (a == nullptr) return fail(SAF_EINVAL, "args is NULL");
  PagedAppendParams p{};
  const saf_tensor_t &v = a->v, &vc = a->v_cache;
  if (!present(v) || !present(vc)) return fail(SAF_EINVAL, "v and v_cache are required");
  if (!act_dtype(v.dtype)) return fail(SAF_EUNSUPPORTED, "unsupported v dtype %s", dtype_name(v.dtype));
  if (int rc = check_rows(v, "v", v.dtype)) return rc;
  if (int rc = check_cache(vc, "v_cache", v.dtype)) return rc;
  const int64_t B = v.size[0], T = v.size[2], hd = v.size[3];
  if (!supported_hd(hd)) return fail(SAF_EUNSUPPORTED, "head_dim %lld is not supported (32, 64, 96, 128, 256)", (long long)hd);
  if (vc.size[1] != v.size[1] || vc.size[3] != hd) return fail(SAF_EINVAL, "v_cache must hold v's heads and head dimension");
  if (int rc = check_i32(a->page_table, "page_table", 2, B)) return rc;
  if (int rc = check_i32(a->positions, "positions", 1, B)) return rc;
  if (present(a->counts))
    if (int rc = check_i32(a->counts, "counts", 1, B)) return rc;
  if (int rc = check_capacity(a->page_table, vc.size[2], p.capacity)) return rc;
  const bool has_k = present(a->k), has_q = present(a->q);
  if (has_k) {
    const saf_tensor_t &k = a->k, &kc = a->k_cache;
    if (!present(kc)) return fail(SAF_EINVAL, "k needs k_cache");
    if (int rc = check_rows(k, "k", v.dtype)) return rc;
    if (int rc = check_cache(kc, "k_cache", v.dtype)) return rc;
    if (k.size[0] != B || k.size[2] != T || k.size[3] != hd) return fail(SAF_EINVAL, "k and v batch, tokens and head dimension must match");
    if (kc.size[0] != vc.size[0] || kc.size[1] != k.size[1] || kc.size[2] != vc.size[2] || kc.size[3] != hd)
      return fail(SAF_EINVAL, "k_cache must hold k's heads in v_cache's pages");
    p.k = k.data; p.k_sb = k.stride[0]; p.k_sh = k.stride[1]; p.k_st = k.stride[2];
    p.kc = kc.data; p.kc_sp = kc.stride[0]; p.kc_sh = kc.stride[1]; p.kc_st = kc.stride[2];
    p.Uk = (int)k.size[1];
  }
  if (has_q) {
    const saf_tensor_t &q = a->q, &qo = a->q_out;
    if (!present(qo)) return fail(SAF_EINVAL, "q needs q_out");
    if (int rc = check_rows(q, "q", v.dtype)) return rc;
    if (int rc = check_rows(qo, "q_out", v.dtype)) return rc;
    if (q.size[0] != B || q.size[2] != T || q.size[3] != hd) return fail(SAF_EINVAL, "q and v batch, tokens and head dimension must match");
    for (int i = 0; i < 4; ++i)
      if (qo.size[i] != q.size[i]) return fail(SAF_EINVAL, "q_out must have q's shape");
    if (q.size[1] > 32767) return fail(SAF_EUNSUPPORTED, "too many query heads");
    p.q = q.data; p.q_sb = q.stride[0]; p.q_sh = q.stride[1]; p.q_st = q.stride[2];
    p.q_out = qo.data; p.qo_sb = qo.stride[0]; p.qo_sh = qo.stride[1]; p.qo_st = qo.stride[2];
    p.Uq = (int)q.size[1];
  }
  if (present(a->cos) != present(a->sin)) return fail(SAF_EINVAL, "cos and sin go together");
  if (present(a->cos)) {
    const saf_tensor_t* cs[2] = {&a->cos, &a->sin};
    for (int i = 0; i < 2; ++i) {
      const saf_tensor_t& t = *cs[i];
      if (t.ndim != 2 || !act_dtype(t.dtype) || t.dtype != a->cos.dtype || t.size[0] != a->cos.size[0] ||
          t.size[1] != a->cos.size[1] || t.size[0] > kMaxGrid)
        return fail(SAF_EINVAL, "cos and sin must be (T', RD) caches of one shape and floating dtype");
      if (t.stride[1] != 1) return fail(SAF_EALIGN, "cos and sin need a unit column stride");
    }
    const int64_t rd = a->cos.size[1];
    if (rd < 16 || rd > hd || rd % 16 != 0)
      return fail(SAF_EUNSUPPORTED, "rotary dimension %lld is not a multiple of 16 up to the head dimension", (long long)rd);
    p.cos = a->cos.data; p.sin = a->sin.data; p.cs_st = a->cos.stride[0]; p.sn_st = a->sin.stride[0];
    p.cs_dtype = a->cos.dtype; p.cs_rows = (int)a->cos.size[0]; p.rd = (int)rd;
    auto al = [](const saf_tensor_t& t) {
      return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && (t.size[0] <= 1 || t.stride[0] * elem_size(t.dtype) % 16 == 0);
    };
    p.cs_vec = al(a->cos) && al(a->sin);
  }
  if (present(a->q_weight) != present(a->k_weight)) return fail(SAF_EINVAL, "q_weight and k_weight go together");
  if (present(a->q_weight)) {
    if (int rc = check_vec(a->q_weight, "q_weight", hd)) return rc;
    if (int rc = check_vec(a->k_weight, "k_weight", hd)) return rc;
    if (a->q_weight.dtype != a->k_weight.dtype) return fail(SAF_EINVAL, "q_weight and k_weight must share a dtype");
    if (!(a->eps >= 0.f)) return fail(SAF_EINVAL, "eps must be a non-negative number");
    p.q_w = a->q_weight.data; p.k_w = a->k_weight.data; p.w_dtype = a->q_weight.dtype; p.eps = a->eps;
    p.w_vec = (reinterpret_cast<uintptr_t>(p.q_w) | reinterpret_cast<uintptr_t>(p.k_w)) % 16 == 0;
  }
  if (B > 65535 || T > (int64_t(1) << 20)) return fail(SAF_EUNSUPPORTED, "paged_append: at most 65535 sequences and 2^20 tokens");
  p.v = v.data; p.v_sb = v.stride[0]; p.v_sh = v.stride[1]; p.v_st = v.stride[2];
  p.vc = vc.data; p.vc_sp = vc.stride[0]; p.vc_sh = vc.stride[1]; p.vc_st = vc.stride[2];
  p.table = reinterpret_cast<const int32_t*>(a->page_table.data); p.t_sb = a->page_table.stride[0];
  p.positions = reinterpret_cast<const int32_t*>(a->positions.data);
  p.counts = present(a->counts) ? reinterpret_cast<const int32_t*>(a->counts.data) : nullptr;
  p.page_shift = page_shift_of(vc.size[2]);
  p.n_pages = (int)vc.size[0];
  p.B = (int)B; p.T = (int)T; p.Hv = (int)v.size[1]; p.hd = (int)hd;
  const int64_t rows = T * (p.Uq + p.Uk + p.Hv);
  if (rows > kMaxGrid) return fail(SAF_EUNSUPPORTED, "paged_append: too many rows (%lld)", (long long)rows);
  if (B == 0 || rows == 0) return SAF_OK;
  return launched(launch_paged_append(p, v.dtype, reinterpret_cast<hipStream_t>(stream)), "paged_append");
}

int64_t saf_token_logprobs_workspace_bytes(const saf_token_logprobs_args* args) {
  LogprobParams p{};
  if (plan_logprobs(args, p, true) != SAF_OK) return -1;
  return logprob_ws(p);
}

int saf_token_logprobs(const saf_token_logprobs_args* args, void* stream) {
  LogprobParams p{};
  if (int rc = plan_logprobs(args, p, true)) return rc;
  if (p.R == 0) return SAF_OK;
  const int64_t need = logprob_ws(p);
  if (need > 0) {
    if (args->workspace == nullptr || args->workspace_bytes < need)
      return fail(SAF_EWORKSPACE, "token_logprobs needs a %lld-byte workspace (got %lld)", (long long)need,
                  (long long)args->workspace_bytes);
    if (reinterpret_cast<uintptr_t>(args->workspace) % 16 != 0) return fail(SAF_EALIGN, "workspace must be 16-byte aligned");
    p.part_top = reinterpret_cast<uint64_t*>(args->workspace);
    p.part = reinterpret_cast<float*>(p.part_top + p.R * p.n_seg * p.top);
  }
  return launched(launch_token_logprobs(p, args->logits.dtype, reinterpret_cast<hipStream_t>(stream)), "token_logprobs");
}

int saf_token_logprobs_bwd(const saf_token_logprobs_args* args, const saf_tensor_t* dlogp, const saf_tensor_t* dentropy,
                           const saf_tensor_t* dlogits, void* stream) {
  LogprobParams f{};
  if (int rc = plan_logprobs(args, f, false)) return rc;
  if (dlogp == nullptr || dlogits == nullptr) return fail(SAF_EINVAL, "dlogp and dlogits are required");
  const bool ent = dentropy != nullptr && present(*dentropy);
  const saf_tensor_t* g[2] = {dlogp, ent ? dentropy : dlogp};
  for (int i = 0; i < 2; ++i)
    if (g[i]->dtype != SAF_F32 || g[i]->ndim != 1 || g[i]->size[0] != f.R || (f.R > 0 && !present(*g[i])))
      return fail(SAF_EINVAL, "dlogp and dentropy must be fp32 (R,)");
  if (ent && f.entropy == nullptr) return fail(SAF_EINVAL, "dentropy needs the forward's entropy");
  if (dlogits->ndim != 2 || dlogits->size[0] != f.R || dlogits->size[1] != f.V || dlogits->dtype != args->logits.dtype ||
      (f.R > 0 && !present(*dlogits)))
    return fail(SAF_EINVAL, "dlogits must have the logits' shape and dtype");
  if (f.V > 1 && dlogits->stride[1] != 1) return fail(SAF_EALIGN, "dlogits needs a unit column stride");
  if (f.R == 0) return SAF_OK;
  if (f.R > kMaxGrid / ((f.V + 4095) / 4096)) return fail(SAF_EUNSUPPORTED, "too many rows (%lld)", (long long)f.R);
  LogprobBwdParams p{};
  p.logits = f.logits; p.x_rs = f.x_rs; p.dx = dlogits->data; p.d_rs = dlogits->stride[0];
  p.R = f.R; p.V = f.V; p.tokens = f.tokens; p.tok_i64 = f.tok_i64; p.tok_st = f.tok_st; p.ignore = f.ignore;
  p.scale = f.scale; p.stats = f.stats; p.entropy = f.entropy;
  p.dlogp = reinterpret_cast<const float*>(dlogp->data); p.g_st = dlogp->stride[0];
  if (ent) {
    p.dent = reinterpret_cast<const float*>(dentropy->data);
    p.ge_st = dentropy->stride[0];
  }
  return launched(launch_token_logprobs_bwd(p, args->logits.dtype, reinterpret_cast<hipStream_t>(stream)),
                  "token_logprobs_bwd");
}

}  // extern "C"
