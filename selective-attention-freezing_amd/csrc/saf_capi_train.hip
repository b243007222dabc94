// Host side of the operators around the products of a training step: embedding,
// residual LayerNorm, 8-bit activations.  Argument checks and launches of the
// C-ABI in include/saf_attn.h; nothing here allocates or throws.
#include <cmath>

#include "saf_host.h"

using namespace saf;

namespace {

constexpr int64_t kMaxUnits = 0x7fffffff;
constexpr int64_t kMaxC = int64_t(1) << 23;
constexpr int64_t kMaxThreads = (int64_t(1) << 32) - 1024;  // of a launch, whose workgroups have 1024 at most
constexpr int64_t kMaxTokens = int64_t(1) << 28;             // of an embedding's gradient

bool float_dtype(int d) { return d == SAF_F32 || d == SAF_F16 || d == SAF_BF16; }
bool given(const saf_tensor_t* t) { return t != nullptr && t->ndim > 0; }

// Rows (R, C) with a unit column stride; contiguous where asked.
int check_rows(const saf_tensor_t* t, const char* name, int64_t R, int64_t C, bool packed) {
  if (!given(t)) return fail(SAF_EINVAL, "%s is required", name);
  if (t->ndim != 2 || t->size[0] != R || t->size[1] != C)
    return fail(SAF_EINVAL, "%s must be (%lld, %lld)", name, (long long)R, (long long)C);
  if (R > 0 && C > 0 && !present(*t)) return fail(SAF_EINVAL, "%s is required", name);
  if (C > 1 && t->stride[1] != 1) return fail(SAF_EALIGN, "%s needs a unit column stride", name);
  if (packed && R > 1 && t->stride[0] != C) return fail(SAF_EALIGN, "%s must be contiguous", name);
  if (present(*t) && reinterpret_cast<uintptr_t>(t->data) % elem_size(t->dtype))
    return fail(SAF_EALIGN, "%s is not aligned to its elements", name);
  return SAF_OK;
}

int check_vec(const saf_tensor_t* t, const char* name, int64_t C, int dtype) {
  if (!given(t) || !present(*t) || t->ndim != 1 || t->size[0] != C || !float_dtype(t->dtype) || (C > 1 && t->stride[0] != 1) ||
      (dtype >= 0 && t->dtype != dtype))
    return fail(SAF_EINVAL, "%s must be a contiguous floating (%lld,) vector%s", name, (long long)C,
                dtype >= 0 ? " of the weight's dtype" : "");
  return SAF_OK;
}

int check_float(const saf_tensor_t* t, const char* name) {
  if (!given(t)) return fail(SAF_EINVAL, "%s is required", name);
  if (!float_dtype(t->dtype)) return fail(SAF_EUNSUPPORTED, "%s: unsupported dtype %s", name, dtype_name(t->dtype));
  return SAF_OK;
}

int check_workspace(const char* what, const void* ws, int64_t bytes, int64_t need) {
  if (need <= 0) return SAF_OK;
  if (ws == nullptr || bytes < need)
    return fail(SAF_EWORKSPACE, "%s needs a %lld-byte workspace (got %lld)", what, (long long)need, (long long)bytes);
  if (reinterpret_cast<uintptr_t>(ws) % 256 != 0) return fail(SAF_EALIGN, "workspace must be 256-byte aligned");
  return SAF_OK;
}

hipStream_t stream_of(void* s) { return reinterpret_cast<hipStream_t>(s); }

// Two of the three types in one operator: the same, or fp32 beside another.
bool types_meet(int a, int b) { return a == b || a == SAF_F32 || b == SAF_F32; }

// Units of 8 channels of R rows.
int units_of(const char* what, int64_t R, int64_t per_row, FastDiv& div, uint32_t& units) {
  if (per_row > kMaxUnits || R > kMaxUnits / (per_row ? per_row : 1))
    return fail(SAF_EUNSUPPORTED, "%s: more than 2^31 groups of 8 channels", what);
  div = FastDiv::of((uint32_t)per_row);
  units = (uint32_t)(R * per_row);
  return SAF_OK;
}

// ---- embedding -----------------------------------------------------------------

int check_tokens(const saf_tensor_t* t) {
  if (!given(t) || t->ndim != 1 || (t->dtype != SAF_I32 && t->dtype != SAF_I64))
    return fail(SAF_EINVAL, "tokens must be int32 or int64 (N,)");
  if (t->size[0] > 0 && !present(*t)) return fail(SAF_EINVAL, "tokens are required");
  return SAF_OK;
}

int check_table(int64_t V, int64_t C) {
  if (V < 1 || C < 1) return fail(SAF_EINVAL, "the embedding must have rows and channels");
  if (V >= kMaxUnits || C > kMaxC) return fail(SAF_EUNSUPPORTED, "an embedding of 2^31 rows, or of more than 2^23 channels");
  return SAF_OK;
}

// The plan of a gradient of N tokens: how they are sorted and where the parts of
// the workspace are.
struct EmbedPlan {
  int n_tiles, passes, bits, chunk;
  int64_t n_chunks, at_sorted2, at_counts, at_head, at_tail, bytes;
};

// Positions per chunk: as many as leave the card 1024 waves, from 16 to 64.  Longer
// chunks cut fewer words in two, shorter ones fill the card: the sums and the joining
// of their parts together took, for 2048 waves at least and for 1024, 16 and 15 us for
// 16384 tokens of a natural distribution at 768 channels, 25 and 20 for 32768, 35 and
// 31 for 65536.
int chunk_of(int64_t N, int64_t C) {
  const int64_t waves = (N + 63) / 64 * ((C + 255) / 256);
  return waves >= 1024 ? 64 : (waves >= 512 ? 32 : 16);
}

int64_t up256(int64_t n) { return (n + 255) / 256 * 256; }

EmbedPlan embed_plan(int64_t N, int64_t V, int64_t C) {
  EmbedPlan e{};
  if (N <= kEmbedFew) return e;
  e.n_tiles = (int)((N + kEmbedTile - 1) / kEmbedTile);
  int key_bits = 1;  // of the words and of the key behind them, V
  while ((V >> key_bits) != 0) ++key_bits;
  e.passes = (key_bits + kEmbedDigit - 1) / kEmbedDigit;
  e.bits = (key_bits + e.passes - 1) / e.passes;
  e.chunk = chunk_of(N, C);
  e.n_chunks = (N + e.chunk - 1) / e.chunk;
  int64_t at = up256(8 * N);
  e.at_sorted2 = at;
  if (N > kEmbedOnce && e.passes > 1) at += up256(8 * N);
  e.at_counts = at;
  if (N >= kEmbedCounted) at += up256(4 * ((int64_t)(e.n_tiles + 1) << kEmbedDigit));
  e.at_head = at;
  if (e.n_chunks > 1) at += up256(4 * e.n_chunks * C);
  e.at_tail = at;
  if (e.n_chunks > 1) at += up256(4 * e.n_chunks * C);
  e.bytes = at;
  return e;
}

// ---- 8-bit activations ------------------------------------------------------------

int pack_params(const char* what, const saf_tensor_t* x, const char* x_name, const saf_tensor_t* q, const saf_tensor_t* exp,
                ActPackParams& p, bool held = true) {
  if (int rc = check_float(x, x_name)) return rc;
  if (x->ndim != 2) return fail(SAF_EINVAL, "%s must be 2-D (rows, C)", x_name);
  const int64_t R = x->size[0], C = x->size[1];
  if (C < 1 || C > kMaxC) return fail(SAF_EUNSUPPORTED, "%s: C = %lld is not supported (1 to 2^23)", what, (long long)C);
  if (int rc = check_rows(x, x_name, R, C, false)) return rc;
  const int64_t nb = (C + 31) / 32;
  if (held) {
    if (int rc = check_rows(q, "q", R, C, true)) return rc;
    if (int rc = check_rows(exp, "exp", R, nb, true)) return rc;
    if (q->dtype != SAF_I8 || exp->dtype != SAF_U8) return fail(SAF_EINVAL, "q must be int8 and exp uint8");
    p.q = reinterpret_cast<int8_t*>(q->data);
    p.exp = reinterpret_cast<uint8_t*>(exp->data);
  }
  if (int rc = units_of(what, R, 4 * nb, p.per_row, p.units)) return rc;
  p.x = x->data;
  p.x_rs = x->stride[0];
  p.C = (int)C;
  return SAF_OK;
}

int run_pack(const char* what, const ActPackParams& p, int dtype, ActPackOp op, void* stream) {
  if (p.units == 0) return SAF_OK;
  return launched(launch_act_pack(p, dtype, op, stream_of(stream)), what);
}

}  // namespace

extern "C" {

int saf_embed_fwd(const saf_tensor_t* tokens, const saf_tensor_t* weight, float scale, int64_t ignore_index,
                  const saf_tensor_t* out, void* stream) {
  if (int rc = check_tokens(tokens)) return rc;
  if (int rc = check_float(weight, "weight")) return rc;
  if (int rc = check_float(out, "out")) return rc;
  if (weight->ndim != 2) return fail(SAF_EINVAL, "weight must be (V, C)");
  const int64_t N = tokens->size[0], V = weight->size[0], C = weight->size[1];
  if (int rc = check_table(V, C)) return rc;
  if (int rc = check_rows(weight, "weight", V, C, false)) return rc;
  if (int rc = check_rows(out, "out", N, C, true)) return rc;
  if (!types_meet(weight->dtype, out->dtype)) return fail(SAF_EUNSUPPORTED, "embed: bf16 beside fp16");
  EmbedParams p{};
  if (int rc = units_of("embed", N, (C + 7) / 8, p.per_row, p.units)) return rc;
  if (N == 0) return SAF_OK;
  p.tokens = tokens->data;
  p.tok_i64 = tokens->dtype == SAF_I64;
  p.tok_st = tokens->stride[0];
  p.ignore = ignore_index;
  p.V = V;
  p.w = weight->data;
  p.w_rs = weight->stride[0];
  p.y = out->data;
  p.scale = scale;
  p.C = (int)C;
  return launched(launch_embed(p, weight->dtype, out->dtype, stream_of(stream)), "embed");
}

int64_t saf_embed_bwd_workspace_bytes(int64_t n_tokens, int64_t vocab, int64_t channels) {
  if (n_tokens < 0 || n_tokens > kMaxTokens) {
    fail(SAF_EUNSUPPORTED, "embed_bwd: %lld tokens (at most 2^28)", (long long)n_tokens);
    return -1;
  }
  if (check_table(vocab, channels) != SAF_OK) return -1;
  return embed_plan(n_tokens, vocab, channels).bytes;
}

int saf_embed_bwd(const saf_tensor_t* tokens, const saf_tensor_t* dout, float scale, int64_t ignore_index,
                  const saf_tensor_t* dweight, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_tokens(tokens)) return rc;
  if (int rc = check_float(dweight, "dweight")) return rc;
  if (int rc = check_float(dout, "dout")) return rc;
  if (dweight->ndim != 2) return fail(SAF_EINVAL, "dweight must be (V, C)");
  const int64_t N = tokens->size[0], V = dweight->size[0], C = dweight->size[1];
  if (int rc = check_table(V, C)) return rc;
  if (N > kMaxTokens) return fail(SAF_EUNSUPPORTED, "embed_bwd: %lld tokens (at most 2^28)", (long long)N);
  if (int rc = check_rows(dweight, "dweight", V, C, true)) return rc;
  if (reinterpret_cast<uintptr_t>(dweight->data) % 16 != 0) return fail(SAF_EALIGN, "dweight must be 16-byte aligned");
  if (int rc = check_rows(dout, "dout", N, C, false)) return rc;
  if (!types_meet(dweight->dtype, dout->dtype)) return fail(SAF_EUNSUPPORTED, "embed: bf16 beside fp16");
  const EmbedPlan e = embed_plan(N, V, C);
  EmbedBwdParams p{};
  if (int rc = units_of("embed", e.n_chunks, (C + 255) / 256, p.per_row, p.units)) return rc;
  if (p.units > kMaxThreads / 64) return fail(SAF_EUNSUPPORTED, "embed_bwd: too many tokens of %lld channels", (long long)C);
  if (int rc = check_workspace("embed_bwd", workspace, workspace_bytes, e.bytes)) return rc;
  char* ws = reinterpret_cast<char*>(workspace);
  p.tokens = tokens->data;
  p.tok_i64 = tokens->dtype == SAF_I64;
  p.tok_st = tokens->stride[0];
  p.ignore = ignore_index;
  p.V = V;
  p.N = N;
  p.dy = dout->data;
  p.dy_rs = dout->stride[0];
  p.dw = dweight->data;
  p.dw_bytes = V * C * elem_size(dweight->dtype);
  p.scale = scale;
  p.C = (int)C;
  p.sorted = reinterpret_cast<uint2*>(ws);
  p.sorted2 = reinterpret_cast<uint2*>(ws + e.at_sorted2);
  p.counts = N >= kEmbedCounted ? reinterpret_cast<uint32_t*>(ws + e.at_counts) : nullptr;
  p.head = reinterpret_cast<float*>(ws + e.at_head);
  p.tail = reinterpret_cast<float*>(ws + e.at_tail);
  p.n_tiles = e.n_tiles;
  p.passes = e.passes;
  p.bits = e.bits;
  p.chunk = e.chunk;
  // workgroups that clear: 64 KB each, 16 of a few tokens', at most one a CU
  const int64_t part = N <= kEmbedFew ? 16384 : 65536, want = (p.dw_bytes + part - 1) / part;
  p.n_clear = (int)(want < cu_count() ? want : cu_count());
  return launched(launch_embed_bwd(p, dweight->dtype, dout->dtype, stream_of(stream)), "embed_bwd");
}

int saf_layernorm_fwd(const saf_tensor_t* x, const saf_tensor_t* delta, const saf_tensor_t* weight,
                      const saf_tensor_t* bias, float eps, const saf_tensor_t* r, const saf_tensor_t* y,
                      const saf_tensor_t* stats, void* stream) {
  if (int rc = check_float(x, "x")) return rc;
  if (int rc = check_float(y, "y")) return rc;
  if (x->ndim != 2) return fail(SAF_EINVAL, "x must be 2-D (rows, C)");
  const int64_t R = x->size[0], C = x->size[1];
  if (C < 1 || C > kLnMaxC) return fail(SAF_EUNSUPPORTED, "layernorm: C = %lld is not supported (1 to %d)", (long long)C, kLnMaxC);
  if (R > kMaxThreads / layernorm_row_threads((int)C))
    return fail(SAF_EUNSUPPORTED, "layernorm: too many rows (%lld) of %lld channels", (long long)R, (long long)C);
  if (int rc = check_rows(x, "x", R, C, false)) return rc;
  if (int rc = check_rows(y, "y", R, C, true)) return rc;
  if (y->dtype != x->dtype && x->dtype != SAF_F32)
    return fail(SAF_EUNSUPPORTED, "layernorm: %s x with %s y", dtype_name(x->dtype), dtype_name(y->dtype));
  if (given(delta) != given(r)) return fail(SAF_EINVAL, "delta and r go together");
  if (given(delta)) {
    if (int rc = check_rows(delta, "delta", R, C, false)) return rc;
    if (int rc = check_rows(r, "r", R, C, true)) return rc;
    if (delta->dtype != y->dtype || r->dtype != x->dtype)
      return fail(SAF_EINVAL, "r must have x's dtype and delta y's");
  }
  if (int rc = check_vec(weight, "weight", C, -1)) return rc;
  if (given(bias))
    if (int rc = check_vec(bias, "bias", C, weight->dtype)) return rc;
  if (given(stats)) {
    if (int rc = check_rows(stats, "stats", R, 2, true)) return rc;
    if (stats->dtype != SAF_F32) return fail(SAF_EINVAL, "stats must be fp32");
  }
  if (!(eps >= 0.f)) return fail(SAF_EINVAL, "eps must be a non-negative number");
  if (R == 0) return SAF_OK;
  LnTrainParams p{};
  p.x = x->data;
  p.x_rs = x->stride[0];
  if (given(delta)) {
    p.delta = delta->data;
    p.d_rs = delta->stride[0];
    p.r = r->data;
  }
  p.y = y->data;
  p.w = weight->data;
  p.b = given(bias) ? bias->data : nullptr;
  p.wb_dtype = weight->dtype;
  p.stats = given(stats) ? reinterpret_cast<float*>(stats->data) : nullptr;
  p.rows = R;
  p.C = (int)C;
  p.eps = eps;
  return launched(launch_layernorm_train(p, x->dtype, y->dtype, stream_of(stream)), "layernorm");
}

int64_t saf_layernorm_bwd_workspace_bytes(int64_t rows, int64_t channels) {
  if (rows < 0 || rows > kMaxUnits || channels < 1 || channels > kLnMaxC) {
    fail(SAF_EINVAL, "layernorm: rows of %lld channels are not supported", (long long)channels);
    return -1;
  }
  const int n_wg = rows == 0 ? 0 : layernorm_bwd_groups(rows, (int)channels, cu_count());
  return n_wg > 1 ? (int64_t)n_wg * 2 * channels * 4 : 0;
}

int saf_layernorm_bwd(const saf_tensor_t* r, const saf_tensor_t* stats, const saf_tensor_t* weight,
                      const saf_tensor_t* dy, const saf_tensor_t* dr, const saf_tensor_t* dx,
                      const saf_tensor_t* ddelta, const saf_tensor_t* dweight, const saf_tensor_t* dbias,
                      void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_float(r, "r")) return rc;
  if (int rc = check_float(dy, "dy")) return rc;
  if (r->ndim != 2) return fail(SAF_EINVAL, "r must be 2-D (rows, C)");
  const int64_t R = r->size[0], C = r->size[1];
  const int64_t ws_bytes = saf_layernorm_bwd_workspace_bytes(R, C);
  if (ws_bytes < 0) return SAF_EUNSUPPORTED;
  if (int rc = check_rows(r, "r", R, C, false)) return rc;
  if (int rc = check_rows(dy, "dy", R, C, false)) return rc;
  if (dy->dtype != r->dtype && r->dtype != SAF_F32)
    return fail(SAF_EUNSUPPORTED, "layernorm: %s r with %s dy", dtype_name(r->dtype), dtype_name(dy->dtype));
  if (int rc = check_rows(stats, "stats", R, 2, true)) return rc;
  if (stats->dtype != SAF_F32) return fail(SAF_EINVAL, "stats must be fp32");
  if (int rc = check_vec(weight, "weight", C, -1)) return rc;
  const saf_tensor_t* same[2] = {dr, dx};
  for (int i = 0; i < 2; ++i)
    if (given(same[i])) {
      if (int rc = check_rows(same[i], i ? "dx" : "dr", R, C, i == 1)) return rc;
      if (same[i]->dtype != r->dtype) return fail(SAF_EINVAL, "dr and dx must have r's dtype");
    }
  if (given(ddelta)) {
    if (int rc = check_rows(ddelta, "ddelta", R, C, true)) return rc;
    if (ddelta->dtype != dy->dtype) return fail(SAF_EINVAL, "ddelta must have dy's dtype");
  }
  const saf_tensor_t* vecs[2] = {dweight, dbias};
  for (int i = 0; i < 2; ++i)
    if (given(vecs[i]))
      if (int rc = check_vec(vecs[i], i ? "dbias" : "dweight", C, weight->dtype)) return rc;
  LnTrainBwdParams p{};
  p.dw = given(dweight) ? dweight->data : nullptr;
  p.db = given(dbias) ? dbias->data : nullptr;
  if (R == 0 && !p.dw && !p.db) return SAF_OK;
  if (p.dw || p.db) {
    if (int rc = check_workspace("layernorm_bwd", workspace, workspace_bytes, ws_bytes)) return rc;
    if (ws_bytes > 0) p.part = reinterpret_cast<float*>(workspace);
  }
  p.r = r->data;
  p.r_rs = r->stride[0];
  p.dy = dy->data;
  p.dy_rs = dy->stride[0];
  if (given(dr)) {
    p.dr = dr->data;
    p.dr_rs = dr->stride[0];
  }
  auto al16 = [](const saf_tensor_t& t) {
    return reinterpret_cast<uintptr_t>(t.data) % 16 == 0 && (t.size[0] <= 1 || t.stride[0] * elem_size(t.dtype) % 16 == 0);
  };
  p.once = al16(*dy) && (!given(dr) || al16(*dr));
  p.dx = given(dx) ? dx->data : nullptr;
  p.ddelta = given(ddelta) ? ddelta->data : nullptr;
  p.w = weight->data;
  p.w_dtype = weight->dtype;
  p.stats = reinterpret_cast<const float*>(stats->data);
  p.rows = R;
  p.C = (int)C;
  p.n_wg = R > 0 ? layernorm_bwd_groups(R, (int)C, cu_count()) : 0;  // no rows: empty sums
  return launched(launch_layernorm_train_bwd(p, r->dtype, dy->dtype, stream_of(stream)), "layernorm_bwd");
}

int saf_act_pack(const saf_tensor_t* x, const saf_tensor_t* q, const saf_tensor_t* exp, void* stream) {
  ActPackParams p{};
  if (int rc = pack_params("act_pack", x, "x", q, exp, p)) return rc;
  return run_pack("act_pack", p, x->dtype, ActPackOp::kPack, stream);
}

int saf_act_unpack(const saf_tensor_t* q, const saf_tensor_t* exp, const saf_tensor_t* out, void* stream) {
  ActPackParams p{};
  if (int rc = pack_params("act_unpack", out, "out", q, exp, p)) return rc;
  if (out->size[0] > 1 && out->stride[0] < out->size[1]) return fail(SAF_EINVAL, "out has rows that overlap");
  p.y = out->data;
  p.y_rs = out->stride[0];
  return run_pack("act_unpack", p, out->dtype, ActPackOp::kUnpack, stream);
}

int saf_gelu_pack_fwd(const saf_tensor_t* x, const saf_tensor_t* y, const saf_tensor_t* q, const saf_tensor_t* exp,
                      void* stream) {
  ActPackParams p{};
  const bool held = given(q) || given(exp);
  if (int rc = pack_params("gelu_pack", x, "x", q, exp, p, held)) return rc;
  if (int rc = check_rows(y, "y", x->size[0], x->size[1], true)) return rc;
  if (y->dtype != x->dtype) return fail(SAF_EINVAL, "y must have x's dtype");
  p.y = y->data;
  p.y_rs = x->size[1];
  return run_pack("gelu_pack", p, x->dtype, held ? ActPackOp::kGelu : ActPackOp::kGeluOnly, stream);
}

int saf_gelu_pack_bwd(const saf_tensor_t* q, const saf_tensor_t* exp, const saf_tensor_t* dy, const saf_tensor_t* dx,
                      const saf_tensor_t* y, void* stream) {
  ActPackParams p{};
  if (int rc = pack_params("gelu_pack_bwd", dy, "dy", q, exp, p)) return rc;
  if (int rc = check_rows(dx, "dx", dy->size[0], dy->size[1], true)) return rc;
  if (dx->dtype != dy->dtype) return fail(SAF_EINVAL, "dx must have dy's dtype");
  p.dx = dx->data;
  if (given(y)) {
    if (int rc = check_rows(y, "y", dy->size[0], dy->size[1], true)) return rc;
    if (y->dtype != dy->dtype) return fail(SAF_EINVAL, "y must have dy's dtype");
    p.y = y->data;
    p.y_rs = dy->size[1];
  }
  return run_pack("gelu_pack_bwd", p, dy->dtype, ActPackOp::kGeluBwd, stream);
}

}  // extern "C"
