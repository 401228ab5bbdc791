// The C ABI of attention and of the norms and rotation in front of it (include/psgdk.h, level 3): argument validation, workspace
// layout and launches. Host code only; every launch goes to the caller's stream, nothing synchronizes.
#include <algorithm>
#include <cmath>

#include "attn.h"
#include "capi_util.h"
#include "rope.h"

using namespace psgdk;

namespace {

// Strides in elements: what a tile of up to 128 rows reaches stays within 32-bit byte offsets.
constexpr int64_t kMaxStride = (int64_t)1 << 21, kFar = (int64_t)1 << 40;
int64_t query_heads(const psgdk_window_attention_t* q) { return kMaxStride * 128 / std::max(q->heads, 128); }

// rows of 16-byte vectors: a base and strides that keep them aligned
int check_side(const psgdk_heads_t& t, int dt, int64_t tokens, int64_t heads, int64_t max_head_stride, const char* name, AttnSide& out) {
  if (!t.p) return fail(PSGDK_EINVAL, "%s: null device pointer", name);
  const int64_t unit = dt == PSGDK_BF16 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(t.p) & 15) return fail(PSGDK_EINVAL, "%s: 16-byte alignment", name);
  if (t.batch_stride % unit || t.token_stride % unit || t.head_stride % unit)
    return fail(PSGDK_ESHAPE, "%s: strides of whole 16 bytes", name);
  if (t.batch_stride < 0) return fail(PSGDK_ESHAPE, "%s: negative stride", name);
  if (tokens > 1) PSGDK_TRY(check_size(t.token_stride, 0, kMaxStride, name));
  if (heads > 1) PSGDK_TRY(check_size(t.head_stride, 0, max_head_stride, name));
  out = AttnSide{t.p, t.batch_stride, tokens > 1 ? t.token_stride : 0, heads > 1 ? t.head_stride : 0};
  return PSGDK_OK;
}
int check_launch(int64_t pairs, int64_t tiles, int64_t limit, const char* name) {
  if (pairs * tiles >= limit)
    return fail(PSGDK_ESHAPE, "batch * kv_heads = %lld with %lld tiles of %s each: too many for a launch", (long long)pairs, (long long)tiles, name);
  return PSGDK_OK;
}
int attn_args(const psgdk_window_attention_t* q, AttnArgs& a) {
  if (!q) return fail(PSGDK_EINVAL, "null argument block");
  PSGDK_TRY(check_dt(q->dtype, "dtype"));
  PSGDK_TRY(check_size(q->batch, 1, (int64_t)1 << 20, "batch"));
  PSGDK_TRY(check_size(q->n, 1, (int64_t)1 << 28, "n"));
  PSGDK_TRY(check_size(q->m, 1, (int64_t)1 << 28, "m"));
  PSGDK_TRY(check_size(q->kv_heads, 1, 1 << 16, "kv_heads"));
  PSGDK_TRY(check_size(q->heads, 1, 1 << 16, "heads"));
  PSGDK_TRY(check_size(q->d, 8, kAttnMaxD, "d"));
  if (q->d % 8) return fail(PSGDK_ESHAPE, "d = %d: must be a multiple of 8", q->d);
  if (q->heads % q->kv_heads) return fail(PSGDK_ESHAPE, "heads = %d: must be a multiple of kv_heads = %d", q->heads, q->kv_heads);
  if (q->window < 0) return fail(PSGDK_EINVAL, "window = %lld: must be >= 0", (long long)q->window);
  if (q->sinks < 0) return fail(PSGDK_EINVAL, "sinks = %lld: must be >= 0", (long long)q->sinks);
  if (!(q->scale > 0.f && std::isfinite(q->scale))) return fail(PSGDK_EINVAL, "scale = %g: must be positive", (double)q->scale);
  a = AttnArgs{};
  a.batch = (int)q->batch;
  a.n = (int)q->n;
  a.m = (int)q->m;
  a.kv = q->kv_heads;
  a.group = q->heads / q->kv_heads;
  a.d = q->d;
  a.dt = q->dtype;
  const int64_t rows = q->n * a.group;
  PSGDK_TRY(check_size(rows, 1, ((int64_t)1 << 31) - 256, "n * heads / kv_heads"));
  a.rows = (int)rows;
  // no row sees further back than m - 1 tokens
  a.window = (int)(q->window ? std::min<int64_t>(q->window, q->m) : q->m);
  a.sinks = (int)std::min<int64_t>(q->sinks, q->m);
  // rounded up to 31 + ceil(log2 group) fractional bits: exact quotients for rows below 2^31
  int bits = 0;
  while (((int64_t)1 << bits) < a.group) ++bits;
  a.div_shift = 31 + bits;
  a.div = (uint32_t)((((uint64_t)1 << a.div_shift) + a.group - 1) / a.group);
  a.scale = q->scale;
  a.scale2 = (float)((double)q->scale * 1.4426950408889634);
  a.lengths = q->lengths;
  a.starts = q->starts;
  a.lse = q->lse;
  a.parts = 1;
  // a launch holds less than 2^32 threads: a workgroup of 32 rows has 128 (several for one tile only where tiles are few)
  return check_launch(q->batch * a.kv, (rows + 31) / 32, (int64_t)1 << 24, "rows");
}
int attn_pointers(const psgdk_window_attention_t* q, AttnArgs& a) {
  // (a tile's rows are of several query heads, its keys of one)
  PSGDK_TRY(check_side(q->q, a.dt, q->n, q->heads, query_heads(q), "q", a.q));
  PSGDK_TRY(check_side(q->k, a.dt, q->m, q->kv_heads, kFar, "k", a.k));
  PSGDK_TRY(check_side(q->v, a.dt, q->m, q->kv_heads, kFar, "v", a.v));
  if (!q->o || (reinterpret_cast<uintptr_t>(q->o) & 15)) return fail(PSGDK_EINVAL, "o: a device pointer of 16-byte alignment");
  const int64_t sn = (int64_t)q->heads * q->d;
  a.o = AttnSide{q->o, q->n * sn, sn, q->d};
  if (reinterpret_cast<uintptr_t>(q->o_rest) & 15) return fail(PSGDK_EINVAL, "o_rest: 16-byte alignment");
  a.rest = a.dt == PSGDK_BF16 ? static_cast<bf16_t*>(q->o_rest) : nullptr;
  return PSGDK_OK;
}

// the argument checks and the kernels' argument block of both calls; `aligned` says for which vectors base and strides are
struct Aligned {
  bool by16 = true, by8 = true;
  void add(const void* p, const int64_t (&s)[3], size_t e) {
    const uintptr_t all = reinterpret_cast<uintptr_t>(p) | s[0] * e | s[1] * e | s[2] * e;
    by16 = by16 && !(all & 15);
    by8 = by8 && !(all & 7);
  }
};
RopeSide rope_side(const psgdk_heads_t& t, int64_t batch, int64_t tokens, int64_t heads, int dt, Aligned& al) {
  const int64_t s[3] = {batch > 1 ? t.batch_stride : 0, tokens > 1 ? t.token_stride : 0, heads > 1 ? t.head_stride : 0};
  if (t.p) al.add(t.p, s, esize(dt));
  return RopeSide{t.p, s[0], s[1], s[2]};
}
int rope_args(const psgdk_qk_norm_rope_t* q, RopeArgs& a, Aligned& al) {
  if (!q) return fail(PSGDK_EINVAL, "null argument block");
  PSGDK_TRY(check_dt(q->dtype, "dtype"));
  PSGDK_TRY(check_size(q->batch, 1, (int64_t)1 << 30, "batch"));
  PSGDK_TRY(check_size(q->n, 1, (int64_t)1 << 30, "n"));
  PSGDK_TRY(check_size(q->batch * q->n, 1, (int64_t)1 << 30, "batch * n"));
  PSGDK_TRY(check_size(q->heads, 1, 1 << 16, "heads"));
  PSGDK_TRY(check_size(q->kv_heads, 0, 1 << 16, "kv_heads"));
  PSGDK_TRY(check_size(q->d, 2, kRopeMaxD, "d"));
  PSGDK_TRY(check_size(q->rotary_dim, 0, q->d, "rotary_dim"));
  if (q->d % 2 || q->rotary_dim % 2) return fail(PSGDK_ESHAPE, "d = %d, rotary_dim = %d: must be even", q->d, q->rotary_dim);
  if (q->norm < PSGDK_NORM_NONE || q->norm > PSGDK_NORM_LAYER) return fail(PSGDK_EINVAL, "norm = %d", q->norm);
  if (!(q->eps >= 0.f)) return fail(PSGDK_EINVAL, "eps = %g: must be >= 0", (double)q->eps);
  if (!(q->theta >= 1.0 && std::isfinite(q->theta))) return fail(PSGDK_EINVAL, "theta = %g: must be at least 1", q->theta);
  if (q->norm == PSGDK_NORM_NONE && (q->q_w || q->k_w)) return fail(PSGDK_EINVAL, "weight of a norm that has none");
  if (q->q_w || q->k_w) PSGDK_TRY(check_dt(q->w_dtype, "w_dtype"));
  if (!q->q.p || (q->kv_heads && !q->k.p)) return fail(PSGDK_EINVAL, "q, k: null device pointer");
  if (!q->kv_heads && q->k_w) return fail(PSGDK_EINVAL, "k_w needs keys");
  a = RopeArgs{};
  a.tokens = q->batch * q->n;
  a.n = (int)q->n;
  a.heads = q->heads;
  a.all = q->heads + q->kv_heads;
  a.d = q->d;
  a.rot = q->rotary_dim;
  a.dt = q->dtype;
  a.norm = q->norm;
  a.eps = q->eps;
  a.pos = q->positions;
  a.pos_sb = q->positions_stride;
  // (squared in 64 bits of mantissa, so that each power is the nearest double: squared as doubles the 2^7th is 2^7 roundings off)
  long double p = q->rotary_dim ? std::pow((long double)q->theta, -2.0L / q->rotary_dim) : 1.0L;
  for (int k = 0; k < kRopePowers; ++k, p *= p) a.ratio[k] = (double)p;
  a.interleaved = q->interleaved != 0;
  a.x[0] = rope_side(q->q, q->batch, q->n, q->heads, a.dt, al);
  if (q->kv_heads) a.x[1] = rope_side(q->k, q->batch, q->n, q->kv_heads, a.dt, al);
  a.w[0] = Vec{q->q_w, q->w_dtype};
  a.w[1] = Vec{q->k_w, q->w_dtype};
  const int64_t none[3] = {0, 0, 0};
  for (const void* w : {q->q_w, q->k_w})
    if (w) al.add(w, none, 1);
  return PSGDK_OK;
}

}  // namespace

extern "C" {

int psgdk_qk_norm_rope(const psgdk_qk_norm_rope_t* q, void* qo, void* ko, psgdk_stream_t stream) {
  RopeArgs a;
  Aligned al;
  PSGDK_TRY(rope_args(q, a, al));
  if (!qo || (q->kv_heads && !ko)) return fail(PSGDK_EINVAL, "qo, ko: null device pointer");
  a.y[0] = qo;
  a.y[1] = ko;
  const int64_t none[3] = {0, 0, 0};
  for (const void* p : {qo, ko})
    if (p) al.add(p, none, 1);
  rope_plan(a, false, al.by16, al.by8);
  return hip_check(rope_launch(a, false, (hipStream_t)stream), "qk_norm_rope");
}

int psgdk_qk_norm_rope_backward(const psgdk_qk_norm_rope_t* q, const psgdk_qk_norm_rope_grads_t* g, void* ws, size_t* ws_bytes,
                                psgdk_stream_t stream) {
  RopeArgs a;
  Aligned al;
  PSGDK_TRY(rope_args(q, a, al));
  if (!g) return fail(PSGDK_EINVAL, "null gradient block");
  if (!ws_bytes) return fail(PSGDK_EINVAL, "ws_bytes is null");
  if ((g->dqw && !q->q_w) || (g->dkw && !q->k_w)) return fail(PSGDK_EINVAL, "gradient of a weight that is absent");
  if (g->dk && !q->kv_heads) return fail(PSGDK_EINVAL, "gradient of keys that are absent");
  a.dy[0] = rope_side(g->dqo, q->batch, q->n, q->heads, a.dt, al);
  if (q->kv_heads) a.dy[1] = rope_side(g->dko, q->batch, q->n, q->kv_heads, a.dt, al);
  a.dx[0] = g->dq;
  a.dx[1] = g->dk;
  const int64_t none[3] = {0, 0, 0};
  for (const void* p : {g->dq, g->dk})
    if (p) al.add(p, none, 1);
  rope_plan(a, true, al.by16, al.by8);
  const bool sums = g->dqw || g->dkw;
  Ws m(ws);
  if (sums) a.part = m.take<float>((size_t)2 * kRopeParts * a.d);  // (the parts go by alignment: room for the most there are)
  if (!ws) {
    *ws_bytes = m.off;
    return PSGDK_OK;
  }
  if (*ws_bytes < m.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *ws_bytes, m.off);
  if (!g->dq && !g->dk && !sums) return PSGDK_OK;
  PSGDK_TRY(hip_check(rope_launch(a, true, (hipStream_t)stream), "qk_norm_rope backward"));
  if (!sums) return PSGDK_OK;
  ColumnSums s{};
  s.d = a.d;
  void* const out[2] = {g->dqw, g->dkw};
  for (int k = 0; k < 2; ++k) {
    if (!out[k]) continue;
    auto& e = s.e[s.n++];
    e.in = a.part + (size_t)k * a.parts * a.d;
    e.out = out[k];
    e.dt = q->w_dtype;
    e.groups = 1;
    e.per = a.parts;
    e.ldo = a.d;
  }
  return hip_check(column_sums_launch(s, (hipStream_t)stream), "column sums");
}

int psgdk_window_attention(const psgdk_window_attention_t* q, void* ws, size_t* ws_bytes, psgdk_stream_t stream) {
  AttnArgs a;
  PSGDK_TRY(attn_args(q, a));
  if (!ws_bytes) return fail(PSGDK_EINVAL, "ws_bytes is null");
  a.parts = attn_parts(a);
  Ws m(ws);
  if (a.parts > 1) {
    const size_t rows = (size_t)a.parts * a.batch * a.kv * a.rows;
    a.part_o = m.take<float>(rows * a.d);
    a.part_ml = m.take<float>(rows * 2);
  }
  if (!ws) {
    *ws_bytes = m.off;
    return PSGDK_OK;
  }
  if (*ws_bytes < m.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *ws_bytes, m.off);
  PSGDK_TRY(attn_pointers(q, a));
  return hip_check(attn_forward_launch(a, (hipStream_t)stream), "attention");
}

int psgdk_window_attention_backward(const psgdk_window_attention_t* q, const psgdk_window_attention_grads_t* g, void* ws,
                                    size_t* ws_bytes, psgdk_stream_t stream) {
  AttnArgs a;
  PSGDK_TRY(attn_args(q, a));
  if (!g) return fail(PSGDK_EINVAL, "null gradient block");
  if (!ws_bytes) return fail(PSGDK_EINVAL, "ws_bytes is null");
  PSGDK_TRY(check_launch(q->batch * a.kv, (q->m + kAttnKeys - 1) / kAttnKeys, (int64_t)1 << 23, "keys"));  // (256 threads each)
  attn_backward_parts(a);
  a.dq = g->dq;
  a.dk = g->dk;
  a.dv = g->dv;
  Ws m(ws);
  a.delta = m.take<float>((size_t)a.batch * a.kv * a.rows);
  a.row_pos = m.take<int>((size_t)a.batch * a.kv * a.rows);
  if (a.dk || a.dv) a.part_kv = m.take<float>((size_t)attn_part_tiles(a) * 2 * kAttnKeys * attn_dp(a.d));
  if (!ws) {
    *ws_bytes = m.off;
    return PSGDK_OK;
  }
  if (*ws_bytes < m.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *ws_bytes, m.off);
  PSGDK_TRY(attn_pointers(q, a));
  PSGDK_TRY(check_side(g->dout, a.dt, q->n, q->heads, query_heads(q), "dout", a.dout));
  if (!a.lse) return fail(PSGDK_EINVAL, "lse: null device pointer");
  for (const void* p : {(const void*)a.dq, (const void*)a.dk, (const void*)a.dv})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(PSGDK_EINVAL, "dq, dk, dv: 16-byte alignment");
  PSGDK_TRY(hip_check(attn_dq_launch(a, (hipStream_t)stream), "attention dq"));
  if (!a.dk && !a.dv) return PSGDK_OK;
  return hip_check(attn_dkv_launch(a, (hipStream_t)stream), "attention dk, dv");
}

}  // extern "C"
