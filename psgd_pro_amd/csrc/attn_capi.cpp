// The C ABI of attention (include/psgdk.h, level 3): argument validation, workspace layout and launches. Host code only; every
// launch goes to the caller's stream, nothing synchronizes.
#include <algorithm>
#include <cmath>

#include "attn.h"
#include "capi_util.h"

using namespace psgdk;

namespace {

// Strides in elements: what a tile of up to 128 rows reaches stays within 32-bit byte offsets.
constexpr int64_t kMaxStride = (int64_t)1 << 21;

// rows of 16-byte vectors: a base and strides that keep them aligned
int check_side(const psgdk_heads_t& t, int dt, int64_t tokens, int64_t heads, const char* name, AttnSide& out) {
  if (!t.p) return fail(PSGDK_EINVAL, "%s: null device pointer", name);
  const int64_t unit = dt == PSGDK_BF16 ? 8 : 4;
  if (reinterpret_cast<uintptr_t>(t.p) & 15) return fail(PSGDK_EINVAL, "%s: 16-byte alignment", name);
  if (t.batch_stride % unit || t.token_stride % unit || t.head_stride % unit)
    return fail(PSGDK_ESHAPE, "%s: strides of whole 16 bytes", name);
  if (t.batch_stride < 0) return fail(PSGDK_ESHAPE, "%s: negative stride", name);
  if (tokens > 1) PSGDK_TRY(check_size(t.token_stride, 0, kMaxStride, name));
  if (heads > 1) PSGDK_TRY(check_size(t.head_stride, 0, kMaxStride * 128 / std::max<int64_t>(heads, 128), name));
  out = AttnSide{t.p, t.batch_stride, tokens > 1 ? t.token_stride : 0, heads > 1 ? t.head_stride : 0};
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
  // A launch holds less than 2^32 threads: a forward workgroup of 32 rows has 128, one of 128 keys backward 256. (More than one
  // for a tile of keys or rows there are only where the tiles are few.)
  const int64_t pairs = q->batch * a.kv;
  a.parts = 1;
  if (pairs * ((rows + 31) / 32) >= (int64_t)1 << 24 || pairs * ((q->m + 127) / 128) >= (int64_t)1 << 23)
    return fail(PSGDK_ESHAPE, "batch * kv_heads = %lld with %lld rows and %lld keys each: too many for a launch", (long long)pairs,
                (long long)rows, (long long)q->m);
  return PSGDK_OK;
}
int attn_pointers(const psgdk_window_attention_t* q, AttnArgs& a) {
  PSGDK_TRY(check_side(q->q, a.dt, q->n, q->heads, "q", a.q));
  PSGDK_TRY(check_side(q->k, a.dt, q->m, q->kv_heads, "k", a.k));
  PSGDK_TRY(check_side(q->v, a.dt, q->m, q->kv_heads, "v", a.v));
  if (!q->o || (reinterpret_cast<uintptr_t>(q->o) & 15)) return fail(PSGDK_EINVAL, "o: a device pointer of 16-byte alignment");
  const int64_t sn = (int64_t)q->heads * q->d;
  a.o = AttnSide{q->o, q->n * sn, sn, q->d};
  return PSGDK_OK;
}

}  // namespace

extern "C" {

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
  attn_backward_parts(a);
  a.dq = g->dq;
  a.dk = g->dk;
  a.dv = g->dv;
  Ws m(ws);
  a.delta = m.take<float>((size_t)a.batch * a.kv * a.rows);
  if (a.dk || a.dv) a.part_kv = m.take<float>((size_t)attn_part_tiles(a) * 2 * kAttnKeys * attn_dp(a.d));
  if (!ws) {
    *ws_bytes = m.off;
    return PSGDK_OK;
  }
  if (*ws_bytes < m.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *ws_bytes, m.off);
  PSGDK_TRY(attn_pointers(q, a));
  PSGDK_TRY(check_side(g->dout, a.dt, q->n, q->heads, "dout", a.dout));
  if (!a.lse) return fail(PSGDK_EINVAL, "lse: null device pointer");
  for (const void* p : {(const void*)a.dq, (const void*)a.dk, (const void*)a.dv})
    if (reinterpret_cast<uintptr_t>(p) & 15) return fail(PSGDK_EINVAL, "dq, dk, dv: 16-byte alignment");
  PSGDK_TRY(hip_check(attn_dq_launch(a, (hipStream_t)stream), "attention dq"));
  if (!a.dk && !a.dv) return PSGDK_OK;
  return hip_check(attn_dkv_launch(a, (hipStream_t)stream), "attention dk, dv");
}

}  // extern "C"
