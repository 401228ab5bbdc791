// The C ABI of the AdamW step (include/psgdk.h, level 3): argument validation, the tensors' tables and the launches. Host code
// only; every launch goes to the caller's stream, nothing synchronizes.
#include <algorithm>
#include <cmath>

#include "adamw.h"
#include "capi_util.h"

using namespace psgdk;

namespace {

constexpr int64_t kMaxTensors = (int64_t)1 << 20;
constexpr int64_t kMaxElements = (int64_t)1 << 40;

int check_beta(double b, const char* name) {
  if (!(b >= 0.0 && b < 1.0)) return fail(PSGDK_EINVAL, "%s = %g: must be in 0..1, below 1", name, b);
  return PSGDK_OK;
}

// Calls f(table, dtype) for tables of up to kAdamTensors tensors of one dtype; a launch has less than 2^32 threads, so that a
// tensor of more chunks than that goes in several pieces of whole blocks.
template <typename F>
int each_table(const psgdk_adamw_t* q, const AdamArgs& common, F f) {
  constexpr int64_t kMost = ((int64_t)1 << 23) * kAdamChunk;  // elements of a launch: 2^23 workgroups of 256 threads
  for (int dt : {PSGDK_F32, PSGDK_BF16}) {
    AdamArgs a = common;
    int64_t chunks = 0;
    auto flush = [&]() {
      if (!a.count) return (int)PSGDK_OK;
      const int rc = f(a, dt);
      a.count = 0;
      chunks = 0;
      return rc;
    };
    for (int64_t t = 0; t < q->nb; ++t) {
      if (q->dtype[t] != dt) continue;
      for (int64_t at = 0; at < q->n[t]; at += kMost) {
        const int64_t n = std::min(q->n[t] - at, kMost), c = (n + kAdamChunk - 1) / kAdamChunk;
        if (a.count == kAdamTensors || chunks + c > kMost / kAdamChunk) PSGDK_TRY(flush());
        const int k = a.count++;
        a.first[k] = (int)chunks;
        a.first[k + 1] = (int)(chunks += c);
        a.index[k] = (int)t;
        a.n[k] = n;
        a.at[k] = at;
        a.g[k] = static_cast<const char*>(q->g[t]) + at * esize(dt);
        if (!q->p) continue;
        const size_t e = q->bits == 32 ? 4 : 1;
        a.p[k] = static_cast<char*>(q->p[t]) + at * esize(dt);
        a.m[k] = static_cast<char*>(q->m[t]) + at * e;
        a.v[k] = static_cast<char*>(q->v[t]) + at * e;
        if (q->bits == 8) {
          a.ms[k] = static_cast<uint8_t*>(q->m_scale[t]) + at / kAdamBlock;
          a.vs[k] = static_cast<uint8_t*>(q->v_scale[t]) + at / kAdamBlock;
        }
      }
    }
    PSGDK_TRY(flush());
  }
  return PSGDK_OK;
}

}  // namespace

extern "C" {

int psgdk_adamw(const psgdk_adamw_t* q, void* ws, size_t* ws_bytes, psgdk_stream_t stream) {
  if (!q) return fail(PSGDK_EINVAL, "null argument block");
  if (!ws_bytes) return fail(PSGDK_EINVAL, "ws_bytes is null");
  PSGDK_TRY(check_size(q->nb, 0, kMaxTensors, "nb"));
  if (q->bits != 8 && q->bits != 32) return fail(PSGDK_EINVAL, "bits = %d: 8 or 32", q->bits);
  if (!(std::isfinite(q->lr) && std::isfinite(q->weight_decay))) return fail(PSGDK_EINVAL, "lr, weight_decay: must be finite");
  if (!(q->eps >= 0.0)) return fail(PSGDK_EINVAL, "eps = %g: must be >= 0", q->eps);
  PSGDK_TRY(check_beta(q->beta1, "beta1"));
  PSGDK_TRY(check_beta(q->beta2, "beta2"));
  PSGDK_TRY(check_size(q->step, 1, (int64_t)1 << 32, "step"));
  if (!(q->max_norm >= 0.0)) return fail(PSGDK_EINVAL, "max_norm = %g: must be >= 0", q->max_norm);
  if (q->nb && (!q->n || !q->dtype || !q->g)) return fail(PSGDK_EINVAL, "n, dtype, g: null pointer");
  if (q->nb && q->p && (!q->m || !q->v || (q->bits == 8 && (!q->m_scale || !q->v_scale))))
    return fail(PSGDK_EINVAL, "m, v or their scales: null pointer");
  const bool clip = q->p && q->max_norm > 0.0, norm = clip || q->norm;
  int64_t chunks = 0, some = 0;
  for (int64_t t = 0; t < q->nb; ++t) {
    PSGDK_TRY(check_dt(q->dtype[t], "dtype"));
    PSGDK_TRY(check_size(q->n[t], 0, kMaxElements, "n"));
    chunks += (q->n[t] + kAdamChunk - 1) / kAdamChunk;
    some += q->n[t] > 0;
    if (!q->n[t] || !ws) continue;
    if (!q->g[t] || (q->p && (!q->p[t] || !q->m[t] || !q->v[t] || (q->bits == 8 && (!q->m_scale[t] || !q->v_scale[t])))))
      return fail(PSGDK_EINVAL, "tensor %lld: null device pointer", (long long)t);
  }
  // sums of the norm's workgroups: no more than chunks, and no more than kAdamParts for each table
  const int64_t tables = 2 + some / kAdamTensors + (chunks >> 22);
  const int64_t parts = norm ? std::min(chunks, tables * kAdamParts) : 0;
  Ws m(ws);
  AdamArgs a{};
  double* const part = norm ? m.take<double>((size_t)parts) : nullptr;
  float* const coef = clip ? m.take<float>(1) : nullptr;
  if (!ws) {
    *ws_bytes = m.off;
    return PSGDK_OK;
  }
  if (*ws_bytes < m.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *ws_bytes, m.off);
  const hipStream_t st = (hipStream_t)stream;
  if (norm) {
    int64_t done = 0;
    PSGDK_TRY(each_table(q, a, [&](AdamArgs& x, int dt) {
      int n = 0;
      if (done + std::min(x.first[x.count], kAdamParts) > parts) return fail(PSGDK_EWORKSPACE, "more tables than planned");
      x.part = part + done;
      const int rc = hip_check(adamw_norm_launch(x, dt, n, st), "gradient norm");
      done += n;
      return rc;
    }));
    PSGDK_TRY(hip_check(adamw_coef_launch(part, done, q->max_norm, q->norm, coef, st), "gradient norm"));
  }
  if (!q->p) return PSGDK_OK;
  const double c1 = -std::expm1((double)q->step * std::log(q->beta1)), c2 = -std::expm1((double)q->step * std::log(q->beta2));
  a.b1 = (float)q->beta1;
  a.c1 = (float)(1.0 - q->beta1);
  a.b2 = (float)q->beta2;
  a.c2 = (float)(1.0 - q->beta2);
  a.keep = (float)(1.0 - q->lr * q->weight_decay);
  a.rate = (float)(q->lr / c1);
  a.root = (float)(1.0 / std::sqrt(c2));
  a.eps = (float)q->eps;
  a.coef = coef;
  a.k0 = (uint32_t)q->seed;
  a.k1 = (uint32_t)(q->seed >> 32);
  a.step = (uint32_t)q->step;
  return each_table(q, a, [&](AdamArgs& x, int dt) { return hip_check(adamw_launch(x, dt, q->bits, st), "adamw"); });
}

}  // extern "C"
