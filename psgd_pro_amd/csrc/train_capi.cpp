// The C ABI of the training step's operators (include/psgdk.h, level 3): argument validation, workspace layout and the
// sequencing of the launches. Host code only; every launch goes to the caller's stream, nothing synchronizes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/psgdk.h"
#include "block.h"
#include "xent.h"

namespace psgdk {
int set_error(int code, const char* msg);
}

using namespace psgdk;

namespace {

int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}
int hip_check(hipError_t e, const char* what) {
  return e == hipSuccess ? PSGDK_OK : fail(PSGDK_EHIP, "%s: %s", what, hipGetErrorString(e));
}
#define PSGDK_TRY(expr)              \
  do {                               \
    const int _rc = (expr);          \
    if (_rc != PSGDK_OK) return _rc; \
  } while (0)

int check_dt(int dt, const char* name) {
  if (dt != PSGDK_F32 && dt != PSGDK_BF16) return fail(PSGDK_EINVAL, "%s = %d", name, dt);
  return PSGDK_OK;
}
int check_size(int64_t v, int64_t lo, int64_t hi, const char* name) {
  if (v < lo || v > hi)
    return fail(PSGDK_ESHAPE, "%s = %lld: must be in %lld..%lld", name, (long long)v, (long long)lo, (long long)hi);
  return PSGDK_OK;
}
// a tensor of rows: present, row stride at least d
int check_rows(const void* p, int64_t ld, int64_t d, const char* name) {
  if (!p) return fail(PSGDK_EINVAL, "%s: null device pointer", name);
  if (ld < d) return fail(PSGDK_ESHAPE, "%s: row stride %lld < %lld", name, (long long)ld, (long long)d);
  return PSGDK_OK;
}
constexpr int64_t kMaxRows = (int64_t)1 << 40;

int make_drop(float p, uint64_t seed, uint64_t stream_id, Drop& d) {
  if (!(p >= 0.f && p <= 1.f)) return fail(PSGDK_EINVAL, "p = %g: must be in 0..1", (double)p);
  d.k0 = (unsigned)seed;
  d.k1 = (unsigned)(seed >> 32);
  d.s0 = (unsigned)stream_id;
  d.s1 = (unsigned)(stream_id >> 32);
  d.thr = (unsigned)std::nearbyint(65536.0 * p);
  d.scale = d.thr < 65536 ? (float)(65536.0 / (65536 - d.thr)) : 0.f;
  return PSGDK_OK;
}

size_t esize(int dt) { return dt == PSGDK_BF16 ? 2 : 4; }

// Bump allocator over the caller's workspace; with base == nullptr it only measures.
struct Ws {
  char* base;
  size_t off = 0;
  explicit Ws(void* b) : base(static_cast<char*>(b)) {}
  template <typename T>
  T* take(size_t count) {
    off = (off + 255) & ~size_t(255);
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += count * sizeof(T);
    return p;
  }
};

// the argument checks and the kernels' argument block of both residual_norm calls
int res_args(const psgdk_residual_norm_t* q, ResArgs& a) {
  if (!q) return fail(PSGDK_EINVAL, "null argument block");
  PSGDK_TRY(check_dt(q->dtype, "dtype"));
  PSGDK_TRY(check_size(q->d, 1, kMaxNormD, "d"));
  // the launches hold at most 2^32 threads: one for each 8 elements of a row, 1024 for res_wide rows
  const int64_t threads = res_wide(q->d) ? 1024 : q->d <= 512 ? 64 : q->d <= 1024 ? 128 :
                          q->d <= 2048 ? 256 : q->d <= 4096 ? 512 : 1024;
  PSGDK_TRY(check_size(q->rows, 0, (((int64_t)1 << 32) - 1024) / threads, "rows"));
  if (q->pre < PSGDK_NORM_NONE || q->pre > PSGDK_NORM_LAYER) return fail(PSGDK_EINVAL, "pre = %d", q->pre);
  if (q->post < PSGDK_NORM_NONE || q->post > PSGDK_NORM_LAYER) return fail(PSGDK_EINVAL, "post = %d", q->post);
  if (!(q->eps >= 0.f)) return fail(PSGDK_EINVAL, "eps = %g: must be >= 0", (double)q->eps);
  if ((q->pre == PSGDK_NORM_NONE && (q->pre_w || q->pre_b)) || (q->pre == PSGDK_NORM_RMS && q->pre_b))
    return fail(PSGDK_EINVAL, "pre: weight or bias of a norm that has none");
  if ((q->post == PSGDK_NORM_NONE && (q->post_w || q->post_b)) || (q->post == PSGDK_NORM_RMS && q->post_b))
    return fail(PSGDK_EINVAL, "post: weight or bias of a norm that has none");
  if (!q->f && (q->post != PSGDK_NORM_NONE || q->gate_rows || q->p != 0.f))
    return fail(PSGDK_EINVAL, "post, gate and dropout need f");
  if (q->pre_w || q->pre_b || q->post_w || q->post_b) PSGDK_TRY(check_dt(q->w_dtype, "w_dtype"));
  a = ResArgs{};
  PSGDK_TRY(make_drop(q->p, q->seed, q->stream_id, a.drop));
  PSGDK_TRY(check_size(q->gate_rows, 0, std::max<int64_t>(q->rows, 1), "gate_rows"));
  if (q->gate_rows) {
    if (q->rows % q->gate_rows)
      return fail(PSGDK_ESHAPE, "gate_rows = %lld does not divide rows = %lld", (long long)q->gate_rows, (long long)q->rows);
    PSGDK_TRY(check_dt(q->gate_dtype, "gate_dtype"));
    PSGDK_TRY(check_rows(q->gate, q->ldgate, q->d, "gate"));
  }
  a.rows = q->rows;
  a.d = (int)q->d;
  a.dt = q->dtype;
  a.pre = q->pre;
  a.post = q->post;
  a.eps = q->eps;
  a.scale = q->scale;
  a.gate_every = q->gate_rows ? std::max<int64_t>(q->rows / q->gate_rows, 1) : std::max<int64_t>(q->rows, 1);
  a.gate = Vec{q->gate_rows ? q->gate : nullptr, q->gate_dtype};
  a.ldg = q->gate_rows ? q->ldgate : 0;
  a.x = q->x;
  a.ldx = q->ldx;
  a.f = q->f;
  a.ldf = q->ldf;
  if (q->f && q->ldf < q->d) return fail(PSGDK_ESHAPE, "f: row stride %lld < %lld", (long long)q->ldf, (long long)q->d);
  a.pre_w = Vec{q->pre_w, q->w_dtype};
  a.pre_b = Vec{q->pre_b, q->w_dtype};
  a.post_w = Vec{q->post_w, q->w_dtype};
  a.post_b = Vec{q->post_b, q->w_dtype};
  a.y = q->y;
  a.ldy = q->ldy;
  a.h = q->h;
  a.ldh = q->ldh;
  if (reinterpret_cast<uintptr_t>(q->stats) & 15) return fail(PSGDK_EINVAL, "stats: 16-byte alignment");
  a.stats = reinterpret_cast<float4*>(q->stats);
  for (int& k : a.slot) k = -1;
  return PSGDK_OK;
}

// Rows whose logits (fp32) are in memory at once: up to 1 GiB of them.
constexpr int64_t kLogitBytes = (int64_t)1 << 30;

}  // namespace

extern "C" {

int psgdk_dropout(int64_t rows, int64_t d, int dtype, const void* x, int64_t ldx, void* y, int64_t ldy, float p,
                  uint64_t seed, uint64_t stream_id, psgdk_stream_t stream) {
  PSGDK_TRY(check_dt(dtype, "dtype"));
  PSGDK_TRY(check_size(rows, 0, kMaxRows, "rows"));
  PSGDK_TRY(check_size(d, 1, (int64_t)1 << 30, "d"));
  DropArgs a{};
  PSGDK_TRY(make_drop(p, seed, stream_id, a.drop));
  if (!rows) return PSGDK_OK;
  PSGDK_TRY(check_rows(x, ldx, d, "x"));
  PSGDK_TRY(check_rows(y, ldy, d, "y"));
  a.rows = rows;
  a.d = (int)d;
  a.dt = dtype;
  a.x = x;
  a.ldx = ldx;
  a.y = y;
  a.ldy = ldy;
  return hip_check(dropout_launch(a, (hipStream_t)stream), "dropout");
}

int psgdk_residual_norm(const psgdk_residual_norm_t* q, psgdk_stream_t stream) {
  ResArgs a;
  PSGDK_TRY(res_args(q, a));
  if (!q->rows) return PSGDK_OK;
  PSGDK_TRY(check_rows(q->x, q->ldx, q->d, "x"));
  if (q->y) PSGDK_TRY(check_rows(q->y, q->ldy, q->d, "y"));
  if (q->pre != PSGDK_NORM_NONE) PSGDK_TRY(check_rows(q->h, q->ldh, q->d, "h"));
  else if (!q->y) return fail(PSGDK_EINVAL, "nothing to compute: no y and no norm");
  return hip_check(residual_norm_launch(a, (hipStream_t)stream), "residual norm");
}

int psgdk_residual_norm_backward(const psgdk_residual_norm_t* q, const psgdk_residual_norm_grads_t* g, void* ws,
                                 size_t* ws_bytes, psgdk_stream_t stream) {
  ResArgs a;
  PSGDK_TRY(res_args(q, a));
  if (!g) return fail(PSGDK_EINVAL, "null gradient block");
  if (!ws_bytes) return fail(PSGDK_EINVAL, "ws_bytes is null");
  if (g->dh && q->pre == PSGDK_NORM_NONE) return fail(PSGDK_EINVAL, "dh without a norm before the block");
  if ((g->dpre_w || g->dpre_b) && q->pre == PSGDK_NORM_NONE) return fail(PSGDK_EINVAL, "dpre_w, dpre_b without that norm");
  if ((g->dpost_w || g->dpost_b) && q->post == PSGDK_NORM_NONE)
    return fail(PSGDK_EINVAL, "dpost_w, dpost_b without that norm");
  if ((g->df || g->dpost_w || g->dpost_b || g->dgate) && !q->f) return fail(PSGDK_EINVAL, "df, dpost or dgate without f");
  if (g->dgate && !q->gate_rows) return fail(PSGDK_EINVAL, "dgate without a gate");
  if (g->dpre_w || g->dpre_b || g->dpost_w || g->dpost_b) PSGDK_TRY(check_dt(q->w_dtype, "w_dtype"));
  a.dy = g->dy;
  a.lddy = g->lddy;
  a.dh = g->dh;
  a.lddh = g->lddh;
  a.dx = g->dx;
  a.lddx = g->lddx;
  a.df = g->df;
  a.lddf = g->lddf;
  a.dgate = g->dgate;
  a.lddg = g->lddgate;
  const bool gate_sums = g->dgate && a.gate_every > 1;
  residual_norm_split(a, gate_sums);
  void* const sums[4] = {g->dpre_w, g->dpre_b, g->dpost_w, g->dpost_b};
  int n = 0;
  for (int k = 0; k < 4; ++k)
    if (sums[k]) a.slot[k] = n++;
  Ws w(ws);
  a.part = w.take<float>((size_t)n * a.parts * a.d);
  a.gpart = w.take<float>(gate_sums ? (size_t)(a.per_gate > 1 ? a.parts : q->gate_rows) * a.d : 0);
  if (!gate_sums) a.gpart = nullptr;
  a.means = w.take<float4>(res_wide(a.d) ? q->rows : 0);
  if (!ws) {
    *ws_bytes = w.off;
    return PSGDK_OK;
  }
  if (*ws_bytes < w.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *ws_bytes, w.off);
  if (q->rows) {
    if (g->dy) PSGDK_TRY(check_rows(g->dy, g->lddy, q->d, "dy"));
    if (g->dh) {
      PSGDK_TRY(check_rows(g->dh, g->lddh, q->d, "dh"));
      PSGDK_TRY(check_rows(q->x, q->ldx, q->d, "x"));
    }
    if ((g->dh || q->post != PSGDK_NORM_NONE) && !q->stats) return fail(PSGDK_EINVAL, "stats: null device pointer");
    if (g->dx) PSGDK_TRY(check_rows(g->dx, g->lddx, q->d, "dx"));
    if (g->df) PSGDK_TRY(check_rows(g->df, g->lddf, q->d, "df"));
    if (g->dgate) PSGDK_TRY(check_rows(g->dgate, g->lddgate, q->d, "dgate"));
    PSGDK_TRY(hip_check(residual_norm_backward_launch(a, (hipStream_t)stream), "residual norm backward"));
  }
  ColumnSums s{};
  s.d = a.d;
  for (int k = 0; k < 4; ++k) {
    if (!sums[k]) continue;
    auto& e = s.e[s.n++];
    e.in = a.part + (size_t)a.slot[k] * a.parts * a.d;
    e.out = sums[k];
    e.dt = q->w_dtype;
    e.groups = 1;
    e.per = a.parts;
    e.ldo = a.d;
  }
  if (gate_sums) {
    auto& e = s.e[s.n++];
    e.in = a.gpart;
    e.out = g->dgate;
    e.dt = q->gate_dtype;
    e.groups = q->gate_rows;
    e.per = a.per_gate;
    e.ldo = g->lddgate;
  }
  return hip_check(column_sums_launch(s, (hipStream_t)stream), "column sums");
}

int psgdk_linear_cross_entropy(int64_t rows, int64_t d, int64_t vocab, int dtype, const void* x, int64_t ldx,
                               const void* w, int64_t ldw, const int64_t* target, int64_t ignore,
                               const float* row_weight, int mean, float* loss, float* mean_loss, void* dx,
                               int64_t lddx, void* dw, int64_t lddw, void* ws, size_t* ws_bytes,
                               psgdk_stream_t stream) {
  PSGDK_TRY(check_dt(dtype, "dtype"));
  PSGDK_TRY(check_size(rows, 1, (int64_t)1 << 30, "rows"));
  PSGDK_TRY(check_size(d, 1, (int64_t)1 << 20, "d"));
  PSGDK_TRY(check_size(vocab, 1, (int64_t)1 << 28, "vocab"));
  if (!ws_bytes) return fail(PSGDK_EINVAL, "ws_bytes is null");
  if (mean && row_weight) return fail(PSGDK_EINVAL, "mean and row_weight exclude each other");
  const hipStream_t st = (hipStream_t)stream;
  const bool grad = dx || dw, cvt = dtype == PSGDK_BF16;
  const int64_t ldz = (vocab + 3) / 4 * 4, slab = std::min(rows, std::max<int64_t>(1, kLogitBytes / 4 / ldz));
  Ws m(ws);
  float* const weight = m.take<float>(1);
  float* const z = m.take<float>(slab * ldz);
  float* const dxf = m.take<float>(cvt && dx ? slab * d : 0);
  float* const dwf = m.take<float>(cvt && dw ? vocab * d : 0);
  char* const xm = m.take<char>(slab * d * esize(dtype));
  if (!ws) {
    *ws_bytes = m.off;
    return PSGDK_OK;
  }
  if (*ws_bytes < m.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *ws_bytes, m.off);
  PSGDK_TRY(check_rows(x, ldx, d, "x"));
  PSGDK_TRY(check_rows(w, ldw, d, "w"));
  if (!target || !loss) return fail(PSGDK_EINVAL, "target, loss: null device pointer");
  if (dx) PSGDK_TRY(check_rows(dx, lddx, d, "dx"));
  if (dw) PSGDK_TRY(check_rows(dw, lddw, d, "dw"));
  const int prec = dtype == PSGDK_BF16 ? PSGDK_PREC_BF16 : PSGDK_PREC_F32;
  PSGDK_TRY(hip_check(xent_weight_launch(target, rows, ignore, mean, weight, st), "cross entropy weight"));
  for (int64_t r0 = 0; r0 < rows; r0 += slab) {
    const int64_t n = std::min(slab, rows - r0);
    const void* xs = static_cast<const char*>(x) + r0 * ldx * esize(dtype);
    // an ignored row's x must reach nothing: 0 times an infinity is not 0, and a product scales its operands together
    PSGDK_TRY(hip_check(xent_mask_rows_launch(xs, ldx, xm, target + r0, ignore, n, (int)d, dtype, st), "mask rows"));
    const void *zc = z, *xc = xm;
    PSGDK_TRY(psgdk_gemm(prec, 0, 1, n, vocab, d, 1.f, dtype, dtype, 1, &xc, d, &w, ldw, 0.f, &z, ldz, stream));
    XentRowsArgs a{};
    a.z = z;
    a.ldz = ldz;
    a.rows = n;
    a.vocab = (int)vocab;
    a.grad = grad;
    a.ignore = ignore;
    a.target = target + r0;
    a.row_weight = row_weight ? row_weight + r0 : nullptr;
    a.weight = weight;
    a.loss = loss + r0;
    PSGDK_TRY(hip_check(xent_rows_launch(a, st), "cross entropy rows"));
    if (dx) {
      float* out = cvt ? dxf : static_cast<float*>(dx) + r0 * lddx;
      PSGDK_TRY(psgdk_gemm(prec, 0, 0, n, d, vocab, 1.f, PSGDK_F32, dtype, 1, &zc, ldz, &w, ldw, 0.f, &out,
                           cvt ? d : lddx, stream));
      if (cvt)
        PSGDK_TRY(hip_check(to_bf16_rows_launch(dxf, d, static_cast<bf16_t*>(dx) + r0 * lddx, lddx, n, (int)d, st),
                            "cross entropy dx"));
    }
    if (dw) {
      float* out = cvt ? dwf : static_cast<float*>(dw);
      PSGDK_TRY(psgdk_gemm(prec, 1, 0, vocab, d, n, 1.f, PSGDK_F32, dtype, 1, &zc, ldz, &xc, d, r0 ? 1.f : 0.f, &out,
                           cvt ? d : lddw, stream));
    }
  }
  if (cvt && dw)
    PSGDK_TRY(hip_check(to_bf16_rows_launch(dwf, d, static_cast<bf16_t*>(dw), lddw, vocab, (int)d, st), "cross entropy dw"));
  if (mean_loss)
    PSGDK_TRY(hip_check(xent_mean_launch(loss, row_weight, weight, rows, mean_loss, st), "cross entropy mean"));
  return PSGDK_OK;
}

int psgdk_scale_by(int nb, const int64_t* n, int dtype, void* const* x, const float* scale, psgdk_stream_t stream) {
  if (nb < 1 || nb > kMaxScale) return fail(PSGDK_EINVAL, "nb = %d: must be in 1..%d", nb, kMaxScale);
  PSGDK_TRY(check_dt(dtype, "dtype"));
  if (!n || !x || !scale) return fail(PSGDK_EINVAL, "null pointer");
  ScaleArgs a{};
  a.nb = nb;
  a.scale = scale;
  for (int b = 0; b < nb; ++b) {
    PSGDK_TRY(check_size(n[b], 0, (int64_t)1 << 46, "n"));
    if (n[b] && !x[b]) return fail(PSGDK_EINVAL, "x[%d]: null device pointer", b);
    a.n[b] = n[b];
    a.x[b] = x[b];
  }
  return hip_check(scale_by_launch(a, dtype, (hipStream_t)stream), "scale");
}

}  // extern "C"
