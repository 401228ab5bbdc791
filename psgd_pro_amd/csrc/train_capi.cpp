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
  // A launch holds less than 2^32 threads: these are the forward and backward kernels' of a row, one for each 8 elements,
  // 1024 for res_wide rows. The other launches' grids do not grow with the rows.
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

// Rows whose logits (4 bytes each in fp32, 2 on the bf16 path) are in memory at once: up to 1 GiB of them. Fewer rows a
// slab mean more sums of dw in fp32, more of them nothing (12288 x 2048 x 131072: 20.6 ms with 512 MiB, 18.7 with 1 GiB,
// 19.4 with 2, whose slabs are uneven there).
constexpr int64_t kLogitBytes = (int64_t)1 << 30;
// and no more than this many: xent_rows_launch has 256 threads or more for each, and a launch less than 2^32 (the bf16 path's
// codes lie in rows of at least 64: 2^23 rows of 256 threads)
constexpr int64_t kSlabRows = (int64_t)1 << 22;
// 256 rows of a product's operand stay within 32-bit byte offsets
constexpr int64_t kMaxVocab = (int64_t)1 << 22;

// To here lce_small's fewer launches win over lce_bf16's fewer bytes and its gathered rows. us (with gradients), small /
// large: 64 x 256 x 8192 48 / 75, 512 x 1024 x 16384 123 / 134, 256 x 1024 x 32768 132 / 155; beyond: 512 x 1024 x 32768
// 191 / 183, 1024 x 1024 x 8192 133 / 131, 4096 x 256 x 2048 223 / 132.
constexpr int64_t kSmallRows = 512, kSmallLogits = (int64_t)1 << 23;

struct Lce {
  int64_t rows, d, vocab;
  int dtype;
  const void* x;
  int64_t ldx;
  const void* w;
  int64_t ldw;
  const int64_t* target;
  int64_t ignore;
  const float* row_weight;
  int mean;
  float *loss, *mean_loss;
  void* dx;
  int64_t lddx;
  void* dw;
  int64_t lddw;
  void* ws;
  size_t* ws_bytes;
  hipStream_t st;
};

// The workspace's size (ws null: PSGDK_OK with `done` set) or the check of the caller's.
int lce_ws(const Lce& p, const Ws& m, bool& done) {
  done = !p.ws;
  if (done) *p.ws_bytes = m.off;
  else if (*p.ws_bytes < m.off) return fail(PSGDK_EWORKSPACE, "workspace %zu < %zu bytes", *p.ws_bytes, m.off);
  return PSGDK_OK;
}
int lce_pointers(const Lce& p) {
  PSGDK_TRY(check_rows(p.x, p.ldx, p.d, "x"));
  PSGDK_TRY(check_rows(p.w, p.ldw, p.d, "w"));
  if (!p.target || !p.loss) return fail(PSGDK_EINVAL, "target, loss: null device pointer");
  if (p.dx) PSGDK_TRY(check_rows(p.dx, p.lddx, p.d, "dx"));
  if (p.dw) PSGDK_TRY(check_rows(p.dw, p.lddw, p.d, "dw"));
  return PSGDK_OK;
}
// whether the bf16 products cannot read the vocabulary matrix where it is
bool needs_copy(const Lce& p) {
  return p.d % 8 != 0 || p.ldw % 8 != 0 || p.ldw > kMaxVocab || (reinterpret_cast<uintptr_t>(p.w) & 15) != 0;
}
int lce_mean(const Lce& p, const float* weight) {
  if (!p.mean_loss) return PSGDK_OK;
  return hip_check(xent_mean_launch(p.loss, p.row_weight, weight, p.target, p.rows, p.ignore, p.mean, p.mean_loss, p.st),
                   "cross entropy mean");
}

// rows r0 .. r0 + n - 1 of x for the products; with weight what all rows share besides
int lce_copy(const Lce& p, int64_t r0, int64_t n, void* xm, int64_t ldm, float* weight, int* count, int* ended) {
  XentCopyArgs a{};
  a.rows = n;
  a.ldx = p.ldx;
  a.ldm = ldm;
  a.d = (int)p.d;
  a.mean = p.mean;
  a.x = static_cast<const char*>(p.x) + r0 * p.ldx * esize(p.dtype);
  a.xm = xm;
  a.ignore = p.ignore;
  a.target = p.target + r0;
  a.all_targets = p.target;
  a.all_rows = p.rows;
  a.weight = weight;
  a.count = count;
  a.done = ended;
  return hip_check(xent_copy_launch(a, p.dtype, p.st), "cross entropy copy");
}
// their losses from their logits, and the logits' gradients in their place or in dz; the mean or sum of up to kSmallRows
// with the last
int lce_rows(const Lce& p, int64_t r0, int64_t n, float* z, int64_t ldz, bf16_t* dz, int64_t ldq, const float* weight,
             int* ended) {
  XentRowsArgs a{};
  a.z = z;
  a.ldz = ldz;
  a.rows = n;
  a.vocab = (int)p.vocab;
  a.grad = p.dx || p.dw;
  a.dz = dz;
  a.ldq = ldq;
  a.ignore = p.ignore;
  a.target = p.target + r0;
  a.row_weight = p.row_weight ? p.row_weight + r0 : nullptr;
  a.weight = weight;
  a.loss = p.loss + r0;
  a.mean_loss = p.rows <= kSmallRows ? p.mean_loss : nullptr;  // (more rows would queue at the count of those that ended)
  a.done = ended;
  a.all_rows = p.rows;
  a.all_loss = p.loss;
  a.all_weight = p.row_weight;
  return hip_check(xent_rows_launch(a, p.st), "cross entropy rows");
}

// An m x d product with a long k has few of the 128 x 256 tiles that fill the CUs: parts of k as problems of one launch then
// (0: one part). 2048 x 512 x 10007: dx 216 us in one part, 115 + 16 in parts; 65536 x 256 x 1024: dw 1160 in one part, 321 + 7 in parts.
int64_t f32_parts(int64_t m, int64_t d, int64_t k, const void* out, int64_t ldo) {
  const int64_t tiles = ((m + 127) / 128) * ((d + 255) / 256);
  if (tiles >= 128 || ldo != d || d % 4 || (reinterpret_cast<uintptr_t>(out) & 15)) return 0;
  const int64_t parts = std::min<int64_t>({PSGDK_MAXB, 256 / tiles, k / 512});
  return parts > 1 ? parts : 0;
}
// out (m x d) = z w (z: m x k) or, with ta, z^T w (z: k x m), w: k x d; sums: room for parts + 1 of them
int f32_split_k(const Lce& p, int ta, int64_t m, int64_t k, int parts, const float* z, int64_t ldz, const float* w, int64_t ldw,
                float* sums, float* out) {
  const int64_t part = k / parts / 4 * 4, done = parts * part, step = ta ? ldz : 1;
  const psgdk_stream_t st = (psgdk_stream_t)p.st;
  const void *za[PSGDK_MAXB], *wa[PSGDK_MAXB];
  float* oa[PSGDK_MAXB];
  for (int64_t i = 0; i < parts; ++i) {
    za[i] = z + i * part * step;
    wa[i] = w + i * part * ldw;
    oa[i] = sums + i * m * p.d;
  }
  PSGDK_TRY(psgdk_gemm(PSGDK_PREC_F32, ta, 0, m, p.d, part, 1.f, PSGDK_F32, PSGDK_F32, parts, za, ldz, wa, ldw, 0.f, oa, p.d,
                       st));
  if (done < k) {
    za[0] = z + done * step;
    wa[0] = w + done * ldw;
    oa[0] = sums + parts * m * p.d;
    PSGDK_TRY(psgdk_gemm(PSGDK_PREC_F32, ta, 0, m, p.d, k - done, 1.f, PSGDK_F32, PSGDK_F32, 1, za, ldz, wa, ldw, 0.f, oa,
                         p.d, st));
  }
  return hip_check(sum_parts_launch(sums, parts + (done < k ? 1 : 0), m * p.d / 4, out, p.st), "sums of parts");
}

// float32: the logits of a slab of rows by the converting engine, a pass over them, and its products with W and x.
int lce_f32(const Lce& p) {
  const int64_t ldz = (p.vocab + 3) / 4 * 4, slab = std::min({p.rows, kSlabRows, std::max<int64_t>(1, kLogitBytes / 4 / ldz)});
  Ws m(p.ws);
  float* const weight = m.take<float>(1);
  int* const count = m.take<int>(1);
  int* const ended = m.take<int>(1);
  float* const z = m.take<float>(slab * ldz);
  float* const xm = m.take<float>(slab * p.d);
  const int64_t dx_parts = p.dx ? f32_parts(slab, p.d, p.vocab, p.dx, p.lddx) : 0;
  const int64_t dw_parts = p.dw && slab == p.rows ? f32_parts(p.vocab, p.d, p.rows, p.dw, p.lddw) : 0;
  float* const sums = m.take<float>(std::max(dx_parts ? (dx_parts + 1) * slab * p.d : 0,
                                             dw_parts ? (dw_parts + 1) * p.vocab * p.d : 0));
  bool done;
  PSGDK_TRY(lce_ws(p, m, done));
  if (done) return PSGDK_OK;
  PSGDK_TRY(lce_pointers(p));
  for (int64_t r0 = 0; r0 < p.rows; r0 += slab) {
    const int64_t n = std::min(slab, p.rows - r0);
    // an ignored row's x must reach nothing: 0 times an infinity is not 0, and a product scales its operands together
    PSGDK_TRY(lce_copy(p, r0, n, xm, p.d, r0 ? nullptr : weight, count, ended));
    const void *zc = z, *xc = xm;
    const psgdk_stream_t st = (psgdk_stream_t)p.st;
    PSGDK_TRY(psgdk_gemm(PSGDK_PREC_F32, 0, 1, n, p.vocab, p.d, 1.f, PSGDK_F32, PSGDK_F32, 1, &xc, p.d, &p.w, p.ldw, 0.f,
                         &z, ldz, st));
    PSGDK_TRY(lce_rows(p, r0, n, z, ldz, nullptr, 0, weight, ended));
    if (p.dx) {
      float* out = static_cast<float*>(p.dx) + r0 * p.lddx;
      if (dx_parts)
        PSGDK_TRY(f32_split_k(p, 0, n, p.vocab, (int)dx_parts, z, ldz, static_cast<const float*>(p.w), p.ldw, sums, out));
      else
        PSGDK_TRY(psgdk_gemm(PSGDK_PREC_F32, 0, 0, n, p.d, p.vocab, 1.f, PSGDK_F32, PSGDK_F32, 1, &zc, ldz, &p.w, p.ldw,
                             0.f, &out, p.lddx, st));
    }
    if (p.dw) {
      float* out = static_cast<float*>(p.dw);
      if (dw_parts)
        PSGDK_TRY(f32_split_k(p, 1, p.vocab, n, (int)dw_parts, z, ldz, xm, p.d, sums, out));
      else
        PSGDK_TRY(psgdk_gemm(PSGDK_PREC_F32, 1, 0, p.vocab, p.d, n, 1.f, PSGDK_F32, PSGDK_F32, 1, &zc, ldz, &xc, p.d,
                             r0 ? 1.f : 0.f, &out, p.lddw, st));
    }
  }
  return p.rows <= kSmallRows ? PSGDK_OK : lce_mean(p, weight);
}

// bfloat16, a few rows, losses only
int lce_few(const Lce& p) {
  XentFewArgs a{};
  a.rows = (int)p.rows;
  a.d = (int)p.d;
  a.vocab = (int)p.vocab;
  a.wgs = xent_few_wgs(a.vocab);
  Ws m(p.ws);
  a.zt = m.take<float>(64);
  a.part = m.take<float2>((size_t)a.wgs * 64);
  bool done;
  PSGDK_TRY(lce_ws(p, m, done));
  if (done) return PSGDK_OK;
  PSGDK_TRY(lce_pointers(p));
  a.x = static_cast<const bf16_t*>(p.x);
  a.ldx = p.ldx;
  a.w = static_cast<const bf16_t*>(p.w);
  a.ldw = p.ldw;
  a.ignore = p.ignore;
  a.target = p.target;
  a.loss = p.loss;
  PSGDK_TRY(hip_check(xent_few_launch(a, p.st), "cross entropy of a few rows"));
  return lce_mean(p, nullptr);
}

// bfloat16, rows and vocabulary small: the logits in fp32, a pass over them, and the products of their gradients: half as
// many launches as the way below.
int lce_small(const Lce& p) {
  const bool grad = p.dx || p.dw;
  const int64_t ld = (p.d + 7) / 8 * 8, ldz = (p.vocab + 3) / 4 * 4, ldq = (p.vocab + 63) / 64 * 64, n = p.rows;
  const bool copy_w = needs_copy(p);
  const XgPlan z_plan = xgemm_plan(p.vocab, n, ld, false), dx_plan = xgemm_plan(p.d, n, ldq, true),
               dw_plan = xgemm_plan(p.d, p.vocab, n, false);
  const int splits = p.dx ? dx_plan.splits : 1;
  Ws m(p.ws);
  float* const weight = m.take<float>(1);
  int* const count = m.take<int>(1);
  int* const ended = m.take<int>(1);
  float* const z = m.take<float>(n * ldz);
  bf16_t* const xm = m.take<bf16_t>(n * ld);
  bf16_t* const wp = m.take<bf16_t>(copy_w ? p.vocab * ld : 0);
  bf16_t* const dz = m.take<bf16_t>(grad ? n * ldq : 0);
  float* const dxp = m.take<float>(splits > 1 ? splits * n * ld : 0);
  bool done;
  PSGDK_TRY(lce_ws(p, m, done));
  if (done) return PSGDK_OK;
  PSGDK_TRY(lce_pointers(p));
  XgArgs g{};
  g.A = static_cast<const bf16_t*>(p.w);
  g.lda = p.ldw;
  if (copy_w) {
    PSGDK_TRY(hip_check(pad_rows_launch(g.A, p.ldw, wp, ld, p.vocab, (int)p.d, p.st), "cross entropy copy"));
    g.A = wp;
    g.lda = ld;
  }
  PSGDK_TRY(lce_copy(p, 0, n, xm, ld, weight, count, ended));
  g.count = count;
  g.M = (int)p.vocab;
  g.N = (int)n;
  g.K = (int)ld;
  g.B = xm;
  g.ldb = ld;
  g.splits = 1;
  g.outf = z;
  g.ldo = ldz;
  XgArgs x = g;
  PSGDK_TRY(hip_check(xgemm_launch(x, XG_Z, z_plan.bm, p.st), "logits"));
  PSGDK_TRY(lce_rows(p, 0, n, z, ldz, grad ? dz : nullptr, ldq, weight, ended));
  const float* const alpha = p.mean ? weight : nullptr;
  if (p.dx) {
    x = g;
    x.M = (int)p.d;
    x.K = (int)ldq;
    x.kreal = (int)p.vocab;
    x.B = dz;
    x.ldb = ldq;
    x.splits = splits;
    x.kchunk = dx_plan.kchunk;
    x.out = static_cast<bf16_t*>(p.dx);
    x.ldo = splits > 1 ? ld : p.lddx;
    x.alpha = alpha;
    x.outf = splits > 1 ? dxp : nullptr;
    PSGDK_TRY(hip_check(xgemm_launch(x, XG_DX, dx_plan.bm, p.st), "dx"));
    if (splits > 1)
      PSGDK_TRY(hip_check(to_bf16_rows_launch(dxp, splits, ld, alpha, x.out, p.lddx, n, (int)p.d, nullptr, nullptr, 0, p.st),
                          "dx sums"));
  }
  if (p.dw) {
    x = g;
    x.M = (int)p.d;
    x.N = (int)p.vocab;
    x.K = (int)n;
    x.A = xm;
    x.lda = ld;
    x.B = dz;
    x.ldb = ldq;
    x.out = static_cast<bf16_t*>(p.dw);
    x.ldo = p.lddw;
    x.alpha = alpha;
    x.outf = nullptr;
    PSGDK_TRY(hip_check(xgemm_launch(x, XG_DW, dw_plan.bm, p.st), "dw"));
  }
  return PSGDK_OK;
}

// bfloat16: the logits of a slab of rows as 16-bit codes with the sums of their exponentials (one product), a pass that
// makes them the logits' gradients, and the products of those with W and x.
int lce_bf16(const Lce& p) {
  const bool grad = p.dx || p.dw;
  const int64_t ld = (p.d + 7) / 8 * 8, ldq = (p.vocab + 63) / 64 * 64;
  int64_t slab = std::max<int64_t>(kXgRows, kLogitBytes / 2 / ldq / kXgRows * kXgRows);
  if (slab >= p.rows) slab = p.rows;
  const int64_t blocks = (slab + kXgRows - 1) / kXgRows, parts = 2 * ((p.vocab + 255) / 256);
  const bool copy_w = needs_copy(p);
  const XgPlan dx_plan = xgemm_plan(p.d, slab, ldq, true), dw_plan = xgemm_plan(p.d, p.vocab, slab, true);
  const bool sum_w = p.dw && (slab < p.rows || dw_plan.splits > 1);
  const int splits = p.dx ? dx_plan.splits : 1;
  Ws m(p.ws);
  float* const weight = m.take<float>(1);
  int* const count = m.take<int>(1);
  int* const order = m.take<int>(p.rows);
  XentBf16Args a{};
  a.xm = m.take<bf16_t>(slab * ld);
  a.zt = m.take<float>(slab);
  a.ref = m.take<float>(slab);
  a.sum = m.take<float>(slab);
  a.col = m.take<int>(slab);
  a.redo = m.take<int>(1 + blocks);
  a.mark = m.take<int>(blocks);
  float* const sums = m.take<float>(slab * parts);
  bf16_t* const wp = m.take<bf16_t>(copy_w ? p.vocab * ld : 0);
  a.q = m.take<int16_t>(grad ? slab * ldq : 0);
  float* const dxp = m.take<float>(splits > 1 ? splits * slab * ld : 0);
  float* const dwf = m.take<float>(sum_w ? dw_plan.splits * p.vocab * ld : 0);
  bool done;
  PSGDK_TRY(lce_ws(p, m, done));
  if (done) return PSGDK_OK;
  PSGDK_TRY(lce_pointers(p));
  const bf16_t* w = static_cast<const bf16_t*>(p.w);
  int64_t ldw = p.ldw;
  if (copy_w) {
    PSGDK_TRY(hip_check(pad_rows_launch(w, ldw, wp, ld, p.vocab, (int)p.d, p.st), "cross entropy copy"));
    w = wp;
    ldw = ld;
  }
  a.d = (int)p.d;
  a.vocab = (int)p.vocab;
  a.parts = (int)parts;
  a.count = count;
  a.target = p.target;
  a.row_weight = p.row_weight;
  a.x = static_cast<const bf16_t*>(p.x);
  a.loss = p.loss;
  a.dx = static_cast<bf16_t*>(p.dx);
  a.lddx = p.lddx;
  a.w = w;
  a.ldw = ldw;
  a.ldx = p.ldx;
  a.ldm = ld;
  a.ldq = ldq;
  a.sums = sums;
  const float* const alpha = p.mean ? weight : nullptr;
  PSGDK_TRY(hip_check(xent_order_launch(p.target, p.rows, p.ignore, p.mean, order, count, weight, p.loss, p.st),
                      "cross entropy order"));
  for (int64_t r0 = 0; r0 < p.rows; r0 += slab) {
    const int64_t n = std::min(slab, p.rows - r0);
    a.rows = n;
    a.first = r0;
    a.order = order + r0;
    PSGDK_TRY(hip_check(xent_prep_launch(a, p.st), "cross entropy rows"));
    XgArgs g{};
    g.M = (int)p.vocab;
    g.N = (int)n;
    g.K = (int)ld;
    g.A = w;
    g.lda = ldw;
    g.B = a.xm;
    g.ldb = ld;
    g.splits = 1;
    g.count = count;
    g.first = (int)r0;
    g.q = grad ? a.q : nullptr;
    g.ldo = ldq;
    g.ref = a.ref;
    g.target = a.col;
    g.sums = sums;
    PSGDK_TRY(hip_check(xgemm_launch(g, XG_LOGITS, 256, p.st), "logits"));
    PSGDK_TRY(hip_check(xent_join_launch(a, 0, p.st), "cross entropy sums"));
    // rows whose reference was too low: their maximum, then their blocks once more (nothing where there are none)
    XgArgs t = g;
    t.q = nullptr;
    t.max_only = 1;
    t.tops = sums;  // of whole blocks, which all get their sums again
    t.redo = g.redo = a.redo;
    PSGDK_TRY(hip_check(xgemm_launch(t, XG_LOGITS, 256, p.st), "largest logits"));
    PSGDK_TRY(hip_check(xent_top_launch(a, p.st), "largest logits of rows"));
    PSGDK_TRY(hip_check(xgemm_launch(g, XG_LOGITS, 256, p.st), "logits again"));
    if (!grad) {
      PSGDK_TRY(hip_check(xent_join_launch(a, 1, p.st), "cross entropy sums again"));
      continue;
    }
    PSGDK_TRY(hip_check(xent_dz_launch(a, p.st), "logits' gradients"));
    if (p.dx) {
      bf16_t* const out = static_cast<bf16_t*>(p.dx);
      XgArgs x{};
      x.count = count;
      x.first = (int)r0;
      x.order = a.order;
      x.M = (int)p.d;
      x.N = (int)n;
      x.K = (int)ldq;
      x.A = w;
      x.lda = ldw;
      x.B = reinterpret_cast<const bf16_t*>(a.q);
      x.ldb = ldq;
      x.splits = splits;
      x.kchunk = dx_plan.kchunk;
      x.out = out;
      x.ldo = splits > 1 ? ld : p.lddx;
      x.alpha = alpha;
      x.outf = splits > 1 ? dxp : nullptr;
      x.kreal = (int)p.vocab;
      PSGDK_TRY(hip_check(xgemm_launch(x, XG_DX, dx_plan.bm, p.st), "dx"));
      if (splits > 1)
        PSGDK_TRY(hip_check(to_bf16_rows_launch(dxp, splits, ld, alpha, out, p.lddx, n, (int)p.d, a.order, count, r0,
                                      p.st), "dx sums"));
    }
    if (p.dw) {
      XgArgs x{};
      x.count = count;
      x.first = (int)r0;
      x.M = (int)p.d;
      x.N = (int)p.vocab;
      x.K = (int)n;
      x.A = a.xm;
      x.lda = ld;
      x.B = reinterpret_cast<const bf16_t*>(a.q);
      x.ldb = ldq;
      x.splits = dw_plan.splits;  // (of few rows that count, the last ones have none and add zeros)
      x.kchunk = dw_plan.kchunk;
      x.out = static_cast<bf16_t*>(p.dw);
      x.ldo = sum_w ? ld : p.lddw;
      x.alpha = alpha;
      x.outf = sum_w ? dwf : nullptr;
      x.accumulate = r0 != 0;
      PSGDK_TRY(hip_check(xgemm_launch(x, XG_DW, dw_plan.bm, p.st), "dw"));
    }
  }
  if (sum_w)
    PSGDK_TRY(hip_check(to_bf16_rows_launch(dwf, dw_plan.splits, ld, alpha, static_cast<bf16_t*>(p.dw), p.lddw, p.vocab,
                                            (int)p.d, nullptr, nullptr, 0, p.st), "dw sums"));
  return lce_mean(p, weight);
}

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
  a.means = w.take<float4>(res_backward_wide(a) ? q->rows : 0);
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
  PSGDK_TRY(check_size(vocab, 1, kMaxVocab, "vocab"));
  if (!ws_bytes) return fail(PSGDK_EINVAL, "ws_bytes is null");
  if (mean && row_weight) return fail(PSGDK_EINVAL, "mean and row_weight exclude each other");
  if (ldx < d || ldw < d || (dx && lddx < d) || (dw && lddw < d)) return fail(PSGDK_ESHAPE, "row stride < d = %lld", (long long)d);
  const Lce p{rows, d, vocab, dtype, x, ldx, w, ldw, target, ignore, row_weight, mean, loss, mean_loss, dx, lddx, dw, lddw,
              ws, ws_bytes, (hipStream_t)stream};
  if (dtype == PSGDK_F32) return lce_f32(p);
  if (rows <= xent_few_rows(vocab) && !dx && !dw) return lce_few(p);
  return rows <= kSmallRows && rows * vocab <= kSmallLogits ? lce_small(p) : lce_bf16(p);
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
