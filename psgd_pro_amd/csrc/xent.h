// Softmax cross entropy of a vocabulary's logits: argument blocks and launchers.
#pragma once
#include "common.h"
#include "xgemm.h"

namespace psgdk {

// out[0] = sum_i w_i loss[i] in a fixed order, w_i = row_weight[i], or where that is null weight[0], or where that is null
// too (mean) 1 / max(1, rows whose target is not `ignore`) or 1
hipError_t xent_mean_launch(const float* loss, const float* row_weight, const float* weight, const int64_t* target,
                            long long rows, int64_t ignore, int mean, float* out, hipStream_t st);
// order = the rows whose target is not `ignore`, in their order, then the others, whose losses become 0; count[0] = how
// many are not; weight[0] = mean ? 1 / max(1, count[0]) : 1
hipError_t xent_order_launch(const int64_t* target, long long rows, int64_t ignore, int mean, int* order, int* count,
                             float* weight, float* loss, hipStream_t st);

// Rows of logits held in memory (fp32, row stride ldz): loss of each row and, with grad, the logits replaced by their
// gradients.
struct XentRowsArgs {
  float* z;                 // 16-byte aligned; ldz a multiple of 4, less than vocab + 4
  long long ldz, rows;
  int vocab, grad;
  // null, or: the gradients go there, without the mean's weight, rounded to bf16 for the matrix cores of the bf16 products
  // that follow (rows of ldq, a multiple of 64, zeros behind the vocabulary)
  bf16_t* dz;
  long long ldq;
  int64_t ignore;
  const int64_t* target;
  const float* row_weight;  // null: weight[0] for every row
  const float* weight;
  float* loss;
  // null, or: the workgroup that ends last of all_rows ones (done counts them) adds their losses, all_loss[i] times
  // all_weight[i] (null: weight[0]), in a fixed order
  float* mean_loss;
  int* done;
  long long all_rows;
  const float *all_loss, *all_weight;
};
hipError_t xent_rows_launch(const XentRowsArgs& a, hipStream_t st);

// The bf16 path's rows. Reference of row i: r = z_t, the logit of its target, so that the target's exponential is 1 and
// S = sum of the others' gives loss = log(1 + S), softmax_t - 1 = -S / (1 + S). Rows with S over kSumLimit (their loss is
// over 31, or z_t is -inf) take their largest logit as r instead, and the target's exponential e_t = e^(z_t - r).
constexpr float kSumLimit = 2.9e13f;  // e^31: every e^(z - r) below it, z - r within the coded logits' range
struct XentBf16Args {
  // The rows of a slab are places first .. first + rows - 1 of the order: those before count[0] are there and are numbered
  // from 0 in everything made here; the others are ignored ones.
  long long rows, first;
  const int* order;         // from `first` on
  const int* count;
  int d, vocab, parts;      // parts: sums of a row (2 tiles of m)
  const int64_t* target;    // of all rows, as row_weight, x, dx and loss
  const float* row_weight;  // null: 1 (the mean's weight is the products' alpha)
  const bf16_t* x;
  const bf16_t* w;
  bf16_t* dx;               // null, or: its ignored rows become zeros
  long long ldx, ldw, ldm, ldq, lddx;
  bf16_t* xm;               // x's rows with zeros behind d, row stride ldm
  float* zt;                // z_t
  float* ref;               // r
  float* sum;               // S
  int* col;                 // the target's column; vocab for a foreign target (r is NaN then)
  int* redo;                // number of blocks of kXgRows rows with a row over the limit, and their numbers
  int* mark;                // of each block: whether it is listed
  const float* sums;        // or, for xent_top_launch, the largest logits
  int16_t* q;               // coded logits, replaced by the logits' gradients in bf16
  float* loss;
};
hipError_t xent_prep_launch(const XentBf16Args& a, hipStream_t st);
// S and loss of each row from its sums; with `again` only of the rows over the limit, else those are listed in redo.
// (xent_dz_launch makes those rows' again by itself.)
hipError_t xent_join_launch(const XentBf16Args& a, int again, hipStream_t st);
// r = the largest logit for the rows over the limit
hipError_t xent_top_launch(const XentBf16Args& a, hipStream_t st);
// the logits' gradients (without the mean's weight), zeros behind the vocabulary
hipError_t xent_dz_launch(const XentBf16Args& a, hipStream_t st);
// out (bf16, row stride ldo) = alpha[0] sum over s of in[s] (fp32, rows x d, row stride ldi; alpha null: 1); with order,
// only of the count[0] - first rows that are there, row r to row order[r]
hipError_t to_bf16_rows_launch(const float* in, int splits, long long ldi, const float* alpha, bf16_t* out, long long ldo,
                               long long rows, int d, const int* order, const int* count, long long first, hipStream_t st);
// out = the sum of the parts of in, n4 float4 each, in order
hipError_t sum_parts_launch(const float* in, int parts, long long n4, float* out, hipStream_t st);
// out (row stride ldo) = in with zeros behind d
hipError_t pad_rows_launch(const bf16_t* in, long long ldi, bf16_t* out, long long ldo, long long rows, int d,
                           hipStream_t st);

// Losses of up to xent_few_rows rows without gradients: the vocabulary matrix is read once, straight into registers.
struct XentFewArgs {
  int rows, d, vocab;
  long long ldx, ldw;
  const bf16_t* x;
  const bf16_t* w;
  int64_t ignore;
  const int64_t* target;
  int wgs;
  float* zt;     // [rows]
  float2* part;  // [wgs][64]: largest logit, sum of e^(z - largest), the target left out of both
  float* loss;
};
// 32, or 64 where the vocabulary is short: to there the matrix's bytes bound the call, and the tiles of 256 rows of the
// large products would be mostly empty. us, this way / those: 32 rows against 131072 x 4096 227 / 236, 64 rows 362 / 249;
// 64 rows against 32768 x 1024 35 / 56, against 16384 x 1024 28 / 56; 1 row against 131072 x 4096 207 / 230.
int xent_few_rows(int64_t vocab);
int xent_few_wgs(int vocab);
hipError_t xent_few_launch(const XentFewArgs& a, hipStream_t st);
// The rows of x (of a slab) for the products: row stride ldm, zeros in the rows whose target is `ignore` and (bf16, ldm a
// multiple of 8) behind d. With weight also, for all rows: weight[0] = mean ? 1 / max(1, those not ignored) : 1,
// count[0] = rows, done[0] = 0.
struct XentCopyArgs {
  long long rows, ldx, ldm;
  int d, mean;
  const void* x;
  void* xm;
  int64_t ignore;
  const int64_t* target;
  const int64_t* all_targets;
  long long all_rows;
  float* weight;
  int *count, *done;
};
hipError_t xent_copy_launch(const XentCopyArgs& a, int dt, hipStream_t st);

// x[b][0 .. n[b]) *= *scale (no access where *scale is 1)
constexpr int kMaxScale = 4;
struct ScaleArgs {
  int nb;
  const float* scale;
  long long n[kMaxScale];
  void* x[kMaxScale];
};
hipError_t scale_by_launch(const ScaleArgs& a, int dt, hipStream_t st);

}  // namespace psgdk
