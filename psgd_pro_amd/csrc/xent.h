// Softmax cross entropy of a vocabulary's logits: argument blocks and launchers.
#pragma once
#include "common.h"

namespace psgdk {

// weight[0] = mean ? 1 / max(1, rows whose target is not `ignore`) : 1
hipError_t xent_weight_launch(const int64_t* target, long long rows, int64_t ignore, int mean, float* weight,
                              hipStream_t st);
// out[0] = sum_i w_i loss[i], w_i = row_weight[i], or weight[0] where row_weight is null; in a fixed order
hipError_t xent_mean_launch(const float* loss, const float* row_weight, const float* weight, long long rows, float* out,
                            hipStream_t st);

// Rows of logits held in memory (fp32, row stride ldz): loss of each row and, with grad, the logits replaced by their
// gradients.
struct XentRowsArgs {
  float* z;                 // rows of vocab values, ldz < vocab + 1024
  long long ldz, rows;
  int vocab, grad;
  int64_t ignore;
  const int64_t* target;
  const float* row_weight;  // null: weight[0] for every row
  const float* weight;
  float* loss;
};
hipError_t xent_rows_launch(const XentRowsArgs& a, hipStream_t st);

// out (bf16, row stride ldo) = in (fp32, row stride ldi), rows x d
hipError_t to_bf16_rows_launch(const float* in, long long ldi, bf16_t* out, long long ldo, long long rows, int d,
                               hipStream_t st);
// out (rows of d) = x, with zeros for the rows whose target is `ignore`
hipError_t xent_mask_rows_launch(const void* x, long long ldx, void* out, const int64_t* target, int64_t ignore,
                                 long long rows, int d, int dt, hipStream_t st);

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
