// One AdamW step over many tensors: argument block and launchers.
#pragma once
#include "common.h"

namespace psgdk {

constexpr int kAdamTensors = 128;  // of a launch: their table is a kernel argument
constexpr int kAdamChunk = 4096;   // elements of a workgroup
constexpr int kAdamBlock = 256;    // elements that share a scale
constexpr int kAdamParts = 2048;   // workgroups of a launch over the gradients' norm at most

struct AdamArgs {
  int count;                        // tensors
  int first[kAdamTensors + 1];      // chunks in front of tensor t
  int index[kAdamTensors];          // tensor t's number in the call
  long long n[kAdamTensors];
  long long at[kAdamTensors];       // its first element here, where a long tensor is cut
  void* p[kAdamTensors];
  const void* g[kAdamTensors];
  void* m[kAdamTensors];            // fp32, or e4m3 codes
  void* v[kAdamTensors];
  uint8_t* ms[kAdamTensors];        // scales (8 bits)
  uint8_t* vs[kAdamTensors];
  float b1, c1, b2, c2;             // betas and 1 - beta
  float keep, rate, root, eps;      // p = keep p - rate m / (root sqrt(v) + eps)
  const float* coef;                // of the gradients (null: 1)
  uint32_t k0, k1, step;
  double* part;                     // sums of squares of the norm's workgroups
};
hipError_t adamw_launch(const AdamArgs& a, int dt, int bits, hipStream_t st);
// sums of squares of the gradients: returns the workgroups in `parts` (at most kAdamParts), one double each at a.part
hipError_t adamw_norm_launch(const AdamArgs& a, int dt, int& parts, hipStream_t st);
// norm = sqrt(sum of n parts), coef = min(1, max_norm / norm); either may be null
hipError_t adamw_coef_launch(const double* part, long long n, double max_norm, float* norm, float* coef, hipStream_t st);

}  // namespace psgdk
