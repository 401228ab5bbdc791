// Dropout and the residual sum between two blocks of a transformer with its norms: argument blocks and launchers.
#pragma once
#include "common.h"

namespace psgdk {

enum Norm : int { NORM_NONE = 0, NORM_RMS = 1, NORM_LAYER = 2 };

// Which elements dropout keeps: element (i, c) of rows of d elements takes the 16-bit number c % 8 (the low half of a
// word first) of the Philox4x32-10 block i ceil(d / 8) + c / 8 (key k0, k1; upper counter words s0, s1) and is kept
// where that number is at least thr; kept elements are scaled by `scale`. thr = 0: everything is kept.
struct Drop {
  unsigned k0, k1, s0, s1;
  unsigned thr;  // 0 .. 65536
  float scale;   // 65536 / (65536 - thr), 0 for thr = 65536
};

struct DropArgs {
  long long rows;
  int d, dt;  // dt: storage dtype (0 fp32, 1 bf16)
  long long ldx, ldy;
  const void* x;
  void* y;
  Drop drop;
};
hipError_t dropout_launch(const DropArgs& a, hipStream_t st);

// A weight, bias or gate vector set with its own storage dtype (p null: absent).
struct Vec {
  const void* p;
  int dt;
};

struct ResArgs {
  long long rows;
  int d, dt;                // x, f, y, h and their gradients share one storage dtype
  int pre, post;            // Norm
  float eps, scale;
  long long gate_every;     // rows that share a gate row (1: one for each)
  long long ldx, ldf, ldg, ldy, ldh;
  const void* x;
  const void* f;            // null: y is x
  Vec gate, pre_w, pre_b, post_w, post_b;
  void* y;                  // null: not stored
  void* h;                  // null without a norm before
  float4* stats;            // forward: optional output (mean, 1/std of y, mean, 1/std of f); backward: input
  Drop drop;
  // backward
  long long lddy, lddh, lddx, lddf, lddg;
  const void* dy;           // null: zero
  const void* dh;           // null: zero
  void* dx;                 // null: not wanted
  void* df;                 // null: not wanted
  void* dgate;              // null: not wanted; in gate.dt
  // Column sums the caller wants, as partial sums over the rows of each workgroup: array k (kSum*) at part + slot[k]
  // parts d, -1 when not wanted. The sums of a gate that several rows share lie at gpart: a row for each gate
  // (per_gate = 1) or for each workgroup.
  float* part;
  float* gpart;
  int slot[4];
  long long parts;          // workgroups
  long long chunk;          // rows of a workgroup: whole gates' rows, or a part of one gate's
  long long per_gate;       // workgroups that share one gate row (1 where a workgroup has whole gates)
  float4* means;            // res_backward_wide: one float4 a row for the column kernel
};
enum { kSumPreW = 0, kSumPreB = 1, kSumPostW = 2, kSumPostB = 3 };
// Rows that do not stay in registers but are read again for each pass: under one vector of 8 elements and over 8192.
inline bool res_wide(long long d) { return d < 8 || d > 8192; }
constexpr int kMaxNormD = 1 << 20;

// What a backward call has beside a root-mean-square norm before the next block.
enum : int { kPost = 1, kGate = 2, kBias = 4 };
inline int res_has(const ResArgs& a) {
  return (a.post != NORM_NONE ? kPost : 0) | (a.gate.p ? kGate : 0) |
         (a.pre == NORM_LAYER || a.post == NORM_LAYER ? kBias : 0);
}
// The backward pass has no registers for two of these in rows over 4096 (nor for a gate alone, where fp32 rows end inside a
// vector): such a row's values are made again from its bits for each pass, the column sums by a kernel of their own.
inline bool res_backward_wide(const ResArgs& a) {
  const int h = res_has(a);
  return res_wide(a.d) || (a.d > 4096 && ((h & (h - 1)) != 0 || (h == kGate && a.d % 8 != 0 && a.dt == 0)));
}

hipError_t residual_norm_launch(const ResArgs& a, hipStream_t st);
// rows of one workgroup and the number of workgroups of the backward pass (chunk, per_gate, parts); whole_gates: the
// gate's gradient sums over rows
void residual_norm_split(ResArgs& a, bool gate_sums);
hipError_t residual_norm_backward_launch(const ResArgs& a, hipStream_t st);

// out[g][c] = sum_p in[g per + p][c], p < per in order, rows of d, for up to five outputs in one launch
struct ColumnSums {
  int n, d;
  struct {
    const float* in;
    void* out;
    int dt;
    long long groups, per, ldo;
  } e[5];
};
hipError_t column_sums_launch(const ColumnSums& s, hipStream_t st);

}  // namespace psgdk
