// The cross entropy's three bf16 products: argument block shared by the host launchers and the kernels.
#pragma once
#include "common.h"

namespace psgdk {

// acc[m][n] = sum_k A[m][k] B[n][k], M x N x K, stored transposed: element (m, n) at out[n ldo + m]. An operand X is
// read k-contiguous (X[mn][k] at mn ld + k) or mn-contiguous (at k ld + mn); 16-byte aligned base, ld a multiple of 8,
// and K a multiple of 8 where an operand is k-contiguous.
struct XgArgs {
  int M, N, K;
  long long lda, ldb, ldo;
  const bf16_t* A;
  const bf16_t* B;
  int tiles_m, tiles_n;
  int kreal;           // rows of an mn-contiguous A (0: K); k behind them reads zeros
  // the rows that are there: count[0] - first of them (count in device memory), at most N (XG_DW: K)
  const int* count;
  int first;
  int splits, kchunk;  // split s covers k in [s kchunk, (s + 1) kchunk), none empty but by count; splits > 1 need outf
  // products with the vocabulary matrix or the rows: out = alpha[0] acc in bf16 (alpha null: 1), or
  bf16_t* out;
  const float* alpha;
  const int* order;    // XG_DX with out: row n goes to row order[n] (null: n)
  float* outf;         // (where set) split s's acc in fp32 at outf + s N ldo: 16-byte aligned, ldo a multiple of 4
  int accumulate;      // outf += acc
  // logits: m counts the vocabulary, n the rows
  int16_t* q;              // coded logits (see kLogitStep), null: sums only
  const float* ref;        // the row's reference r
  const int* target;       // the row's target column
  float* sums;             // of each 128 columns, the sum of e^(z - r) over those that are not the target: [N][2 tiles_m]
  float* tops;             // with `max_only` instead of all that: their largest z, same layout
  int max_only;
  const int* redo;         // null: every tile; else only those of redo[0] blocks of 256 rows, their numbers behind it
};

// A logit is kept as a 16-bit number of steps of 2^-9 above r - 96: z - r in [-96, 32).
constexpr float kLogitStep = 1.f / 512.f;
constexpr float kLogitLow = -96.f;

constexpr int kXgRows = 256;  // rows (n) of a tile

enum XgKind : int {
  XG_LOGITS = 0,  // both operands k-contiguous: m vocabulary (W), n rows (x), k = d
  XG_DX = 1,      // A mn-contiguous, B k-contiguous: m = d (W), n rows (dz), k vocabulary
  XG_DW = 2,      // both mn-contiguous: m = d (x), n vocabulary (dz), k rows
  XG_Z = 3,       // as XG_LOGITS with outf: the logits themselves
};
// How a product with out M x N (XG_DX, XG_DW) is cut: 256 or 128 rows of m a tile, and parts of k (1 without can_split)
struct XgPlan {
  int bm, splits, kchunk;
};
XgPlan xgemm_plan(long long M, long long N, long long K, bool can_split);
// sets the tile counts, and kchunk where splits is 1; bm: 256 for XG_LOGITS
hipError_t xgemm_launch(XgArgs& a, int kind, int bm, hipStream_t st);

}  // namespace psgdk
