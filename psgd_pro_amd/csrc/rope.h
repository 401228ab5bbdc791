// Norms of queries and keys for each head with the position rotation: argument block and launchers.
#pragma once
#include "block.h"
#include "common.h"

namespace psgdk {

constexpr int kRopeMaxD = 512;
constexpr int kRopeParts = 1024;  // workgroups of the backward pass at most
constexpr int kRopePowers = 8;  // pairs up to 2^8

struct RopeSide {
  const void* p;
  long long sb, sn, sh;  // element strides of sequences, tokens and heads
};
struct RopeArgs {
  long long tokens;      // batch n
  int n, heads, all;     // query heads, query and key heads
  int d, rot, dt, norm;  // rot: elements of a head that are rotated
  float eps;
  const int64_t* pos;    // null: the token's index in its sequence
  long long pos_sb;      // between sequences
  double ratio[kRopePowers];  // theta^(-2/rot) to the powers 1, 2, 4, ...
  int interleaved;
  // [0] queries, [1] keys; outputs are contiguous
  RopeSide x[2];
  void* y[2];
  Vec w[2];
  RopeSide dy[2];        // p null: zero
  void* dx[2];           // null: not wanted
  float* part;           // [2][parts][d] sums over a workgroup's rows of the weights' gradients; null: not wanted
  int parts;
  // set by rope_plan
  int pairs_lane;        // element pairs of a lane: 8, 4 or 1
  int lanes;             // lanes of a head, a power of two
  int waves;             // waves of a token
};
// pairs_lane, lanes, waves and parts; aligned16: every base and stride is a multiple of 16 bytes
void rope_plan(RopeArgs& a, bool backward, bool aligned16, bool aligned8);
hipError_t rope_launch(const RopeArgs& a, bool backward, hipStream_t st);

}  // namespace psgdk
