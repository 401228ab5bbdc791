// Attention with a sliding window and first tokens that stay visible: argument blocks and launchers.
#pragma once
#include "common.h"

namespace psgdk {

// Rows of one key head: the queries of its `group` query heads, row r = token r / group, head r % group of them.
// A row's query is at position p = start + r / group of its sequence and sees key j where
//   0 <= p < length,  j <= p  and  (p - j < window or j < sinks).
struct AttnSide {
  const void* p;
  long long sb, sn, sh;  // element strides of sequences, tokens and heads
};
struct AttnArgs {
  int batch, n, m, kv, group, d, dt;  // n queries and m keys a sequence; dt: storage dtype (0 fp32, 1 bf16)
  int rows;                           // n group
  int window, sinks;                  // window: at most 2^30
  uint32_t div;                       // row / group = (uint64) row div >> div_shift for rows below 2^31
  int div_shift;
  float scale, scale2;                // of the scores, and times log2 e
  AttnSide q, k, v;
  AttnSide o, dout;                   // o: written by the forward call, read by the backward call
  bf16_t* rest;                       // laid out as o, bf16 only: o before its rounding less o (null: not kept)
  const int64_t *lengths, *starts;    // one a sequence in device memory (null: m, m - n)
  float* lse;                         // log2 of a row's sum of e^score: [batch][kv][rows] (forward: null, not stored)
  // forward: the key tiles of a row tile in `parts`; with more than one, each leaves its sums and the largest scores
  int parts;
  float* part_o;                      // [part][batch kv][rows][d], fp32, not divided by the sum
  float* part_ml;                     // [part][batch kv][rows][2]: reference score in base 2, sum
  // backward
  void *dq, *dk, *dv;                 // null: not wanted; dq as (batch, n, heads, d), dk and dv as (batch, m, kv, d)
  float* delta;                       // [batch][kv][rows]: sum of o do over d, written by the dq pass
  int* row_pos;                       // the same: the row's position, -1 where it sees nothing
  int sink_tiles, sink_parts, rest_parts;  // key tiles that hold sinks, and parts of the rows they and the others are cut in
  float* part_kv;                     // [tile parts][2][128][dp] sums of dk and dv where a tile has more than one part
};

constexpr int kAttnMaxD = 128;
inline int attn_dp(int d) { return (d + 31) / 32 * 32; }
constexpr int kAttnKeys = 128;  // keys of a dk, dv tile

// Rows of a forward workgroup: 128, or 32 with the keys of a tile on two waves where there are few rows.
bool attn_few(const AttnArgs& a);
int attn_parts(const AttnArgs& a);
void attn_backward_parts(AttnArgs& a);  // sink_tiles, sink_parts, rest_parts
long long attn_part_tiles(const AttnArgs& a);  // tile parts that leave sums

hipError_t attn_forward_launch(const AttnArgs& a, hipStream_t st);
hipError_t attn_dq_launch(const AttnArgs& a, hipStream_t st);   // delta, and dq where wanted
hipError_t attn_dkv_launch(const AttnArgs& a, hipStream_t st);

}  // namespace psgdk
