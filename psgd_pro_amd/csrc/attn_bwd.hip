// Attention backward, two passes without atomics: for 128 rows over their keys (delta, dq), for 128 keys over their rows
// (dk, dv), each making the probabilities again from the scores and the forward pass's sums.
#include <algorithm>

#include "attn_dev.h"

namespace psgdk {

namespace {

// With P the probabilities, dP = dO V^T, delta = sum of o dO over a row:  dS = P (dP - delta),  dQ = scale dS K.
// Transposed as the forward pass: a lane has one row, dS^T is the last product's operand where it is made. 4 x 4096 tokens, 32 / 8
// heads of 128, bf16: 770 to 819 us by the box, 6 d flops a visible pair at 1010 to 1070 TFLOP/s (the matrix cores busy 55% of the
// cycles, the vector unit 42%).
template <typename T, int DP, int BK>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && DP > 64 ? 1 : 2) attn_dq_kernel(const AttnArgs a, int row_tiles) {
  using R = Rows<T, DP>;
  constexpr int LOADS = R::loads(BK, 4), TILE = BK * R::PITCH, KT = BK / 32, DC = DP / 16, DT = DP / 32;
  constexpr int AHEAD = sizeof(T) == 2 && DT > 1 ? 4 : 2;  // at most 2 DT
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned lds0 = (unsigned)(uintptr_t)(LDS_AS unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, h = lane >> 5;

  const int work = xcd_run(blockIdx.x, gridDim.x), pair = work / row_tiles, row0 = (row_tiles - 1 - (work - pair * row_tiles)) * 128;
  const int b = pair / a.kv, head = pair - b * a.kv;
  const Seq s = sequence(a, b);
  const int lo = s.start + row_token(a, row0), hi = s.start + row_token(a, min(row0 + 128, a.rows) - 1);
  const KeyTiles tiles = key_tiles<BK>(a, s, lo, hi);

  const int r = row0 + wave * 32 + c, tok = row_token(a, r), g = r - tok * a.group;
  const bool there = r < a.rows;
  const int pos = there && s.start + tok >= 0 && s.start + tok < s.len ? s.start + tok : -1;
  const long long qh = head * a.group + g;
  const T* const qp = static_cast<const T*>(a.q.p) + b * a.q.sb + tok * a.q.sn + qh * a.q.sh;
  const T* const gp = static_cast<const T*>(a.dout.p) + b * a.dout.sb + tok * a.dout.sn + qh * a.dout.sh;
  const T* const op = static_cast<const T*>(a.o.p) + b * a.o.sb + tok * a.o.sn + qh * a.o.sh;
  const T* const some = static_cast<const T*>(a.q.p);
  const T* const lp = sizeof(T) == 2 && a.rest ? reinterpret_cast<const T*>(a.rest) + (op - static_cast<const T*>(a.o.p)) : nullptr;
  frag_t<T> qf[DC], gf[DC];
  float delta = 0.f;
  {
    frag_t<T> of[DC], rf[DC];
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      const int k = 16 * i + 8 * h;
      gf[i] = row_frag<T>(gp, k, a.d, pos >= 0, some);
      of[i] = row_frag<T>(op, k, a.d, pos >= 0, some);
      if constexpr (sizeof(T) == 2) rf[i] = row_frag<T>(lp, k, a.d, pos >= 0 && lp, some);
      qf[i] = row_frag<T>(qp, k, a.d, pos >= 0, some);
    }
#pragma unroll
    for (int i = 0; i < DC; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        delta += (float)gf[i][e] * (float)of[i][e];
        // (o's rounding would put a tenth on the gradients' error, and .03 of their norm where values lie around 16)
        if constexpr (sizeof(T) == 2) delta += (float)gf[i][e] * (float)rf[i][e];
      }
  }
  delta += other_half(delta);
  const long long at = (long long)pair * a.rows + r;
  if (there && h == 0) {
    a.delta[at] = delta;
    a.row_pos[at] = pos;
  }
  if (!a.dq) return;
  float lse = there ? a.lse[at] : 0.f;
  arrived(lse);
#pragma unroll
  for (int i = 0; i < DC; ++i) {
    arrived(qf[i]);
    arrived(gf[i]);
  }

  int vk[LOADS], vv[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    int row, chunk;
    R::where(wave * LOADS + i, lane, row, chunk);
    const bool in = chunk * R::PER < a.d;
    vk[i] = in ? (int)(row * a.k.sn * R::E) + chunk * 16 : kOob;
    vv[i] = in ? (int)(row * a.v.sn * R::E) + chunk * 16 : kOob;
  }
  const T* const kp = static_cast<const T*>(a.k.p) + b * a.k.sb + head * a.k.sh;
  const T* const vp = static_cast<const T*>(a.v.p) + b * a.v.sb + head * a.v.sh;
  // (as in the forward pass)
  i32x4_t rk, rv;
  unsigned to;
  auto plan = [&](int t) __attribute__((always_inline)) {
    const int j0 = tiles.tile(t) * BK;
    rk = rsrc_words(kp + j0 * a.k.sn, ((s.len - j0 - 1) * a.k.sn + a.d) * R::E);
    rv = rsrc_words(vp + j0 * a.v.sn, ((s.len - j0 - 1) * a.v.sn + a.d) * R::E);
    to = uniform(lds0 + (t & 1) * 2 * TILE + wave * LOADS * 1024);
    asm volatile("s_nop 4" : "+s"(rk), "+s"(rv), "+s"(to));
  };
  auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      load_lds(rk, vk[i], to + i * 1024);
      load_lds(rv, vv[i], to + TILE + i * 1024);
    }
  };

  f32x16_t dq[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) dq[i] = zero16();
  if (tiles.count) {
    plan(0);
    load();
  }
  for (int t = 0; t < tiles.count; ++t) {
    const int j0 = tiles.tile(t) * BK;
    plan(t + 1);
    load_wait<0>();
    if (t + 1 < tiles.count) load();
    const unsigned kt = lds0 + (t & 1) * 2 * TILE;
    const Straight<T, DP> keys(kt, lane), values(kt + TILE, lane);
    const Transposed<T, DP> columns(kt, lane);
    const bool look = j0 + BK - 1 > lo || hi >= s.len || (hi - j0 >= a.window && j0 + BK > a.sinks);
#pragma unroll
    for (int i = 0; i < KT; ++i) {
      f32x16_t x = zero16(), dp = zero16();
      frag_t<T> f[AHEAD];
      const auto row_frags = [&](int s) __attribute__((always_inline)) { return s % 2 ? values(i, s / 2) : keys(i, s / 2); };
      first_loads<T>(f, row_frags);
      __builtin_amdgcn_s_setprio(1);
      ahead<T, 2 * DC>(f, row_frags, [&](int s, frag_t<T> y) __attribute__((always_inline)) {
        if (s % 2) dp = mma(y, gf[s / 2], dp);
        else x = mma(y, qf[s / 2], x);
      });
      __builtin_amdgcn_s_setprio(0);
      const auto key_frags = [&](int s) __attribute__((always_inline)) { return columns(2 * i + s / DT, s % DT); };
      first_loads<T>(f, key_frags);
      if (look) {
        const int j = j0 + 32 * i + 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = j + 8 * (e >> 2) + (e & 3);
          x[e] = (key <= pos) & ((pos - key < a.window) | (key < a.sinks)) ? x[e] : -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.scale2, -lse)) * (dp[e] - delta);
      const frag_t<T> ds[2] = {crossed<T>(x, 0), crossed<T>(x, 1)};
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      ahead<T, 2 * DT>(f, key_frags, [&](int s, frag_t<T> y) __attribute__((always_inline)) {
        dq[s % DT] = mma(y, ds[s / DT], dq[s % DT]);
      });
      __builtin_amdgcn_s_setprio(0);
    }
  }
  if (!there) return;
  T* const out = static_cast<T*>(a.dq) + (((long long)b * a.n + tok) * a.kv * a.group + qh) * a.d;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int col = 32 * i + 2 * e + 4 * h;
      if (col >= a.d) continue;
      const float y0 = dq[i][e] * a.scale, y1 = dq[i][e + 1] * a.scale, y2 = dq[i][e + 2] * a.scale, y3 = dq[i][e + 3] * a.scale;
      if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out + col) = make_uint2(pack2_bf16(y0, y1), pack2_bf16(y2, y3));
      else *reinterpret_cast<f32x4_t*>(out + col) = f32x4_t{y0, y1, y2, y3};
    }
}

// 4 values of dk or dv of one key
template <typename T>
__device__ __forceinline__ void store4(T* out, float y0, float y1, float y2, float y3) {
  if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out) = make_uint2(pack2_bf16(y0, y1), pack2_bf16(y2, y3));
  else *reinterpret_cast<f32x4_t*>(out) = f32x4_t{y0, y1, y2, y3};
}

// dV = P^T dO, dK = scale dS^T Q for 128 keys, 32 of each wave, over the rows that see any of them: all the key head's query
// heads are among them, so that shared heads' gradients need no further sum. S = Q K^T has a key in each lane, P and dS are
// the second products' operands where they are made (dV^T = dO^T P, dK^T = Q^T dS), and a tile of rows serves straight and
// transposed. Key tiles that hold sinks are seen by all rows: their rows are cut in parts, whose sums attn_dkv_sum adds.
// KV: the tile's keys and values are fragments in registers; else the values are in LDS (bf16 heads of 128 then fit two waves
// a SIMD: 1750 -> 1400 us of 4 x 4096 tokens with 32 / 8 heads; 1060 with the tiles of the most rows first,
// 8 d flops a pair at 1040 TFLOP/s; 1017 to 1103 by the box, the matrix cores busy 57% of the cycles, the vector unit 43%).
template <typename T, int DP, int BR, bool KV>
__global__ void __launch_bounds__(256, sizeof(T) == 4 && DP > 32 ? 1 : 2) attn_dkv_kernel(const AttnArgs a, int key_tiles) {
  using R = Rows<T, DP>;
  constexpr int LOADS = R::loads(BR, 4), TILE = BR * R::PITCH, STAGE = 2 * TILE + 1024, RT = BR / 32, DC = DP / 16, DT = DP / 32;
  constexpr int AHEAD = sizeof(T) == 4 ? 2 : KV ? 4 : 3, VALUES = KV ? 0 : kAttnKeys * R::PITCH;  // AHEAD: at most 4 DT
  static_assert(BR <= 64, "a load of 64 floats");
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned lds0 = (unsigned)(uintptr_t)(LDS_AS unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, h = lane >> 5;

  const int sinks = a.sink_tiles * a.sink_parts;
  // the tiles with the most rows first, a pair's on one XCD where there are 8 pairs or a multiple of them
  const int pairs = a.batch * a.kv, pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
  const bool sink = rest < sinks;
  const int parts = sink ? a.sink_parts : a.rest_parts, part = sink ? rest % parts : (rest - sinks) % parts;
  const int tile = sink ? rest / parts : a.sink_tiles + (rest - sinks) / parts, j0 = tile * kAttnKeys;
  const int b = pair / a.kv, head = pair - b * a.kv;
  const Seq s = sequence(a, b);
  // tokens that see any of the keys, and their rows' tiles
  const int from = max(0, j0 - s.start);
  int to = min(a.n, s.len - s.start);
  if (!sink && j0 >= a.sinks) to = min(to, j0 + kAttnKeys - 1 + a.window - s.start);
  const int first = (int)((long long)from * a.group / BR), tiles = to > from ? (int)(((long long)to * a.group + BR - 1) / BR) - first : 0;
  const int t0 = part_begin(tiles, part, parts), t1 = part_begin(tiles, part + 1, parts);

  const int key = j0 + wave * 32 + c;
  const T* const kp = static_cast<const T*>(a.k.p) + b * a.k.sb + head * a.k.sh;
  const T* const vp = static_cast<const T*>(a.v.p) + b * a.v.sb + head * a.v.sh;
  frag_t<T> kf[DC], vf[KV ? DC : 1];
#pragma unroll
  for (int i = 0; i < DC; ++i) {
    kf[i] = row_frag<T>(kp + key * a.k.sn, 16 * i + 8 * h, a.d, key < s.len, static_cast<const T*>(a.k.p));
    if constexpr (KV) vf[i] = row_frag<T>(vp + key * a.v.sn, 16 * i + 8 * h, a.d, key < s.len, static_cast<const T*>(a.v.p));
  }
#pragma unroll
  for (int i = 0; i < DC; ++i) {
    arrived(kf[i]);
    if constexpr (KV) arrived(vf[i]);
  }
  if constexpr (!KV) {
    i32x4_t rv = rsrc_words(vp + (long long)j0 * a.v.sn, 0x7fffffff);
    asm volatile("s_nop 4" : "+s"(rv));  // (as in the forward pass)
#pragma unroll
    for (int i = 0; i < R::loads(kAttnKeys, 4); ++i) {
      int row, chunk;
      R::where(wave * R::loads(kAttnKeys, 4) + i, lane, row, chunk);
      const bool in = chunk * R::PER < a.d && j0 + row < s.len;
      load_lds(rv, in ? (int)(row * a.v.sn * R::E) + chunk * 16 : kOob, lds0 + (wave * R::loads(kAttnKeys, 4) + i) * 1024);
    }
  }

  const T* const qp = static_cast<const T*>(a.q.p) + b * a.q.sb + (long long)head * a.group * a.q.sh;
  const T* const gp = static_cast<const T*>(a.dout.p) + b * a.dout.sb + (long long)head * a.group * a.dout.sh;
  // where this lane's rows are, from the token of the tile's first row: the same in every tile where tokens are not cut
  int tok[LOADS], oq[LOADS], og[LOADS];
  auto place = [&](int r0) __attribute__((always_inline)) {
    const int tok0 = row_token(a, r0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      int row, chunk;
      R::where(wave * LOADS + i, lane, row, chunk);
      const int t = row_token(a, r0 + row), g = r0 + row - t * a.group;
      tok[i] = chunk * R::PER < a.d ? t - tok0 : 1 << 30;
      oq[i] = (int)(((t - tok0) * a.q.sn + g * a.q.sh) * R::E) + chunk * 16;
      og[i] = (int)(((t - tok0) * a.dout.sn + g * a.dout.sh) * R::E) + chunk * 16;
    }
  };
  const bool whole = BR % a.group == 0;
  place(0);
  const float* const of_rows = wave == 0 ? a.lse : wave == 1 ? a.delta : reinterpret_cast<const float*>(a.row_pos);
  i32x4_t rq, rg, rs;
  unsigned ring, sums;
  int lo_tok, hi_tok, next0;
  auto plan = [&](int t) __attribute__((always_inline)) {
    next0 = (first + t) * BR;
    const int tok0 = uniform(row_token(a, next0));
    if (!whole) place(next0);
    rq = rsrc_words(qp + tok0 * a.q.sn, 0x7fffffff);
    rg = rsrc_words(gp + tok0 * a.dout.sn, 0x7fffffff);
    rs = rsrc_words(of_rows + (long long)pair * a.rows + next0, 0x7fffffff);
    ring = uniform(lds0 + VALUES + (t & 1) * STAGE + wave * LOADS * 1024);
    sums = uniform(lds0 + VALUES + (t & 1) * STAGE + 2 * TILE + wave * 256);
    asm volatile("s_nop 4" : "+s"(rq), "+s"(rg), "+s"(rs), "+s"(ring), "+s"(sums));
    lo_tok = from - tok0;
    hi_tok = to - tok0;
  };
  auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const bool in = (tok[i] >= lo_tok) & (tok[i] < hi_tok);
      load_lds(rq, in ? oq[i] : kOob, ring + i * 1024);
      load_lds(rg, in ? og[i] : kOob, ring + TILE + i * 1024);
    }
    if (wave < 3) load_lds4(rs, lane < BR && next0 + lane < a.rows ? lane * 4 : kOob, sums);
  };

  f32x16_t dk[DT], dv[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) dk[i] = dv[i] = zero16();
  const Straight<T, DP> values(lds0 + (KV ? 0 : wave * 32 * R::PITCH), lane);
  if (t0 < t1) {
    plan(t0);
    load();
  }
  for (int t = t0; t < t1; ++t) {
    plan(t + 1);
    load_wait<0>();
    if (t + 1 < t1) load();
    const unsigned qt = lds0 + VALUES + (t & 1) * STAGE, gt = qt + TILE, ls = gt + TILE;
    const Straight<T, DP> queries(qt, lane), grads(gt, lane);
    const Transposed<T, DP> query_cols(qt, lane), grad_cols(gt, lane);
    const int r0 = (first + t) * BR, lo = s.start + row_token(a, r0), hi = s.start + row_token(a, r0 + BR - 1);
    const bool look = lo < j0 + kAttnKeys - 1 || hi >= s.len || hi >= s.start + a.n ||
                      (hi - j0 >= a.window && j0 + kAttnKeys > a.sinks);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      f32x16_t x = zero16(), dp = zero16();
      frag_t<T> f[AHEAD];
      if constexpr (KV) {
        const auto row_frags = [&](int s) __attribute__((always_inline)) { return s % 2 ? grads(i, s / 2) : queries(i, s / 2); };
        first_loads<T>(f, row_frags);
        __builtin_amdgcn_s_setprio(1);
        ahead<T, 2 * DC>(f, row_frags, [&](int s, frag_t<T> y) __attribute__((always_inline)) {
          if (s % 2) dp = mma(y, vf[s / 2], dp);
          else x = mma(y, kf[s / 2], x);
        });
      } else {
        // a query's, a gradient's and a value's fragment in turn
        const auto row_frags = [&](int s) __attribute__((always_inline)) {
          return s % 3 == 0 ? queries(i, s / 3) : s % 3 == 1 ? grads(i, s / 3) : values(0, s / 3);
        };
        frag_t<T> held;
        first_loads<T>(f, row_frags);
        __builtin_amdgcn_s_setprio(1);
        ahead<T, 3 * DC>(f, row_frags, [&](int s, frag_t<T> y) __attribute__((always_inline)) {
          if (s % 3 == 0) x = mma(y, kf[s / 3], x);
          else if (s % 3 == 1) held = y;
          else dp = mma(held, y, dp);
        });
      }
      __builtin_amdgcn_s_setprio(0);
      // 16 rows' dO, then their Q, then the next 16 rows'
      const auto col_frags = [&](int s) __attribute__((always_inline)) {
        return s / DT % 2 ? query_cols(2 * i + s / (2 * DT), s % DT) : grad_cols(2 * i + s / (2 * DT), s % DT);
      };
      first_loads<T>(f, col_frags);
      if (look) {  // (rows that are not loaded see none of the keys)
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const i32x4_t pos = *(LDS_AS i32x4_t*)(uintptr_t)(ls + 512 + (32 * i + 2 * e + 4 * h) * 4);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            x[e + q] = (key <= pos[q]) & ((pos[q] - key < a.window) | (key < a.sinks)) ? x[e + q] : -INFINITY;
        }
      }
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const f32x4_t lse = *(LDS_AS f32x4_t*)(uintptr_t)(ls + (32 * i + 2 * e + 4 * h) * 4);
        const f32x4_t delta = *(LDS_AS f32x4_t*)(uintptr_t)(ls + 256 + (32 * i + 2 * e + 4 * h) * 4);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          x[e + q] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e + q], a.scale2, -lse[q]));
          dp[e + q] = x[e + q] * (dp[e + q] - delta[q]);
        }
      }
      const frag_t<T> p[2] = {crossed<T>(x, 0), crossed<T>(x, 1)}, ds[2] = {crossed<T>(dp, 0), crossed<T>(dp, 1)};
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_setprio(1);
      ahead<T, 4 * DT>(f, col_frags, [&](int s, frag_t<T> y) __attribute__((always_inline)) {
        if (s / DT % 2) dk[s % DT] = mma(y, ds[s / (2 * DT)], dk[s % DT]);
        else dv[s % DT] = mma(y, p[s / (2 * DT)], dv[s % DT]);
      });
      __builtin_amdgcn_s_setprio(0);
    }
  }
  // (no load of values may reach LDS after the workgroup)
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  if (parts > 1) {
    const long long at = sink ? ((long long)pair * a.sink_tiles + tile) * parts + part
                              : (a.sink_parts > 1 ? (long long)a.batch * a.kv * sinks : 0) +
                                    ((long long)pair * (key_tiles - a.sink_tiles) + tile - a.sink_tiles) * parts + part;
    float* const out = a.part_kv + (at * 2 * kAttnKeys + wave * 32 + c) * DP;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int col = 32 * i + 2 * e + 4 * h;
        *reinterpret_cast<f32x4_t*>(out + col) = f32x4_t{dk[i][e], dk[i][e + 1], dk[i][e + 2], dk[i][e + 3]};
        *reinterpret_cast<f32x4_t*>(out + kAttnKeys * DP + col) = f32x4_t{dv[i][e], dv[i][e + 1], dv[i][e + 2], dv[i][e + 3]};
      }
    return;
  }
  if (key >= a.m) return;
  const long long at = (((long long)b * a.m + key) * a.kv + head) * a.d;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int col = 32 * i + 2 * e + 4 * h;
      if (col >= a.d) continue;
      if (a.dk) store4(static_cast<T*>(a.dk) + at + col, dk[i][e] * a.scale, dk[i][e + 1] * a.scale, dk[i][e + 2] * a.scale,
                       dk[i][e + 3] * a.scale);
      if (a.dv) store4(static_cast<T*>(a.dv) + at + col, dv[i][e], dv[i][e + 1], dv[i][e + 2], dv[i][e + 3]);
    }
}

// the parts' sums of the key tiles that have several, in order; a thread has 4 columns of a key's dk or dv
template <typename T>
__global__ void __launch_bounds__(256) attn_dkv_sum_kernel(const AttnArgs a, int first_tile, int tiles, int parts, int dp,
                                                           long long base) {
  const int quads = kAttnKeys * dp / 4, per = 2 * quads / 256;  // workgroups of a tile (dp a multiple of 32)
  const int at = blockIdx.x / per, in = (blockIdx.x - at * per) * 256 + threadIdx.x;
  const int pair = at / tiles, tile = at - pair * tiles, which = in / quads, q = in - which * quads;
  const int row = q / (dp / 4), col = (q - row * (dp / 4)) * 4, key = (first_tile + tile) * kAttnKeys + row;
  void* const to = which ? a.dv : a.dk;
  if (key >= a.m || col >= a.d || !to) return;
  const float* from = a.part_kv + ((base + (long long)at * parts) * 2 + which) * kAttnKeys * dp + row * dp + col;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = 0; p < parts; ++p) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(from + (long long)p * 2 * kAttnKeys * dp);
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[e] += x[e];
  }
  const float by = which ? 1.f : a.scale;
  const int b = pair / a.kv, head = pair - b * a.kv;
  store4(static_cast<T*>(to) + (((long long)b * a.m + key) * a.kv + head) * a.d + col, sum[0] * by, sum[1] * by, sum[2] * by,
         sum[3] * by);
}

template <typename T>
constexpr int kTileRows = sizeof(T) == 2 ? 64 : 32;  // of a tile in LDS, keys or rows

template <typename T, int DP>
hipError_t launch_dq(const AttnArgs& a, hipStream_t st) {
  constexpr int BK = kTileRows<T>, smem = 4 * BK * Rows<T, DP>::PITCH;
  const auto fn = attn_dq_kernel<T, DP, BK>;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (attr != hipSuccess) return attr;
  const int row_tiles = (a.rows + 127) / 128;
  hipLaunchKernelGGL(fn, dim3(a.batch * a.kv * row_tiles), dim3(256), smem, st, a, row_tiles);
  return hipGetLastError();
}
template <typename T, int DP>
hipError_t launch_dkv(const AttnArgs& a, hipStream_t st) {
  constexpr bool KV = sizeof(T) == 4 || DP < 128;
  constexpr int BR = KV ? kTileRows<T> : 32, smem = (KV ? 0 : kAttnKeys * Rows<T, DP>::PITCH) + 2 * (2 * BR * Rows<T, DP>::PITCH + 1024);
  const auto fn = attn_dkv_kernel<T, DP, BR, KV>;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (attr != hipSuccess) return attr;
  const int tiles = (a.m + kAttnKeys - 1) / kAttnKeys, rest = tiles - a.sink_tiles, pairs = a.batch * a.kv;
  hipLaunchKernelGGL(fn, dim3(pairs * (a.sink_tiles * a.sink_parts + rest * a.rest_parts)), dim3(256), smem, st, a, tiles);
  hipError_t e = hipGetLastError();
  const unsigned per = 2 * kAttnKeys * DP / 4 / 256;
  if (e == hipSuccess && a.sink_parts > 1) {
    hipLaunchKernelGGL(attn_dkv_sum_kernel<T>, dim3(pairs * a.sink_tiles * per), dim3(256), 0, st, a, 0, a.sink_tiles, a.sink_parts,
                       DP, 0ll);
    e = hipGetLastError();
  }
  if (e == hipSuccess && a.rest_parts > 1 && rest) {
    const long long base = a.sink_parts > 1 ? (long long)pairs * a.sink_tiles * a.sink_parts : 0;
    hipLaunchKernelGGL(attn_dkv_sum_kernel<T>, dim3(pairs * rest * per), dim3(256), 0, st, a, a.sink_tiles, rest, a.rest_parts, DP,
                       base);
    e = hipGetLastError();
  }
  return e;
}

// rows of a tile of the dk, dv pass
int attn_dkv_rows(const AttnArgs& a) { return a.dt == 0 || a.d > 96 ? 32 : 64; }

}  // namespace

// Key tiles with sinks, which all rows see, are cut in as many parts as leave each about the rows of another tile's. The others
// are cut where a round of workgroups would otherwise leave CUs idle: 512 (256 where a wave has a SIMD's registers to itself) run
// at once, and 564 of equal work take as long as 1024 (16384 tokens, window 1024, 16 / 4 heads of 64: 340 us uncut, 230 in three
// parts and 18 adding them). A part costs about 8 tiles of rows for its keys, its sums and their addition.
void attn_backward_parts(AttnArgs& a) {
  const long long br = attn_dkv_rows(a), pairs = (long long)a.batch * a.kv, tiles = (a.m + kAttnKeys - 1) / kAttnKeys;
  const long long all = (a.rows + br - 1) / br;
  const long long seen = std::min(all, ((long long)(a.window + kAttnKeys - 1) * a.group + br - 1) / br + 1);
  a.sink_tiles = a.sinks && seen < all ? (int)((std::min(a.sinks, a.m) + kAttnKeys - 1) / kAttnKeys) : 0;
  const long long rest = pairs * (tiles - a.sink_tiles), slots = a.dt == 0 && a.d > 32 ? 256 : 512, over = 8;
  long long best = 0;
  a.rest_parts = a.sink_parts = 1;
  for (int parts = 1; parts <= 64 && rest && (parts == 1 || (seen / parts >= 4 && rest * parts <= 4096)); ++parts) {
    const long long per = (seen + parts - 1) / parts;
    const long long cost = (rest * parts + pairs * a.sink_tiles * (all / per + 1) + slots - 1) / slots * (per + over) + (parts > 1 ? over : 0);
    if (!best || cost < best) {
      best = cost;
      a.rest_parts = parts;
    }
  }
  const long long share = std::max<long long>(seen / a.rest_parts, 8);
  if (a.sink_tiles)  // (4096 parts' sums are 512 MiB)
    a.sink_parts = (int)std::max<long long>(1, std::min<long long>({all / share, 64, 4096 / (pairs * a.sink_tiles)}));
}
long long attn_part_tiles(const AttnArgs& a) {
  const long long pairs = (long long)a.batch * a.kv, rest = (a.m + kAttnKeys - 1) / kAttnKeys - a.sink_tiles;
  return pairs * ((a.sink_parts > 1 ? (long long)a.sink_tiles * a.sink_parts : 0) + (a.rest_parts > 1 ? rest * a.rest_parts : 0));
}

#define PSGDK_BY_D(fn)                            \
  switch (attn_dp(a.d)) {                         \
    case 32: return a.dt == 0 ? fn<float, 32>(a, st) : fn<bf16_t, 32>(a, st);   \
    case 64: return a.dt == 0 ? fn<float, 64>(a, st) : fn<bf16_t, 64>(a, st);   \
    case 96: return a.dt == 0 ? fn<float, 96>(a, st) : fn<bf16_t, 96>(a, st);   \
    default: return a.dt == 0 ? fn<float, 128>(a, st) : fn<bf16_t, 128>(a, st); \
  }
hipError_t attn_dq_launch(const AttnArgs& a, hipStream_t st) { PSGDK_BY_D(launch_dq) }
hipError_t attn_dkv_launch(const AttnArgs& a, hipStream_t st) { PSGDK_BY_D(launch_dkv) }

}  // namespace psgdk
