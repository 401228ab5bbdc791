// Attention forward: one pass over the keys with a running reference and sum, and the join of the parts of a long key axis.
#include <cmath>

#include "attn_dev.h"

namespace psgdk {

namespace {

// Scores and outputs are computed transposed, S^T = K Q^T and O^T = V^T P^T: a lane then has one row's scores (of half of the
// keys, the other half is in lane + 32), so that the row's largest score and sum are sums inside a lane, and P^T is the second
// product's operand in the registers where it was made. WQ waves have 32 rows each, WK waves share a tile's keys.
// 4 x 4096 tokens, 32 / 8 heads of 128, bf16: 575 us, 960 TFLOP/s of the visible pairs' 4 d flops (603 to 632 where o's rest
// is stored too, by the box), the matrix cores busy 46% of the cycles and the vector unit 45%: without the exponentials 546, without
// the reads of LDS 535, without the loads 520, without both 465. Tiles of 32 keys with three waves a SIMD: 590; 64 rows a wave, one wave a SIMD,
// products and exponentials in one stream: 910 (two hundred registers moved to and from accumulation registers). A single token
// over 131072 keys of 8 heads: the keys' and values' bytes at 5.4 TB/s, 100 us.
template <typename T, int DP, int WQ, int WK, int BK>
__global__ void __launch_bounds__(64 * WQ * WK, sizeof(T) == 4 && WK == 2 && DP == 128 ? 1 : 2) attn_forward_kernel(const AttnArgs a, int row_tiles) {
  using R = Rows<T, DP>;
  constexpr int W = WQ * WK, LOADS = R::loads(BK, W), TILE = BK * R::PITCH, KT = BK / WK / 32, DC = DP / 16, DT = DP / 32;
  constexpr int AHEAD = DT < 4 || sizeof(T) == 4 ? 2 : 4;  // at most KT DC and 2 KT DT
  // Few rows wait for the keys and values: the matrix cores then take what rounding takes from a probability too, in a product
  // of its own (outputs .0017 of their norm off, as exact ones rounded to bf16, not .0021 to .0024; a token over
  // 131072 keys of 8 heads: 107.3 us without, 107.7 with)
  constexpr bool REST = sizeof(T) == 2 && WK > 1;
  static_assert(LOADS * W * 1024 == TILE && KT * WK * 32 == BK, "whole loads, whole blocks of keys");
  static_assert(!REST || KT == 1, "32 keys a wave");  // (a reference that moves between the first and the second 32 would scale a rest)
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned lds0 = (unsigned)(uintptr_t)(LDS_AS unsigned char*)smem;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, h = lane >> 5, wq = wave % WQ, wk = wave / WQ;

  // each XCD a run of (sequence, key head) pairs, whose keys its L2 holds; of one, the rows with the most keys first
  const int work = xcd_run(blockIdx.x, gridDim.x), pair = work / (row_tiles * a.parts), rest = work - pair * row_tiles * a.parts;
  const int part = rest % a.parts, row0 = (row_tiles - 1 - rest / a.parts) * 32 * WQ;
  const int b = pair / a.kv, head = pair - b * a.kv;
  const Seq s = sequence(a, b);
  const int lo = s.start + row_token(a, row0), hi = s.start + row_token(a, min(row0 + 32 * WQ, a.rows) - 1);
  const KeyTiles tiles = key_tiles<BK>(a, s, lo, hi);
  const int t0 = part_begin(tiles.count, part, a.parts), t1 = part_begin(tiles.count, part + 1, a.parts);

  // this lane's row
  const int r = row0 + wq * 32 + c, tok = row_token(a, r), g = r - tok * a.group;
  const bool there = r < a.rows;
  const int pos = there && s.start + tok >= 0 && s.start + tok < s.len ? s.start + tok : -1;
  const T* const qp = static_cast<const T*>(a.q.p) + b * a.q.sb + tok * a.q.sn + (head * a.group + g) * a.q.sh;
  frag_t<T> qf[DC];
#pragma unroll
  for (int i = 0; i < DC; ++i) qf[i] = row_frag<T>(qp, 16 * i + 8 * h, a.d, pos >= 0, static_cast<const T*>(a.q.p));
#pragma unroll
  for (int i = 0; i < DC; ++i) arrived(qf[i]);

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
  // The next tile's loads: where from, found out in front of the wait for the last ones, and the loads themselves.
  i32x4_t rk, rv;
  unsigned to;
  auto plan = [&](int t, int stage) __attribute__((always_inline)) {
    const int j0 = tiles.tile(t) * BK;
    // (rows behind the sequence, whatever they hold, are behind the buffer's end and read as zeros)
    rk = rsrc_words(kp + j0 * a.k.sn, ((s.len - j0 - 1) * a.k.sn + a.d) * R::E);
    rv = rsrc_words(vp + j0 * a.v.sn, ((s.len - j0 - 1) * a.v.sn + a.d) * R::E);
    to = uniform(lds0 + stage * 2 * TILE + wave * LOADS * 1024);
    // a scalar register that a vector instruction wrote may be read by a load 5 wait states later at the earliest, which
    // the compiler does not see to inside asm statements
    asm volatile("s_nop 4" : "+s"(rk), "+s"(rv), "+s"(to));
  };
  auto load = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      load_lds(rk, vk[i], to + i * 1024);
      load_lds(rv, vv[i], to + TILE + i * 1024);
    }
  };

  float ref = -INFINITY, sum = 0.f;  // the scores' reference, in base 2; this half's sum of 2^(score - reference)
  f32x16_t o[DT];
#pragma unroll
  for (int i = 0; i < DT; ++i) o[i] = zero16();

  if (t0 < t1) {
    plan(t0, 0);
    load();
  }
  for (int t = t0; t < t1; ++t) {
    const int stage = (t - t0) & 1, j0 = tiles.tile(t) * BK;
    plan(t + 1, stage ^ 1);
    load_wait<0>();
    if (t + 1 < t1) load();
    const unsigned kt = lds0 + stage * 2 * TILE + wk * (32 * KT) * R::PITCH;
    const Straight<T, DP> keys(kt, lane);
    const Transposed<T, DP> values(kt + TILE, lane);

    // Keys 32 by 32: their scores, their probabilities beside the products that come next (the next 32 keys' scores, the last
    // ones' values).
    f32x16_t x[KT];
    frag_t<T> p[2 * KT], p_rest[REST ? 2 * KT : 1], f[AHEAD];
    const bool look = j0 + BK - 1 > lo || hi >= s.len || (hi - j0 >= a.window && j0 + BK > a.sinks);
    float mu = 0.f;
    const auto key_frag = [&](int i) __attribute__((always_inline)) { return keys(i / DC, i % DC); };
    const auto value_frag = [&](int i) __attribute__((always_inline)) { return values(i / DT, i % DT); };
    // the mask and the reference of keys i
    const auto follow = [&](int i) __attribute__((always_inline)) {
      if (look) {
        const int j = j0 + wk * 32 * KT + 32 * i + 4 * h;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int key = j + 8 * (e >> 2) + (e & 3);
          x[i][e] = (key <= pos) & ((pos - key < a.window) | (key < a.sinks)) ? x[i][e] : -INFINITY;
        }
      }
      float top = x[i][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) top = fmaxf(top, x[i][e]);
      top = max_halves(top) * a.scale2;
      // The reference follows the largest score only where that is over it by more than 2^8: the sums have room for that, and
      // the products are rarely scaled then.
      if (__any(top > ref + 8.f)) {
        const float next = fmaxf(ref, top), by = ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - next);
        ref = next;
        sum *= by;
#pragma unroll
        for (int k = 0; k < DT; ++k)
#pragma unroll
          for (int e = 0; e < 16; ++e) o[k][e] *= by;
        if (i > 0) {  // (whose values are not added yet)
#pragma unroll
          for (int e = 0; e < 16; ++e) x[0][e] *= by;
          p[0] = crossed<T>(x[0], 0);
          p[1] = crossed<T>(x[0], 1);
        }
      }
      mu = ref == -INFINITY ? 0.f : ref;
    };
    // (bf16: the probabilities are rounded for the matrix cores, and without their rest their sum is of the rounded ones)
    const auto probability = [&](int i, int e) __attribute__((always_inline)) {
      float v = __builtin_amdgcn_exp2f(__builtin_fmaf(x[i][e], a.scale2, -mu));
      arrived(v);  // (here, beside a product)
      x[i][e] = v;
      if constexpr (REST) sum += v;
      if (e % 8 == 7) {
        p[2 * i + e / 8] = crossed<T>(x[i], e / 8);
        if constexpr (REST) p_rest[2 * i + e / 8] = crossed_rest(x[i], e / 8, p[2 * i + e / 8]);
        else sum = sum_of(p[2 * i + e / 8], sum);
      }
    };
    first_loads<T>(f, key_frag);
    __builtin_amdgcn_s_setprio(1);
    x[0] = zero16();
#pragma unroll
    for (int i = 0; i < DC; ++i) {
      x[0] = mma(f[i % AHEAD], qf[i], x[0]);
      if (i + AHEAD < KT * DC) f[i % AHEAD] = key_frag(i + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
    __builtin_amdgcn_s_setprio(0);
    follow(0);
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (KT == 2) {
      x[1] = zero16();
#pragma unroll
      for (int i = 0; i < DC; ++i) {
        x[1] = mma(f[(DC + i) % AHEAD], qf[i], x[1]);
        if (DC + i + AHEAD < 2 * DC) f[(DC + i) % AHEAD] = key_frag(DC + i + AHEAD);
#pragma unroll
        for (int e = i * 16 / DC; e < (i + 1) * 16 / DC; ++e) probability(0, e);
        __builtin_amdgcn_sched_barrier(0);
      }
      first_loads<T>(f, value_frag);
      follow(1);
    } else {
      first_loads<T>(f, value_frag);
#pragma unroll
      for (int e = 0; e < 16; ++e) probability(0, e);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    ahead<T, 2 * KT * DT>(f, value_frag, [&](int i, frag_t<T> y) __attribute__((always_inline)) {
      o[i % DT] = mma(y, p[i / DT], o[i % DT]);
      if constexpr (REST) o[i % DT] = mma(y, p_rest[i / DT], o[i % DT]);
      if (KT == 2 && i < 2 * DT) {
#pragma unroll
        for (int e = i * 16 / (2 * DT); e < (i + 1) * 16 / (2 * DT); ++e) probability(KT - 1, e);
      }
    });
    __builtin_amdgcn_s_setprio(0);
  }
  sum += other_half(sum);

  if constexpr (WK > 1) {  // the waves' sums joined in LDS
    static_assert(WK == 2 && WQ == 1, "two waves");
    constexpr int AT = DT * 16;
    float* const buf = reinterpret_cast<float*>(smem);
    __syncthreads();
    if (wk) {
#pragma unroll
      for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) buf[(i * 16 + e) * 64 + lane] = o[i][e];
      buf[AT * 64 + lane] = ref;
      buf[(AT + 1) * 64 + lane] = sum;
    }
    __syncthreads();
    if (wk) return;
    const float ref1 = buf[AT * 64 + lane], sum1 = buf[(AT + 1) * 64 + lane], next = fmaxf(ref, ref1);
    const float by = ref == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - next);
    const float by1 = ref1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref1 - next);
    ref = next;
    sum = sum * by + sum1 * by1;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; ++e) o[i][e] = o[i][e] * by + buf[(i * 16 + e) * 64 + lane] * by1;
  }
  if (!there) return;

  if (a.parts > 1) {
    const long long at = ((long long)part * a.batch * a.kv + pair) * a.rows + r;
    float* const out = a.part_o + at * a.d;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
      for (int e = 0; e < 16; e += 4) {
        const int col = 32 * i + 2 * e + 4 * h;
        if (col < a.d) *reinterpret_cast<f32x4_t*>(out + col) = f32x4_t{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
      }
    if (h == 0) *reinterpret_cast<float2*>(a.part_ml + at * 2) = make_float2(ref, sum);
    return;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (a row that sees nothing: zeros)
  T* const out = static_cast<T*>(const_cast<void*>(a.o.p)) + b * a.o.sb + tok * a.o.sn + (head * a.group + g) * a.o.sh;
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      const int col = 32 * i + 2 * e + 4 * h;
      if (col >= a.d) continue;
      const float y0 = o[i][e] * inv, y1 = o[i][e + 1] * inv, y2 = o[i][e + 2] * inv, y3 = o[i][e + 3] * inv;
      if constexpr (sizeof(T) == 2) {
        const uint2 w = make_uint2(pack2_bf16(y0, y1), pack2_bf16(y2, y3));
        *reinterpret_cast<uint2*>(out + col) = w;
        if (a.rest)
          *reinterpret_cast<uint2*>(a.rest + (out - static_cast<const T*>(a.o.p)) + col) =
              make_uint2(pack2_bf16(y0 - __uint_as_float(w.x << 16), y1 - __uint_as_float(w.x & 0xffff0000u)),
                         pack2_bf16(y2 - __uint_as_float(w.y << 16), y3 - __uint_as_float(w.y & 0xffff0000u)));
      } else {
        *reinterpret_cast<f32x4_t*>(out + col) = f32x4_t{y0, y1, y2, y3};
      }
    }
  if (a.lse && h == 0) a.lse[(long long)pair * a.rows + r] = sum == 0.f ? 0.f : ref + __builtin_amdgcn_logf(sum);
}

// One row a workgroup: G groups of 32 lanes with 4 columns each take every G-th part, and are added in LDS in order.
template <typename T, int G>
__global__ void __launch_bounds__(32 * G) attn_join_kernel(const AttnArgs a) {
  __shared__ float buf[G][kAttnMaxD];
  __shared__ float red[16], sums[G];
  const long long row = blockIdx.x, all = (long long)a.batch * a.kv * a.rows;
  const int tid = threadIdx.x, grp = tid >> 5, col = (tid & 31) * 4;
  const float2* const ml = reinterpret_cast<const float2*>(a.part_ml);
  float top = -INFINITY;
  for (int p = tid; p < a.parts; p += 32 * G) top = fmaxf(top, ml[p * all + row].x);
  top = block_max(top, red);
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int p = grp; p < a.parts; p += G) {
    const float2 v = ml[p * all + row];
    const float by = v.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(v.x - top);
    sum += v.y * by;
    if (col < a.d) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(a.part_o + (p * all + row) * a.d + col);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += x[e] * by;
    }
  }
  if ((tid & 31) == 0) sums[grp] = sum;
  *reinterpret_cast<f32x4_t*>(&buf[grp][col]) = acc;
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int i = 0; i < G; ++i) total += sums[i];
  const int pair = (int)(row / a.rows), r = (int)(row - (long long)pair * a.rows), b = pair / a.kv, head = pair - b * a.kv;
  const int tok = row_token(a, r), g = r - tok * a.group;
  if (tid < a.d) {
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < G; ++i) x += buf[i][tid];
    T* const out = static_cast<T*>(const_cast<void*>(a.o.p)) + b * a.o.sb + tok * a.o.sn + (head * a.group + g) * a.o.sh;
    const float y = total == 0.f ? 0.f : x / total;
    out[tid] = from_f32<T>(y);
    if constexpr (sizeof(T) == 2) {
      if (a.rest) a.rest[(out - static_cast<const T*>(a.o.p)) + tid] = f32_to_bf16(y - to_f32<T>(out[tid]));
    }
  }
  if (tid == 0 && a.lse) a.lse[row] = total == 0.f ? 0.f : top + __builtin_amdgcn_logf(total);
}

template <typename T, int DP, int WQ, int WK, int BK>
hipError_t launch(const AttnArgs& a, hipStream_t st) {
  constexpr int smem = 4 * BK * Rows<T, DP>::PITCH;
  static_assert(WK == 1 || smem >= (DP / 32 * 16 + 2) * 256, "room for a wave's sums");
  const auto fn = attn_forward_kernel<T, DP, WQ, WK, BK>;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (attr != hipSuccess) return attr;
  const int row_tiles = (a.rows + 32 * WQ - 1) / (32 * WQ);
  hipLaunchKernelGGL(fn, dim3(a.batch * a.kv * row_tiles * a.parts), dim3(64 * WQ * WK), smem, st, a, row_tiles);
  return hipGetLastError();
}

template <typename T, int DP>
hipError_t launch_rows(const AttnArgs& a, hipStream_t st) {
  return attn_few(a) ? launch<T, DP, 1, 2, 64>(a, st) : launch<T, DP, 4, 1, sizeof(T) == 2 ? 64 : 32>(a, st);
}
template <typename T>
hipError_t launch_d(const AttnArgs& a, hipStream_t st) {
  switch (attn_dp(a.d)) {
    case 32: return launch_rows<T, 32>(a, st);
    case 64: return launch_rows<T, 64>(a, st);
    case 96: return launch_rows<T, 96>(a, st);
    default: return launch_rows<T, 128>(a, st);
  }
}

}  // namespace

bool attn_few(const AttnArgs& a) { return a.rows <= 64; }

// Parts of the key axis: so many that there are about 1024 workgroups, none of fewer than 4 tiles of 64 keys.
int attn_parts(const AttnArgs& a) {
  const int tile = attn_few(a) ? 32 : 128;
  const long long wgs = (long long)a.batch * a.kv * ((a.rows + tile - 1) / tile);
  const long long keys = std::min<long long>(a.m, (long long)a.window + a.sinks + tile / a.group);
  return (int)std::max<long long>(1, std::min<long long>({1024 / wgs, keys / 256, 256}));
}

hipError_t attn_forward_launch(const AttnArgs& a, hipStream_t st) {
  const hipError_t e = a.dt == 0 ? launch_d<float>(a, st) : launch_d<bf16_t>(a, st);
  if (e != hipSuccess || a.parts == 1) return e;
  const dim3 grid((unsigned)(a.batch * a.kv * a.rows));
  // (one row of 128 parts: 13 us with 8 groups, 7.5 with 32)
  if (a.parts <= 16) {
    if (a.dt == 0) hipLaunchKernelGGL((attn_join_kernel<float, 8>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((attn_join_kernel<bf16_t, 8>), grid, dim3(256), 0, st, a);
  } else {
    if (a.dt == 0) hipLaunchKernelGGL((attn_join_kernel<float, 32>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((attn_join_kernel<bf16_t, 32>), grid, dim3(1024), 0, st, a);
  }
  return hipGetLastError();
}

}  // namespace psgdk
