// Norms of queries and keys for each head, their weights and the position rotation, one pass each way.
#include <type_traits>

#include "rope.h"

namespace psgdk {

namespace {

template <typename T, int V>
__device__ __forceinline__ void ld_vec(const T* p, float (&x)[V]) {
  if constexpr (sizeof(T) == 4 && V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const f32x4_t v = *reinterpret_cast<const f32x4_t*>(p + i);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[i + e] = v[e];
    }
  } else if constexpr (V >= 4) {
    uint32_t w[V / 2];
    __builtin_memcpy(w, __builtin_assume_aligned(p, 2 * V), 2 * V);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    x[0] = to_f32<T>(p[0]);
  }
}
template <typename T, int V>
__device__ __forceinline__ void st_vec(T* p, const float (&x)[V]) {
  if constexpr (sizeof(T) == 4 && V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<f32x4_t*>(p + i) = f32x4_t{x[i], x[i + 1], x[i + 2], x[i + 3]};
  } else if constexpr (V >= 4) {
    uint32_t w[V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i) w[i] = pack2_bf16(x[2 * i], x[2 * i + 1]);
    __builtin_memcpy(__builtin_assume_aligned(p, 2 * V), w, 2 * V);
  } else {
    p[0] = from_f32<T>(x[0]);
  }
}

// Cosine and sine of a fraction of a turn in 64-bit fixed point: the nearest quarter turn taken off as an integer, so that the
// rest, at most an eighth, loses nothing as a float; then the Taylor series to x^9 and x^10 (next terms below 2^-29).
__device__ __forceinline__ void turn(uint64_t t, float& c, float& s) {
  const uint32_t hi = (uint32_t)(t >> 32), q = (hi + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(hi - (q << 30)) * 1.46291807926715968e-9f, z = x * x;  // 2 pi / 2^32
  float sn = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
  sn = __builtin_fmaf(z, sn, 8.33333333e-3f);
  sn = __builtin_fmaf(z, sn, -1.66666667e-1f);
  sn = __builtin_fmaf(z * x, sn, x);
  float cs = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
  cs = __builtin_fmaf(z, cs, -1.38888889e-3f);
  cs = __builtin_fmaf(z, cs, 4.16666667e-2f);
  cs = __builtin_fmaf(z, cs, -.5f);
  cs = __builtin_fmaf(z, cs, 1.f);
  const float a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
  c = (q + 1) & 2 ? -a : a;
  s = q & 2 ? -b : b;
}

// sum over `lanes` (a power of two) lanes that lie together, every lane getting it
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
  if (lanes > 1) v += dpp<0xB1>(v);
  if (lanes > 2) v += dpp<0x4E>(v);
  if (lanes > 4) v += dpp<0x141>(v);
  if (lanes > 8) v += dpp<0x140>(v);
  if (lanes > 16) v += __shfl_xor(v, 16, 64);
  if (lanes > 32) v += __shfl_xor(v, 32, 64);
  return v;
}

template <typename T>
__device__ __forceinline__ const T* head_of(const RopeSide& x, long long b, long long i, int head) {
  return x.p ? static_cast<const T*>(x.p) + b * x.sb + i * x.sn + head * x.sh : nullptr;
}

// A wave has a token (or `waves` waves share its heads), 64 / lanes heads at a time, so that the rotation's angles are made
// once for all heads. A lane has V pairs of elements S times: pair i of the rotated part is (i, i + rot / 2), or (2 i, 2 i + 1)
// interleaved, and of the rest, which is only normalised, (2 i, 2 i + 1). Forward: memory (4 x 4096 tokens, 32 + 8 heads of 128,
// bf16: 61 us, 5.5 TB/s). Backward the same bytes and half as much again in 119 us, 4.2 TB/s: the vector unit, and two row sums in
// series; with the next heads' loads on their way it took 167 of then 154, and queries apart from keys saved 13 (no weight and
// no sum is chosen by the lane).
template <typename T, int V, int S, bool INTER, bool BACK>
__global__ void __launch_bounds__(256) rope_kernel(const RopeArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int sub = lane & (a.lanes - 1), slot = lane / a.lanes, at_once = 64 / a.lanes;
  const int half = a.rot / 2, pairs = a.d / 2;
  const int q_steps = (a.heads + at_once - 1) / at_once, steps = q_steps + (a.all - a.heads + at_once - 1) / at_once;
  const float inv_d = 1.f / (float)a.d;

  int e0[S], e1[S];
  bool in[S];
  uint64_t rate[S][V];  // of the lane's pairs, turns a token in 64-bit fixed point
  float w[2][S][2 * V];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int i = (sub + s * a.lanes) * V;
    in[s] = i < pairs;
    const bool apart = !INTER && i < half;
    e0[s] = apart ? i : 2 * i;
    e1[s] = apart ? i + half : 2 * i + V;
    // theta^(-2 i / rot) / (2 pi) from the powers of theta^(-2 / rot), of which i has up to 5, 6 or 8 (8, 4 or 1 pairs a lane), and
    // the ratio for the pairs behind the first: each factor and product is off by 2^-53 at most, the rate by 25 of them. An angle
    // is right to float32's rounding up to position 2^24, and to p 2^-48 beyond.
    double f = 0.15915494309189535;
    for (int k = 0; k < kRopePowers; ++k) f *= i >> k & 1 ? a.ratio[k] : 1.0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      rate[s][v] = i < half ? (uint64_t)(f * 0x1p64) : 0;
      f *= a.ratio[0];
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
#pragma unroll
      for (int e = 0; e < 2 * V; ++e) w[k][s][e] = 1.f;
      if (!a.w[k].p || !in[s]) continue;
      float lo[V], hi[V];
      if (a.w[k].dt == 0) {
        ld_vec<float, V>(static_cast<const float*>(a.w[k].p) + e0[s], lo);
        ld_vec<float, V>(static_cast<const float*>(a.w[k].p) + e1[s], hi);
      } else {
        ld_vec<bf16_t, V>(static_cast<const bf16_t*>(a.w[k].p) + e0[s], lo);
        ld_vec<bf16_t, V>(static_cast<const bf16_t*>(a.w[k].p) + e1[s], hi);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) {
        w[k][s][e] = lo[e];
        w[k][s][V + e] = hi[e];
      }
    }
  }
  float dw[2][S][2 * V];
  if constexpr (BACK) {
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) dw[k][s][e] = 0.f;
  }
  // x and y of pair v of a lane's 2 V elements
  auto first = [](int v) { return INTER && V > 1 ? 2 * v : v; };
  auto second = [](int v) { return INTER && V > 1 ? 2 * v + 1 : V + v; };

  const unsigned work = (unsigned)a.tokens * a.waves, stride = gridDim.x * 4;  // (tokens below 2^31, with several waves below 2^14)
  for (unsigned at = blockIdx.x * 4 + wave; at < work; at += stride) {
    const unsigned tok = at / (unsigned)a.waves, seq = tok / (unsigned)a.n;
    const int part = at - tok * a.waves;
    const long long token = tok, b = seq, i = tok - seq * a.n;
    const uint64_t pos = (uint64_t)(a.pos ? a.pos[b * a.pos_sb + i] : i);
    float cs[S][V], sn[S][V];
#pragma unroll
    for (int s = 0; s < S; ++s)
#pragma unroll
      for (int v = 0; v < V; ++v) turn(pos * rate[s][v], cs[s][v], sn[s][v]);

    // heads `head` of the queries (K 0) or keys (K 1)
    auto heads = [&](auto which, int head) __attribute__((always_inline)) {
      constexpr int K = decltype(which)::value;
      const bool there = head < (K ? a.all - a.heads : a.heads);
      const T* const xp = head_of<T>(a.x[K], b, i, head);
      const T* gp = nullptr;
      if constexpr (BACK) gp = head_of<T>(a.dy[K], b, i, head);
      float x[S][2 * V], g[S][2 * V];
      float sum = 0.f, sq = 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s) {
        float lo[V], hi[V];
#pragma unroll
        for (int e = 0; e < V; ++e) lo[e] = hi[e] = 0.f;
        if (there && in[s]) {
          ld_vec<T, V>(xp + e0[s], lo);
          ld_vec<T, V>(xp + e1[s], hi);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
          x[s][e] = lo[e];
          x[s][V + e] = hi[e];
          sum += lo[e] + hi[e];
        }
        if constexpr (BACK) {
#pragma unroll
          for (int e = 0; e < V; ++e) lo[e] = hi[e] = 0.f;
          if (there && in[s] && gp) {
            ld_vec<T, V>(gp + e0[s], lo);
            ld_vec<T, V>(gp + e1[s], hi);
          }
#pragma unroll
          for (int e = 0; e < V; ++e) {
            g[s][e] = lo[e];
            g[s][V + e] = hi[e];
          }
        }
      }
      const float mean = a.norm == NORM_LAYER ? lanes_sum(sum, a.lanes) * inv_d : 0.f;
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          x[s][e] = in[s] ? x[s][e] - mean : 0.f;
          sq += x[s][e] * x[s][e];
        }
      float rstd = a.norm == NORM_NONE ? 1.f : 1.f / sqrtf(lanes_sum(sq, a.lanes) * inv_d + a.eps);
      // lanes without a head hold zeros, whose rstd is infinite where eps is 0: the weights' sums would get NaN
      if constexpr (BACK) rstd = there ? rstd : 0.f;

      float out[S][2 * V];
      if constexpr (!BACK) {
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const int p = first(v), q = second(v);
            const float u0 = x[s][p] * rstd * w[K][s][p], u1 = x[s][q] * rstd * w[K][s][q];
            out[s][p] = u0 * cs[s][v] - u1 * sn[s][v];
            out[s][q] = u1 * cs[s][v] + u0 * sn[s][v];
          }
      } else {
        float dot = 0.f, csum = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int v = 0; v < V; ++v) {
            const int p = first(v), q = second(v);
            const float u0 = g[s][p] * cs[s][v] + g[s][q] * sn[s][v], u1 = g[s][q] * cs[s][v] - g[s][p] * sn[s][v];
            x[s][p] *= rstd;  // the normalised values
            x[s][q] *= rstd;
            const float t0 = u0 * x[s][p], t1 = u1 * x[s][q];
            dw[K][s][p] += t0;
            dw[K][s][q] += t1;
            g[s][p] = u0 * w[K][s][p];
            g[s][q] = u1 * w[K][s][q];
            dot += g[s][p] * x[s][p] + g[s][q] * x[s][q];
            csum += g[s][p] + g[s][q];
          }
        if (a.norm != NORM_NONE) dot = lanes_sum(dot, a.lanes) * inv_d;
        else dot = 0.f;
        const float cmean = a.norm == NORM_LAYER ? lanes_sum(csum, a.lanes) * inv_d : 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
          for (int e = 0; e < 2 * V; ++e) out[s][e] = (g[s][e] - x[s][e] * dot - cmean) * rstd;
      }
      T* const base = static_cast<T*>(BACK ? a.dx[K] : a.y[K]);
      if (there && base) {
        T* const op = base + (token * (K ? a.all - a.heads : a.heads) + head) * a.d;
#pragma unroll
        for (int s = 0; s < S; ++s) {
          if (!in[s]) continue;
          float lo[V], hi[V];
#pragma unroll
          for (int e = 0; e < V; ++e) {
            lo[e] = out[s][e];
            hi[e] = out[s][V + e];
          }
          st_vec<T, V>(op + e0[s], lo);
          st_vec<T, V>(op + e1[s], hi);
        }
      }
    };
    for (int it = part * steps / a.waves; it < (part + 1) * steps / a.waves; ++it) {
      if (it < q_steps) heads(std::integral_constant<int, 0>{}, it * at_once + slot);
      else heads(std::integral_constant<int, 1>{}, (it - q_steps) * at_once + slot);
    }
  }

  if constexpr (BACK) {
    if (!a.part) return;
    // the heads that a wave had at once, then the four waves, in order
    __shared__ float red[4][kRopeMaxD];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      __syncthreads();
#pragma unroll
      for (int s = 0; s < S; ++s)
#pragma unroll
        for (int e = 0; e < 2 * V; ++e) {
          float v = dw[k][s][e];
          for (int o = a.lanes; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
          if (slot == 0 && in[s]) red[wave][(e < V ? e0[s] + e : e1[s] + e - V)] = v;
        }
      __syncthreads();
      float* const out = a.part + ((long long)k * a.parts + blockIdx.x) * a.d;
      for (int c = threadIdx.x; c < a.d; c += 256) out[c] = red[0][c] + red[1][c] + red[2][c] + red[3][c];
    }
  }
}

template <typename T, int V, int S, bool INTER>
hipError_t launch(const RopeArgs& a, bool backward, hipStream_t st) {
  const long long wgs = (a.tokens * a.waves + 3) / 4;
  if constexpr (V < 8) {
    if (backward) {
      hipLaunchKernelGGL((rope_kernel<T, V, S, INTER, true>), dim3(a.parts), dim3(256), 0, st, a);
      return hipGetLastError();
    }
  }
  hipLaunchKernelGGL((rope_kernel<T, V, S, INTER, false>), dim3((unsigned)std::min<long long>(wgs, 1 << 16)), dim3(256), 0, st, a);
  return hipGetLastError();
}
template <typename T>
hipError_t launch_t(const RopeArgs& a, bool backward, hipStream_t st) {
  if (a.pairs_lane == 8) return a.interleaved ? launch<T, 8, 1, true>(a, backward, st) : launch<T, 8, 1, false>(a, backward, st);
  if (a.pairs_lane == 4) return a.interleaved ? launch<T, 4, 1, true>(a, backward, st) : launch<T, 4, 1, false>(a, backward, st);
  return a.interleaved ? launch<T, 1, 4, true>(a, backward, st) : launch<T, 1, 4, false>(a, backward, st);
}

}  // namespace

void rope_plan(RopeArgs& a, bool backward, bool aligned16, bool aligned8) {
  // a lane's pairs are all rotated or none: pairs of the rotated part and of the rest come in whole vectors
  const int half = a.rot / 2, pairs = a.d / 2;
  const bool by8 = half % 8 == 0 && pairs % 8 == 0, by4 = half % 4 == 0 && pairs % 4 == 0;
  // (backward, 8 pairs a lane leave 2 waves a SIMD, 4 pairs 4: 141 and 119 us of 4 x 4096, 32 + 8 heads of 128 bf16)
  a.pairs_lane = by8 && aligned16 && !backward ? 8 : by4 && (a.dt == 0 ? aligned16 : aligned8) ? 4 : 1;
  const int need = (pairs + a.pairs_lane - 1) / a.pairs_lane;
  a.lanes = 1;
  while (a.lanes < need && a.lanes < 64) a.lanes *= 2;
  // all heads of a token on one wave where there are tokens enough to fill the GPU
  const int at_once = 64 / a.lanes;
  const int steps = (a.heads + at_once - 1) / at_once + (a.all - a.heads + at_once - 1) / at_once;
  a.waves = (int)std::max<long long>(1, std::min<long long>(steps, 8192 / std::max<long long>(a.tokens, 1)));
  a.parts = (int)std::min<long long>((a.tokens * a.waves + 3) / 4, kRopeParts);
}

hipError_t rope_launch(const RopeArgs& a, bool backward, hipStream_t st) {
  return a.dt == 0 ? launch_t<float>(a, backward, st) : launch_t<bf16_t>(a, backward, st);
}

}  // namespace psgdk
