// Softmax cross entropy: the kernels around the products with the vocabulary matrix.
#include <type_traits>

#include "xent.h"

namespace psgdk {

// a thread's share of the rows that count, eight loads at a time
__device__ __forceinline__ int count_rows(const int64_t* target, long long rows, int64_t ignore) {
  int n = 0;
  for (long long r0 = threadIdx.x; r0 < rows; r0 += 8 * (long long)blockDim.x) {
    int64_t t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = target[min(r0 + k * (long long)blockDim.x, rows - 1)];
#pragma unroll
    for (int k = 0; k < 8; ++k) n += r0 + k * (long long)blockDim.x < rows && t[k] != ignore;
  }
  return n;
}
// of one workgroup: 1 / the number of rows that count, or 1
__device__ __forceinline__ float count_weight(const int64_t* target, long long rows, int64_t ignore, int mean) {
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  const int n = mean ? count_rows(target, rows, ignore) : 0;
  if (n) atomicAdd(&total, n);  // whole numbers: any order gives the same sum
  __syncthreads();
  return mean ? 1.f / (float)max(total, 1) : 1.f;
}
// The ignored rows' share of the products is saved by numbering the rows that count (1531 x 770 x 50021, half of them
// ignored: 542 -> 420 us in all). One workgroup, 4096 rows a turn (a wave 256 of them, 64 by 64): first how many count, then their places.
__global__ void __launch_bounds__(1024) xent_order_kernel(const int64_t* target, long long rows, int64_t ignore, int mean,
                                                          int* order, int* count, float* weight, float* loss) {
  __shared__ int total, part[2][16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  int n = count_rows(target, rows, ignore);
  if (n) atomicAdd(&total, n);  // whole numbers: any order gives the same sum
  __syncthreads();
  n = total;
  if (threadIdx.x == 0) {
    count[0] = n;
    weight[0] = mean ? 1.f / (float)max(n, 1) : 1.f;
  }
  int before = 0;  // rows that count, in front of this turn
  for (long long r0 = 0; r0 < rows; r0 += 4096) {
    const int turn = (int)(r0 / 4096 & 1);
    unsigned long long has[4];
    int64_t t[4];
    int mine = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = target[min(r0 + wave * 256 + e * 64 + lane, rows - 1)];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      has[e] = __ballot(r0 + wave * 256 + e * 64 + lane < rows && t[e] != ignore);
      mine += __popcll(has[e]);
    }
    if (lane == 0) part[turn][wave] = mine;
    __syncthreads();  // (the next turn's values lie beside these: one barrier a turn)
    int at = before;
    for (int w = 0; w < 16; ++w) {
      at += w < wave ? part[turn][w] : 0;
      before += part[turn][w];
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long long r = r0 + wave * 256 + e * 64 + lane;
      const int rank = at + __popcll(has[e] & ((1ull << lane) - 1));
      if (r < rows) {
        if (has[e] >> lane & 1) {
          order[rank] = (int)r;
        } else {
          order[n + (r - rank)] = (int)r;
          loss[r] = 0.f;
        }
      }
      at += __popcll(has[e]);
    }
  }
}
hipError_t xent_order_launch(const int64_t* target, long long rows, int64_t ignore, int mean, int* order, int* count,
                             float* weight, float* loss, hipStream_t st) {
  hipLaunchKernelGGL(xent_order_kernel, dim3(1), dim3(1024), 0, st, target, rows, ignore, mean, order, count, weight, loss);
  return hipGetLastError();
}

__global__ void __launch_bounds__(1024) xent_mean_kernel(const float* loss, const float* row_weight, const float* weight,
                                                         const int64_t* target, long long rows, int64_t ignore,
                                                         int mean, float* out) {
  __shared__ float red[16];
  const float w = row_weight ? 1.f : weight ? weight[0] : count_weight(target, rows, ignore, mean);
  float s = 0.f;
  for (long long r0 = threadIdx.x; r0 < rows; r0 += 8 * 1024) {  // eight loads at a time
    float v[8], g[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const long long i = min(r0 + k * 1024, rows - 1);
      v[k] = loss[i];
      g[k] = row_weight ? row_weight[i] : 1.f;
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) s += r0 + k * 1024 < rows ? g[k] * v[k] : 0.f;
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) out[0] = s * w;
}
hipError_t xent_mean_launch(const float* loss, const float* row_weight, const float* weight, const int64_t* target,
                            long long rows, int64_t ignore, int mean, float* out, hipStream_t st) {
  hipLaunchKernelGGL(xent_mean_kernel, dim3(1), dim3(1024), 0, st, loss, row_weight, weight, target, rows, ignore, mean,
                     out);
  return hipGetLastError();
}

// One workgroup a row: its maximum and sum in one pass (each thread keeps a running maximum and the sum of
// exponentials under it, four values at a time), the gradient in a second one. The target's own term stays out of the
// sum S of the others: with e_t its exponential, softmax_t - 1 = -S / (S + e_t) and, where the target is the maximum,
// loss = log(1 + S), both without a difference of near numbers. Bound by memory: 2048 x 10007 in 48 us (twice read, once
// written: 5.1 TB/s).
// The products read whole vectors and take another path where they meet a value that is not finite, also behind the
// vocabulary's end: no stale memory may lie there.
template <int TH>
__device__ __forceinline__ void xent_row(const XentRowsArgs& a, long long row, float* red) {
  constexpr float L2E = 1.4426950408889634f;
  float* const z = a.z + row * a.ldz;
  float4* const z4 = reinterpret_cast<float4*>(z);
  const int n4 = (int)(a.ldz / 4);
  const int64_t t = a.target[row];
  const bool skip = t == a.ignore, foreign = !skip && (t < 0 || t >= a.vocab);
  // (agent scope: the workgroup that adds the losses may be on another XCD)
  auto put_loss = [&](float v) { __hip_atomic_store(a.loss + row, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); };
  auto put = [&](int i, const float (&x)[4]) {
    if (a.dz) *reinterpret_cast<uint2*>(a.dz + row * a.ldq + 4 * i) = make_uint2(pack2_bf16(x[0], x[1]), pack2_bf16(x[2], x[3]));
    else z4[i] = make_float4(x[0], x[1], x[2], x[3]);
  };
  const int out4 = a.dz ? (int)(a.ldq / 4) : n4;
  if (skip || foreign) {
    const float fill = skip ? 0.f : NAN, x[4] = {fill, fill, fill, fill};
    if (threadIdx.x == 0) put_loss(fill);
    if (a.grad)
      for (int i = threadIdx.x; i < out4; i += TH) put(i, x);
    return;
  }
  const float zt = z[t];
  auto other = [&](int i, float (&x)[4]) {  // four logits, the target and what lies behind the vocabulary left out
    const float4 q = z4[i];
    const float v[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = 4 * i + e < a.vocab && 4 * i + e != t ? v[e] : -INFINITY;
  };
  float m = -INFINITY, s = 0.f;
  for (int i = threadIdx.x; i < n4; i += TH) {
    float x[4];
    other(i, x);
    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    if (top > m) {
      s *= __builtin_amdgcn_exp2f((m - top) * L2E);
      m = top;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s += x[e] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x[e] - m) * L2E);
  }
  const float most = fmaxf(block_max(m, red), zt);
  s = block_sum(m > -INFINITY ? s * __builtin_amdgcn_exp2f((m - most) * L2E) : s, red);
  const float et = __builtin_amdgcn_exp2f((zt - most) * L2E), all = s + et;
  const float over = most - zt;  // (an infinite logit that is both has no loss: inf - inf)
  if (threadIdx.x == 0) put_loss(over == 0.f ? log1pf(s) : logf(all) + over);
  if (!a.grad) return;
  const float w = a.row_weight ? a.row_weight[row] : a.dz ? 1.f : a.weight[0], q = w / all;
  for (int i = threadIdx.x; i < out4; i += TH) {
    const float4 v = i < n4 ? z4[i] : make_float4(0.f, 0.f, 0.f, 0.f);
    float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int c = 4 * i + e;
      x[e] = c >= a.vocab ? 0.f : c == t ? -s * q : __builtin_amdgcn_exp2f((x[e] - most) * L2E) * q;
    }
    put(i, x);
  }
}
template <int TH>
__global__ void __launch_bounds__(TH) xent_rows_kernel(const XentRowsArgs a) {
  __shared__ float red[16];
  __shared__ bool last;
  xent_row<TH>(a, blockIdx.x, red);
  if (!a.mean_loss) return;
  if (threadIdx.x == 0)
    last = __hip_atomic_fetch_add(a.done, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) + 1 == a.all_rows;
  __syncthreads();
  if (!last) return;
  float s = 0.f;
  for (long long i = threadIdx.x; i < a.all_rows; i += TH) {
    const float v = __hip_atomic_load(a.all_loss + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s += a.all_weight ? a.all_weight[i] * v : v;
  }
  s = block_sum(s, red);
  if (threadIdx.x == 0) a.mean_loss[0] = a.all_weight ? s : s * a.weight[0];
}
// Threads a row: 1024 from 4096 columns on, else 256.
hipError_t xent_rows_launch(const XentRowsArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.rows);
  if (a.vocab >= 4096) hipLaunchKernelGGL(xent_rows_kernel<1024>, grid, dim3(1024), 0, st, a);
  else hipLaunchKernelGGL(xent_rows_kernel<256>, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

__global__ void __launch_bounds__(256) sum_parts_kernel(const float* in, int parts, long long n4, float* out) {
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long long)gridDim.x * 256) {
    float4 v = reinterpret_cast<const float4*>(in)[i];
    for (int s = 1; s < parts; ++s) {
      const float4 q = reinterpret_cast<const float4*>(in)[s * n4 + i];
      v.x += q.x;
      v.y += q.y;
      v.z += q.z;
      v.w += q.w;
    }
    reinterpret_cast<float4*>(out)[i] = v;
  }
}
hipError_t sum_parts_launch(const float* in, int parts, long long n4, float* out, hipStream_t st) {
  const long long want = (n4 + 255) / 256;
  hipLaunchKernelGGL(sum_parts_kernel, dim3((unsigned)(want > 4096 ? 4096 : want)), dim3(256), 0, st, in, parts, n4, out);
  return hipGetLastError();
}

__global__ void __launch_bounds__(256) to_bf16_rows_kernel(const float* in, int splits, long long ldi,
                                                           const float* alpha, bf16_t* out, long long ldo,
                                                           long long rows, int d, const int* order, const int* count,
                                                           long long first) {
  const float al = alpha ? *alpha : 1.f;
  const int per = (d + 3) / 4;
  const long long total = (order ? min(max(count[0] - first, 0ll), rows) : rows) * per;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / per;
    const int c = (int)(i - r * per) * 4;
    float v[4] = {};
    for (int s = 0; s < splits; ++s) {
      const float* q = in + (s * rows + r) * ldi + c;
      if (c + 4 <= d) {
        float t[4];
        __builtin_memcpy(t, q, 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] += t[e];
      } else {
        for (int e = 0; c + e < d; ++e) v[e] += q[e];
      }
    }
    bf16_t h[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = f32_to_bf16(al * v[e]);
    bf16_t* o = out + (order ? order[r] : r) * ldo + c;
    if (c + 4 <= d) __builtin_memcpy(o, h, 8);
    else
      for (int e = 0; c + e < d; ++e) o[e] = h[e];
  }
}
hipError_t to_bf16_rows_launch(const float* in, int splits, long long ldi, const float* alpha, bf16_t* out, long long ldo,
                               long long rows, int d, const int* order, const int* count, long long first,
                               hipStream_t st) {
  const long long want = (rows * ((d + 3) / 4) + 255) / 256;
  hipLaunchKernelGGL(to_bf16_rows_kernel, dim3((unsigned)(want > 8192 ? 8192 : want)), dim3(256), 0, st, in, splits, ldi,
                     alpha, out, ldo, rows, d, order, count, first);
  return hipGetLastError();
}

// 8 consecutive values c .. c + 7 of a row of d (zeros behind it) at any element alignment
__device__ __forceinline__ uint4 ld8_bits(const bf16_t* row, int c, int d) {
  uint4 v = make_uint4(0, 0, 0, 0);
  if (c + 8 <= d) {
    __builtin_memcpy(&v, row + c, 16);
  } else {
    uint32_t w[4] = {};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < d) w[e / 2] |= (uint32_t)row[c + e] << (16 * (e & 1));
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return v;
}
__device__ __forceinline__ float dot8(uint4 a, uint4 b, float s) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s += __uint_as_float(x[i] << 16) * __uint_as_float(y[i] << 16);
    s += __uint_as_float(x[i] & 0xffff0000u) * __uint_as_float(y[i] & 0xffff0000u);
  }
  return s;
}

__global__ void __launch_bounds__(256) pad_rows_kernel(const bf16_t* in, long long ldi, bf16_t* out, long long ldo,
                                                       long long rows, int d) {
  const int per = (int)(ldo / 8);
  const long long total = rows * per;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / per;
    const int c = (int)(i - r * per) * 8;
    *reinterpret_cast<uint4*>(out + r * ldo + c) = ld8_bits(in + r * ldi, c, d);
  }
}
hipError_t pad_rows_launch(const bf16_t* in, long long ldi, bf16_t* out, long long ldo, long long rows, int d,
                           hipStream_t st) {
  const long long want = (rows * (ldo / 8) + 1023) / 1024;
  hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)(want > 16384 ? 16384 : want)), dim3(256), 0, st, in, ldi, out, ldo,
                     rows, d);
  return hipGetLastError();
}

// rows of a slab that are there
__device__ __forceinline__ long long live_rows(const XentBf16Args& a) {
  return min(max(a.count[0] - a.first, 0ll), a.rows);
}

// One wave a row: r = z_t and the row's copy for the products; zeros for an ignored row's gradient.
__global__ void __launch_bounds__(256) xent_prep_kernel(const XentBf16Args a) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.rows) return;
  if (lane == 0) {
    if (row % kXgRows == 0) a.mark[row / kXgRows] = 0;
    if (row == 0) a.redo[0] = 0;
  }
  const long long from = a.order[row];
  if (row >= live_rows(a)) {
    if (!a.dx) return;
    bf16_t* const o = a.dx + from * a.lddx;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c = lane * 8; c < a.d; c += 512)
      if (c + 8 <= a.d) __builtin_memcpy(o + c, &zero, 16);
      else
        for (int e = c; e < a.d; ++e) o[e] = 0;
    return;
  }
  const int64_t t = a.target[from];
  const bool foreign = t < 0 || t >= a.vocab;
  const bf16_t* x = a.x + from * a.ldx;
  const bf16_t* w = a.w + (foreign ? 0 : t) * a.ldw;
  float s = 0.f;
  for (int c = lane * 8; c < a.ldm; c += 512) {
    const uint4 v = ld8_bits(x, c, a.d);
    s = dot8(v, ld8_bits(w, c, a.d), s);
    *reinterpret_cast<uint4*>(a.xm + row * a.ldm + c) = v;
  }
  s = wave_sum(s);
  if (lane) return;
  if (foreign) s = NAN;
  a.zt[row] = s;
  a.ref[row] = s;
  a.col[row] = foreign ? a.vocab : (int)t;
}
hipError_t xent_prep_launch(const XentBf16Args& a, hipStream_t st) {
  hipLaunchKernelGGL(xent_prep_kernel, dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError();
}

// S and loss of a row from its parts, by one wave
__device__ __forceinline__ float join_row(const XentBf16Args& a, long long row, int lane) {
  float s = 0.f;
  for (int i = lane; i < a.parts; i += 64) s += a.sums[row * a.parts + i];
  s = wave_sum(s);
  if (lane == 0) {
    const float under = a.zt[row] - a.ref[row];  // 0 where r is the target's logit
    a.loss[a.order[row]] = under == 0.f ? log1pf(s) : logf(s + expf(under)) - under;
  }
  return s;
}
// One wave a row. A NaN sum is under no limit and stays.
__global__ void __launch_bounds__(256) xent_join_kernel(const XentBf16Args a, int again) {
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= live_rows(a) || (again && (a.redo[0] == 0 || !(a.sum[row] > kSumLimit)))) return;
  float s = join_row(a, row, lane);
  if (lane) return;
  // a target of -inf is no reference: others of -inf made this sum a NaN
  if (!again && a.zt[row] == -INFINITY) s = INFINITY;
  a.sum[row] = s;
  if (!again && s > kSumLimit) {
    const int blk = (int)(row / kXgRows);
    if (atomicExch(&a.mark[blk], 1) == 0) a.redo[1 + atomicAdd(&a.redo[0], 1)] = blk;  // the list's order is free
  }
}
hipError_t xent_join_launch(const XentBf16Args& a, int again, hipStream_t st) {
  hipLaunchKernelGGL(xent_join_kernel, dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a, again);
  return hipGetLastError();
}

__global__ void __launch_bounds__(256) xent_top_kernel(const XentBf16Args a) {
  if (a.redo[0] == 0) return;
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= live_rows(a) || !(a.sum[row] > kSumLimit)) return;
  float m = -INFINITY;
  for (int i = lane; i < a.parts; i += 64) m = fmaxf(m, a.sums[row * a.parts + i]);
  m = wave_max(m);
  if (lane == 0) a.ref[row] = m;
}
hipError_t xent_top_launch(const XentBf16Args& a, hipStream_t st) {
  hipLaunchKernelGGL(xent_top_kernel, dim3((unsigned)((a.rows + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError();
}

// One workgroup a row, in place: the coded logits become softmax - [v = t], each rounded to bf16 once. The step of 2^-9
// between codes moves a softmax entry by at most 2^-10, half of what that rounding may. A pass of its own, and not
// exponentials stored by the logits' product as the next products' operands (scaled rows instead): those are rounded before
// the row's sum is known, so the gradients' error was .0029-.0034 where this has .0018 and torch's own bf16 path .0017.
// Bound by memory: 4096 x 131072 in 439 us, 4.9 TB/s.
__global__ void __launch_bounds__(256) xent_dz_kernel(const XentBf16Args a) {
  const long long row = blockIdx.x;
  uint4* q = reinterpret_cast<uint4*>(a.q + row * a.ldq);
  if (row >= live_rows(a)) return;
  const int n = (int)(a.ldq / 8), t = a.col[row];
  __shared__ float again;
  float s = a.sum[row];
  if (s > kSumLimit) {  // a row whose reference was too low: its sums were made again
    if (threadIdx.x < 64) {
      const float q = join_row(a, row, threadIdx.x);
      if (threadIdx.x == 0) again = q;
    }
    __syncthreads();
    s = again;
  }
  const float all = s + expf(a.zt[row] - a.ref[row]), g = a.row_weight ? a.row_weight[a.order[row]] : 1.f;
  constexpr float L2E = 1.4426950408889634f;
  const float k0 = (kLogitLow + 64.f) * L2E - log2f(all), k1 = kLogitStep * L2E;
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint4 v = q[i];
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = 8 * i + 2 * j;
      float lo = g * __builtin_amdgcn_exp2f(__builtin_fmaf((float)(int16_t)(w[j] & 0xffff), k1, k0));
      float hi = g * __builtin_amdgcn_exp2f(__builtin_fmaf((float)((int32_t)w[j] >> 16), k1, k0));
      lo = c >= a.vocab ? 0.f : c == t ? -g * (s / all) : lo;
      hi = c + 1 >= a.vocab ? 0.f : c + 1 == t ? -g * (s / all) : hi;
      w[j] = pack2(f32_to_bf16(lo), f32_to_bf16(hi));
    }
    q[i] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}
hipError_t xent_dz_launch(const XentBf16Args& a, hipStream_t st) {
  hipLaunchKernelGGL(xent_dz_kernel, dim3((unsigned)a.rows), dim3(256), 0, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// Up to 64 rows, losses only. A wave takes 16 MV rows of the vocabulary at a time against NB blocks of 16 rows of x on
// 16 x 16 x 32 MFMAs (A: vocabulary, B: x), both operands straight from memory: W's bytes are all that counts. Lane l
// holds the logits of row l % 16 of x and vocabulary rows 4 (l / 16) .. + 3 of a tile, and keeps a running maximum and
// the sum of exponentials under it; the lanes' and waves' pairs join at the end. Bound by memory, the vocabulary matrix
// read once: 1 row against 131072 x 4096 in 204 us, 5.25 TB/s (as fast as a copy). MV 4 with the loads of 4 k steps ahead
// of their products; 8 steps took 228 us, 32 vocabulary rows a wave 218, nontemporal loads 280.
template <int MV, int NB>
__global__ void __launch_bounds__(256) xent_few_kernel(const XentFewArgs a) {
  constexpr int UK = 4;
  __shared__ float2 red[4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  float top[NB], sum[NB];
  int t[NB];
  const bf16_t* xr[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int n = b * 16 + r;
    top[b] = -INFINITY;
    sum[b] = 0.f;
    const int64_t tt = n < a.rows ? a.target[n] : -1;
    t[b] = tt >= 0 && tt < a.vocab ? (int)tt : -1;
    xr[b] = a.x + (long long)min(n, a.rows - 1) * a.ldx;
  }
  for (int v0 = (blockIdx.x * 4 + wave) * 16 * MV; v0 < a.vocab; v0 += gridDim.x * 4 * 16 * MV) {
    f32x4_t acc[MV][NB];
#pragma unroll
    for (int i = 0; i < MV; ++i)
#pragma unroll
      for (int b = 0; b < NB; ++b) acc[i][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const bf16_t* wr[MV];
#pragma unroll
    for (int i = 0; i < MV; ++i) wr[i] = a.w + (long long)min(v0 + 16 * i + r, a.vocab - 1) * a.ldw;
    // U steps of 32 k at a time: their loads all go out before the first product
    auto steps = [&](auto count, int k) {
      constexpr int U = decltype(count)::value;
      bf16x8_t fx[U][NB], fw[U][MV];
#pragma unroll
      for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < MV; ++i) __builtin_memcpy(&fw[u][i], wr[i] + k + 32 * u + 8 * g, 16);
#pragma unroll
        for (int b = 0; b < NB; ++b) __builtin_memcpy(&fx[u][b], xr[b] + k + 32 * u + 8 * g, 16);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < MV; ++i)
#pragma unroll
          for (int b = 0; b < NB; ++b)
            acc[i][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw[u][i], fx[u][b], acc[i][b], 0, 0, 0);
    };
    const int whole = a.d & ~31;
    int k = 0;
    for (; k + 32 * UK <= whole; k += 32 * UK) steps(std::integral_constant<int, UK>{}, k);
    for (; k < whole; k += 32) steps(std::integral_constant<int, 1>{}, k);
    if (whole < a.d) {
#pragma unroll
      for (int i = 0; i < MV; ++i) {
        const uint4 wv = ld8_bits(wr[i], whole + 8 * g, a.d);
        bf16x8_t fw;
        __builtin_memcpy(&fw, &wv, 16);
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const uint4 xv = ld8_bits(xr[b], whole + 8 * g, a.d);
          bf16x8_t fx;
          __builtin_memcpy(&fx, &xv, 16);
          acc[i][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fw, fx, acc[i][b], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < MV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int v = v0 + 16 * i + 4 * g + e;
          const float z = acc[i][b][e];
          if (v == t[b]) {
            a.zt[b * 16 + r] = z;
          } else if (v < a.vocab) {
            if (z != z) sum[b] = NAN;
            if (z > top[b]) {
              sum[b] *= expf(top[b] - z);
              top[b] = z;
            }
            if (z > -INFINITY) sum[b] += expf(z - top[b]);
          }
        }
  }
  auto join = [](float2 p, float2 q) {  // -inf and a sum of 0 (or NaN) where there is nothing
    const float m = fmaxf(p.x, q.x);
    const float f = p.x > -INFINITY ? expf(p.x - m) : 1.f, h = q.x > -INFINITY ? expf(q.x - m) : 1.f;
    return make_float2(m, p.y * f + q.y * h);
  };
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float2 p = make_float2(top[b], sum[b]);
#pragma unroll
    for (int o = 16; o < 64; o <<= 1) p = join(p, make_float2(__shfl_xor(p.x, o, 64), __shfl_xor(p.y, o, 64)));
    if (g == 0) red[wave][b * 16 + r] = p;
  }
  __syncthreads();
  if (threadIdx.x < 16 * NB) {
    float2 p = red[0][threadIdx.x];
    for (int i = 1; i < 4; ++i) p = join(p, red[i][threadIdx.x]);
    a.part[(long long)blockIdx.x * 64 + threadIdx.x] = p;
  }
}
__global__ void __launch_bounds__(256) xent_few_join_kernel(const XentFewArgs a) {
  __shared__ float red[16];
  const int n = blockIdx.x;
  const int64_t t = a.target[n];
  float top = -INFINITY;
  for (int i = threadIdx.x; i < a.wgs; i += 256) top = fmaxf(top, a.part[(long long)i * 64 + n].x);
  top = block_max(top, red);
  float s = 0.f;
  for (int i = threadIdx.x; i < a.wgs; i += 256) {
    const float2 p = a.part[(long long)i * 64 + n];
    s += p.x > -INFINITY ? p.y * expf(p.x - top) : p.y;
  }
  s = block_sum(s, red);
  if (threadIdx.x) return;
  float loss;
  if (t == a.ignore) {
    loss = 0.f;
  } else if (t < 0 || t >= a.vocab) {
    loss = NAN;
  } else {
    const float zt = a.zt[n], m = fmaxf(top, zt), over = m - zt, rest = top > -INFINITY ? s * expf(top - m) : s;
    loss = over == 0.f ? log1pf(rest) : logf(rest + expf(zt - m)) + over;  // (NaN where over is: inf - inf, or a NaN z_t)
  }
  a.loss[n] = loss;
}
// Blocks of vocabulary rows a wave takes at a time (MV): as many of 4, 2 or 1 as still give work to three quarters of the
// CUs. us with 4 / 2 / 1: 1 row against 131072 x 4096 207 / - / 224; 32 rows against 50021 x 1024 38 / - / 52, against
// 32768 x 1024 37 / 26 / 32.
static int few_blocks(int64_t vocab) { return vocab >= 192 * 256 ? 4 : vocab >= 192 * 128 ? 2 : 1; }
int xent_few_rows(int64_t vocab) { return few_blocks(vocab) == 4 ? 32 : 64; }
int xent_few_wgs(int vocab) {
  const int per = 64 * few_blocks(vocab), want = (vocab + per - 1) / per;  // 64: four waves' blocks of 16
  return want > 1024 ? 1024 : want;
}
hipError_t xent_few_launch(const XentFewArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.wgs);
#define PSGDK_FEW(MV, NB) hipLaunchKernelGGL((xent_few_kernel<MV, NB>), grid, dim3(256), 0, st, a)
  switch (few_blocks(a.vocab)) {
    case 4:
      if (a.rows <= 16) PSGDK_FEW(4, 1);
      else PSGDK_FEW(4, 2);
      break;
    case 2:
      if (a.rows <= 16) PSGDK_FEW(2, 1);
      else if (a.rows <= 32) PSGDK_FEW(2, 2);
      else PSGDK_FEW(2, 4);
      break;
    default:
      if (a.rows <= 16) PSGDK_FEW(1, 1);
      else if (a.rows <= 32) PSGDK_FEW(1, 2);
      else PSGDK_FEW(1, 4);
  }
#undef PSGDK_FEW
  hipLaunchKernelGGL(xent_few_join_kernel, dim3((unsigned)a.rows), dim3(256), 0, st, a);
  return hipGetLastError();
}

// one wave a row
template <typename T>
__global__ void __launch_bounds__(256) xent_copy_kernel(const XentCopyArgs a) {
  if (a.weight && blockIdx.x == 0) {
    const float w = count_weight(a.all_targets, a.all_rows, a.ignore, a.mean);
    if (threadIdx.x == 0) {
      a.weight[0] = w;
      a.count[0] = (int)a.rows;
      a.done[0] = 0;
    }
  }
  const int lane = threadIdx.x & 63;
  const long long row = (long long)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (row >= a.rows) return;
  const bool skip = a.target[row] == a.ignore;
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  T* m = reinterpret_cast<T*>(a.xm) + row * a.ldm;
  if constexpr (sizeof(T) == 2) {
    for (int c = lane * 8; c < a.ldm; c += 512)
      *reinterpret_cast<uint4*>(m + c) = skip ? make_uint4(0, 0, 0, 0) : ld8_bits(x, c, a.d);
  } else {
    for (int c = lane * 4; c < a.d; c += 256) {
      if (c + 4 <= a.d) {
        float v[4];
        __builtin_memcpy(v, x + c, 16);
#pragma unroll
        for (float& e : v) e = skip ? 0.f : e;
        __builtin_memcpy(m + c, v, 16);
      } else {
        for (int e = c; e < a.d; ++e) m[e] = skip ? 0.f : x[e];
      }
    }
  }
}
hipError_t xent_copy_launch(const XentCopyArgs& a, int dt, hipStream_t st) {
  const dim3 grid((unsigned)((a.rows + 3) / 4));
  if (dt == 1) hipLaunchKernelGGL(xent_copy_kernel<bf16_t>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(xent_copy_kernel<float>, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

template <typename T>
__global__ void __launch_bounds__(256) scale_by_kernel(const ScaleArgs a) {
  const float s = *a.scale;
  if (s == 1.f) return;
  for (int b = 0; b < a.nb; ++b) {
    T* x = reinterpret_cast<T*>(a.x[b]);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < a.n[b]; i += (long long)gridDim.x * 256)
      x[i] = from_f32<T>(to_f32<T>(x[i]) * s);
  }
}
hipError_t scale_by_launch(const ScaleArgs& a, int dt, hipStream_t st) {
  long long n = 1;
  for (int b = 0; b < a.nb; ++b) n = n > a.n[b] ? n : a.n[b];
  const long long want = (n + 1023) / 1024;
  const dim3 grid((unsigned)(want > 4096 ? 4096 : want));
  if (dt == 1) hipLaunchKernelGGL(scale_by_kernel<bf16_t>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(scale_by_kernel<float>, grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace psgdk
