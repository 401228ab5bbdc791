// Softmax cross entropy: the kernels around the products with the vocabulary matrix.
#include "xent.h"

namespace psgdk {

__global__ void __launch_bounds__(1024) xent_weight_kernel(const int64_t* target, long long rows, int64_t ignore,
                                                           int mean, float* weight) {
  __shared__ int total;
  if (threadIdx.x == 0) total = 0;
  __syncthreads();
  int n = 0;
  if (mean)
    for (long long i = threadIdx.x; i < rows; i += 1024) n += target[i] != ignore;
  atomicAdd(&total, n);  // whole numbers: any order gives the same sum
  __syncthreads();
  if (threadIdx.x == 0) weight[0] = mean ? 1.f / (float)max(total, 1) : 1.f;
}
hipError_t xent_weight_launch(const int64_t* target, long long rows, int64_t ignore, int mean, float* weight,
                              hipStream_t st) {
  hipLaunchKernelGGL(xent_weight_kernel, dim3(1), dim3(1024), 0, st, target, rows, ignore, mean, weight);
  return hipGetLastError();
}

__global__ void __launch_bounds__(1024) xent_mean_kernel(const float* loss, const float* row_weight, const float* weight,
                                                         long long rows, float* out) {
  __shared__ float red[16];
  float s = 0.f;
  for (long long i = threadIdx.x; i < rows; i += 1024) s += row_weight ? row_weight[i] * loss[i] : loss[i];
  s = block_sum(s, red);
  if (threadIdx.x == 0) out[0] = row_weight ? s : s * weight[0];
}
hipError_t xent_mean_launch(const float* loss, const float* row_weight, const float* weight, long long rows, float* out,
                            hipStream_t st) {
  hipLaunchKernelGGL(xent_mean_kernel, dim3(1), dim3(1024), 0, st, loss, row_weight, weight, rows, out);
  return hipGetLastError();
}

// One workgroup a row: its maximum and sum in one pass (each thread keeps a running maximum and the sum of
// exponentials under it), the gradient in a second one. The target's own term stays out of the sum S of the others:
// with e_t its exponential, softmax_t - 1 = -S / (S + e_t) and, where the target is the maximum, loss = log(1 + S),
// both without a difference of near numbers.
__global__ void __launch_bounds__(1024) xent_rows_kernel(const XentRowsArgs a) {
  __shared__ float red[16];
  const long long row = blockIdx.x;
  float* z = a.z + row * a.ldz;
  const int64_t t = a.target[row];
  // the products read whole vectors and take another path where they meet a value that is not finite, also behind the
  // vocabulary's end: no stale memory may lie there
  if (a.grad && threadIdx.x < a.ldz - a.vocab) z[a.vocab + threadIdx.x] = 0.f;
  if (t == a.ignore) {
    if (threadIdx.x == 0) a.loss[row] = 0.f;
    if (a.grad)
      for (int v = threadIdx.x; v < a.vocab; v += 1024) z[v] = 0.f;
    return;
  }
  if (t < 0 || t >= a.vocab) {
    if (threadIdx.x == 0) a.loss[row] = NAN;
    if (a.grad)
      for (int v = threadIdx.x; v < a.vocab; v += 1024) z[v] = NAN;
    return;
  }
  const float zt = z[t];
  float m = -INFINITY, s = 0.f;
  bool nan = false;
  for (int v = threadIdx.x; v < a.vocab; v += 1024) {
    const float x = z[v];
    nan = nan || x != x;
    if (x > m) {
      s *= expf(m - x);
      m = x;
    }
    if (v != t && x > -INFINITY) s += expf(x - m);
  }
  const float top = block_max(m, red);
  s = block_sum(nan ? NAN : (m > -INFINITY ? s * expf(m - top) : 0.f), red);
  const float et = expf(zt - top), all = s + et;
  if (threadIdx.x == 0) a.loss[row] = zt == top ? log1pf(s) : logf(all) + (top - zt);
  if (!a.grad) return;
  const float w = a.row_weight ? a.row_weight[row] : a.weight[0], q = w / all;
  __syncthreads();
  for (int v = threadIdx.x; v < a.vocab; v += 1024) z[v] = v == t ? -s * q : expf(z[v] - top) * q;
}
hipError_t xent_rows_launch(const XentRowsArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(xent_rows_kernel, dim3((unsigned)a.rows), dim3(1024), 0, st, a);
  return hipGetLastError();
}

__global__ void __launch_bounds__(256) to_bf16_rows_kernel(const float* in, long long ldi, bf16_t* out, long long ldo,
                                                           long long rows, int d) {
  const long long total = rows * d;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / d;
    const int c = (int)(i - r * d);
    out[r * ldo + c] = f32_to_bf16(in[r * ldi + c]);
  }
}
hipError_t to_bf16_rows_launch(const float* in, long long ldi, bf16_t* out, long long ldo, long long rows, int d,
                               hipStream_t st) {
  const long long want = (rows * d + 255) / 256;
  hipLaunchKernelGGL(to_bf16_rows_kernel, dim3((unsigned)(want > 8192 ? 8192 : want)), dim3(256), 0, st, in, ldi, out,
                     ldo, rows, d);
  return hipGetLastError();
}

template <typename T>
__global__ void __launch_bounds__(256) xent_mask_rows_kernel(const T* x, long long ldx, T* out, const int64_t* target,
                                                             int64_t ignore, long long rows, int d) {
  const long long total = rows * d;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long r = i / d;
    out[i] = target[r] == ignore ? from_f32<T>(0.f) : x[r * ldx + (i - r * d)];
  }
}
hipError_t xent_mask_rows_launch(const void* x, long long ldx, void* out, const int64_t* target, int64_t ignore,
                                 long long rows, int d, int dt, hipStream_t st) {
  const long long want = (rows * d + 255) / 256;
  const dim3 grid((unsigned)(want > 8192 ? 8192 : want));
  if (dt == 1)
    hipLaunchKernelGGL(xent_mask_rows_kernel<bf16_t>, grid, dim3(256), 0, st, reinterpret_cast<const bf16_t*>(x), ldx,
                       reinterpret_cast<bf16_t*>(out), target, ignore, rows, d);
  else
    hipLaunchKernelGGL(xent_mask_rows_kernel<float>, grid, dim3(256), 0, st, reinterpret_cast<const float*>(x), ldx,
                       reinterpret_cast<float*>(out), target, ignore, rows, d);
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
