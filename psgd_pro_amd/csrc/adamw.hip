// One AdamW step over many tensors, its states in fp32 or in 8 bits, and the norm of all gradients.
#include "adamw.h"
#include "philox.h"

namespace psgdk {

namespace {

// The chunk's tensor: the last one with first[t] <= chunk.
__device__ __forceinline__ int tensor_of(const AdamArgs& a, int chunk) {
  int lo = 0, hi = a.count;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a.first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

// 8 elements from i on, n of which are there; wherever the tensor begins (whole vectors may straddle 16 bytes)
template <typename T>
__device__ __forceinline__ void ld8(const T* p, int n, float (&x)[8]) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(x, p, 32);
    } else {
      uint32_t w[4];
      __builtin_memcpy(w, p, 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = i < n ? to_f32<T>(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void st8(T* p, int n, const float (&x)[8]) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 4) {
      __builtin_memcpy(p, x, 32);
    } else {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = pack2_bf16(x[2 * i], x[2 * i + 1]);
      __builtin_memcpy(p, w, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = from_f32<T>(x[i]);
  }
}
__device__ __forceinline__ uint2 ld_codes(const uint8_t* p, int n) {
  uint2 w = make_uint2(0, 0);
  if (n >= 8) {
    __builtin_memcpy(&w, p, 8);
  } else {
    for (int i = 0; i < n; ++i) {
      if (i < 4) w.x |= (uint32_t)p[i] << 8 * i;
      else w.y |= (uint32_t)p[i] << 8 * (i - 4);
    }
  }
  return w;
}
__device__ __forceinline__ void st_codes(uint8_t* p, int n, uint2 w) {
  if (n >= 8) {
    __builtin_memcpy(p, &w, 8);
  } else {
    for (int i = 0; i < n; ++i) p[i] = (uint8_t)((i < 4 ? w.x >> 8 * i : w.y >> 8 * (i - 4)) & 255);
  }
}

// e4m3 codes times a power of two: exact
__device__ __forceinline__ void unpack8(uint2 w, float scale, float (&x)[8]) {
  typedef float f32x2_t __attribute__((ext_vector_type(2)));
  const f32x2_t a = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w.x, true);
  const f32x2_t c = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, false), d = __builtin_amdgcn_cvt_pk_f32_fp8(w.y, true);
  x[0] = a[0] * scale;
  x[1] = a[1] * scale;
  x[2] = b[0] * scale;
  x[3] = b[1] * scale;
  x[4] = c[0] * scale;
  x[5] = c[1] * scale;
  x[6] = d[0] * scale;
  x[7] = d[1] * scale;
}
// a scale byte's value: 2^(byte - 127), 255 NaN
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte == 255 ? 0x7fc00000u : byte << 23); }

// largest over the 32 lanes of a block's elements
__device__ __forceinline__ float max32(float m) {
  m = fmaxf(m, dpp<0xB1>(m));
  m = fmaxf(m, dpp<0x4E>(m));
  m = fmaxf(m, dpp<0x141>(m));
  m = fmaxf(m, dpp<0x140>(m));
  return fmaxf(m, __shfl_xor(m, 16, 64));
}
// The scale's exponent field for a largest magnitude of bits `top`: with it that lies in (224, 448], e4m3's top. The largest
// field is 247, so that 2^(127 - field) is a normal number too. Infinite or NaN: 255.
__device__ __forceinline__ uint32_t scale_field(float top) {
  const uint32_t u = __float_as_uint(top);
  if (u >= 0x7f800000u) return 255;
  return u ? max((int)((u + 0x1fffffu) >> 23) - 8, 1) : 0;
}
// Codes of 8 values, rounded up or down by chance: as a float scaled so that e4m3's exponents and subnormals are fp32's, a
// magnitude's code is its bits above the 20th; a 16-bit number times 16 is added to the bits below. The expected value is the
// value itself, so that changes far below half a code's step are not lost over many steps (an average over 1000 gradients moves
// by a thousandth a step, a code's step is up to an eighth). ROOT: positive values, none becomes 0 (an update divides by them).
template <bool ROOT>
__device__ __forceinline__ uint2 pack8(const float (&x)[8], uint32_t field, const uint32_t (&rnd)[4]) {
  const float up = __uint_as_float((254 - field) << 23);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t number = i & 1 ? rnd[i >> 1] >> 16 : rnd[i >> 1] & 0xffffu;
    const uint32_t u = __float_as_uint(x[i]);
    const float y = __uint_as_float(u & 0x7fffffffu) * up * 0x1p-120f;
    c[i] = (__float_as_uint(y) + number * 16) >> 20;
    if constexpr (ROOT) c[i] = max(c[i], u ? 1u : 0u);
    else c[i] |= x[i] < 0.f ? 128u : 0u;
    c[i] = field == 255 ? 0x7fu : c[i];
  }
  return make_uint2(c[0] | c[1] << 8 | c[2] << 16 | c[3] << 24, c[4] | c[5] << 8 | c[6] << 16 | c[7] << 24);
}

// m = b1 m + (1 - b1) g, v = b2 v + (1 - b2) g^2, each product and sum rounded, so that the same inputs give the same codes
// wherever they are computed; then p. ROOTS: v holds roots before. WIDE: where a square is out of range, its root is made of a
// 2^-64th of root and gradient (infinite and NaN ones stay so).
template <bool ROOTS, bool WIDE>
__device__ __forceinline__ void adam8(const AdamArgs& a, float coef, bool scaled, float (&p)[8], const float (&g0)[8], float (&m)[8],
                                      float (&v)[8], float (&root)[8]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float g = scaled ? g0[i] * coef : g0[i], r = v[i];
    m[i] = m[i] * a.b1 + g * a.c1;
    v[i] = (ROOTS ? r * r : r) * a.b2 + g * g * a.c2;
    root[i] = sqrtf(v[i]);
    if constexpr (WIDE) {
      const float s = r * 0x1p-64f, h = g * 0x1p-64f;
      if (!(v[i] < INFINITY)) root[i] = sqrtf(s * s * a.b2 + h * h * a.c2) * 0x1p64f;
    }
    p[i] = p[i] * a.keep - a.rate * m[i] * __builtin_amdgcn_rcpf(root[i] * a.root + a.eps);
  }
}

// 28 bytes an element with fp32 parameters and states, 10 with bf16 parameters and 8 bits: bound by memory. 386 M elements: fp32
// 2048 us, 5.3 TB/s; bf16 with 8 bits 735 us, 5.3 TB/s, some 65 vector instructions an element (a third of them Philox, which is
// why both states share a number). A thread has 8 elements that lie together, twice, 32 lanes a block of 256.
// WHOLE: the chunk is all there. With 8 bits, false where the block has a moment out of range: nothing is stored then, but
// where WIDE (that path apart, and from memory again, costs the other nothing).
template <typename T, int BITS, bool WHOLE, bool WIDE>
__device__ __forceinline__ bool adamw_elements(const AdamArgs& a, int t, T* p, const T* g, float coef, long long n, long long i) {
  const int left = WHOLE ? 8 : (int)min(max(n - i, 0ll), 8ll);
  float x[8], y[8], m[8], v[8], root[8];
  ld8(p + i, left, x);
  ld8(g + i, left, y);
  if constexpr (BITS == 32) {
    ld8(static_cast<const float*>(a.m[t]) + i, left, m);
    ld8(static_cast<const float*>(a.v[t]) + i, left, v);
    adam8<false, false>(a, coef, a.coef != nullptr, x, y, m, v, root);
    st8(static_cast<float*>(a.m[t]) + i, left, m);
    st8(static_cast<float*>(a.v[t]) + i, left, v);
  } else {
    const long long block = i / kAdamBlock;
    uint8_t* const mc = static_cast<uint8_t*>(a.m[t]) + i;
    uint8_t* const vc = static_cast<uint8_t*>(a.v[t]) + i;
    unpack8(ld_codes(mc, left), left ? scale_of(a.ms[t][block]) : 0.f, m);
    unpack8(ld_codes(vc, left), left ? scale_of(a.vs[t][block]) : 0.f, v);
    adam8<true, WIDE>(a, coef, a.coef != nullptr, x, y, m, v, root);
    float mt = 0.f, vt = 0.f;
    bool bad = false;  // (a largest of NaN and a number is the number)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float am = e < left ? fabsf(m[e]) : 0.f, av = e < left ? root[e] : 0.f;
      bad = bad || !(am < INFINITY) || !(av < INFINITY);
      mt = fmaxf(mt, am);
      vt = fmaxf(vt, av);
    }
    const uint32_t mf = scale_field(max32(bad ? INFINITY : mt)), vf = scale_field(max32(bad ? INFINITY : vt));
    if (!WIDE && mf == 255) return false;
    const long long w = (a.at[t] + i) / 8;
    uint32_t rnd[4] = {(uint32_t)w, (uint32_t)(w >> 32), a.step, (uint32_t)a.index[t]};
    philox4x32_10(rnd, a.k0, a.k1);
    st_codes(mc, left, pack8<false>(m, mf, rnd));
    st_codes(vc, left, pack8<true>(root, vf, rnd));
    if (left && threadIdx.x % 32 == 0) {
      a.ms[t][block] = (uint8_t)mf;
      a.vs[t][block] = (uint8_t)vf;
    }
  }
  st8(p + i, left, x);
  return true;
}
template <typename T, int BITS, bool WHOLE>
__device__ __forceinline__ void adamw_chunk(const AdamArgs& a, int t, long long n, long long i0) {
  T* const p = static_cast<T*>(a.p[t]);
  const T* const g = static_cast<const T*>(a.g[t]);
  const float coef = a.coef ? *a.coef : 1.f;
  i0 += threadIdx.x * 8;
  bool done[kAdamChunk / 2048];
#pragma unroll
  for (int r = 0; r < kAdamChunk / 2048; ++r) done[r] = adamw_elements<T, BITS, WHOLE, false>(a, t, p, g, coef, n, i0 + r * 2048);
  if constexpr (BITS == 8) {
#pragma unroll
    for (int r = 0; r < kAdamChunk / 2048; ++r)
      if (!done[r]) adamw_elements<T, BITS, false, true>(a, t, p, g, coef, n, i0 + r * 2048);
  }
}
template <typename T, int BITS>
__global__ void __launch_bounds__(256) adamw_kernel(const AdamArgs a) {
  const int t = tensor_of(a, blockIdx.x);
  const long long n = a.n[t], i0 = (long long)(blockIdx.x - a.first[t]) * kAdamChunk;
  if (i0 + kAdamChunk <= n) adamw_chunk<T, BITS, true>(a, t, n, i0);
  else adamw_chunk<T, BITS, false>(a, t, n, i0);
}

template <typename T>
__global__ void __launch_bounds__(256) adamw_norm_kernel(const AdamArgs a, int chunks) {
  __shared__ double red[4];
  double sum = 0.0;  // (squares in fp64: no overflow, and millions of them)
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const int t = tensor_of(a, chunk);
    const long long n = a.n[t], i0 = (long long)(chunk - a.first[t]) * kAdamChunk;
#pragma unroll
    for (int r = 0; r < kAdamChunk / 2048; ++r) {
      const long long i = i0 + r * 2048 + threadIdx.x * 8;
      float y[8];
      ld8(static_cast<const T*>(a.g[t]) + i, (int)min(max(n - i, 0ll), 8ll), y);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += (double)y[e] * (double)y[e];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) a.part[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
}

__global__ void __launch_bounds__(1024) adamw_coef_kernel(const double* part, long long n, double max_norm, float* norm, float* coef) {
  __shared__ double red[16];
  double sum = 0.0;
#pragma unroll 4
  for (long long i = threadIdx.x; i < n; i += 1024) sum += part[i];
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x) return;
  sum = 0.0;
  for (int i = 0; i < 16; ++i) sum += red[i];
  const double r = sqrt(sum);
  if (norm) *norm = (float)r;
  if (coef) *coef = r <= max_norm ? 1.f : (float)(max_norm / r);  // (a NaN norm: NaN, and so the step)
}

}  // namespace

hipError_t adamw_launch(const AdamArgs& a, int dt, int bits, hipStream_t st) {
  const dim3 grid(a.first[a.count]), block(256);
  if (dt == 0) {
    if (bits == 32) hipLaunchKernelGGL((adamw_kernel<float, 32>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((adamw_kernel<float, 8>), grid, block, 0, st, a);
  } else {
    if (bits == 32) hipLaunchKernelGGL((adamw_kernel<bf16_t, 32>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((adamw_kernel<bf16_t, 8>), grid, block, 0, st, a);
  }
  return hipGetLastError();
}
hipError_t adamw_norm_launch(const AdamArgs& a, int dt, int& parts, hipStream_t st) {
  const int chunks = a.first[a.count];
  parts = chunks < kAdamParts ? chunks : kAdamParts;
  if (dt == 0) hipLaunchKernelGGL(adamw_norm_kernel<float>, dim3(parts), dim3(256), 0, st, a, chunks);
  else hipLaunchKernelGGL(adamw_norm_kernel<bf16_t>, dim3(parts), dim3(256), 0, st, a, chunks);
  return hipGetLastError();
}
hipError_t adamw_coef_launch(const double* part, long long n, double max_norm, float* norm, float* coef, hipStream_t st) {
  hipLaunchKernelGGL(adamw_coef_kernel, dim3(1), dim3(1024), 0, st, part, n, max_norm, norm, coef);
  return hipGetLastError();
}

}  // namespace psgdk
