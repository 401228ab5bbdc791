// Dropout, and the residual sum between two blocks of a transformer with its norms, gate, scale and dropout. Both are
// bound by memory: every tensor passes once, a row stays in registers between its statistics and its use, sums are fp32.
#include <algorithm>

#include "block.h"
#include "philox.h"

namespace psgdk {

namespace {

constexpr int VE = 8;  // elements a thread holds together: one 16-byte bf16 access, one Philox block of dropout

// VE consecutive elements as floats. The pointers are only element-aligned (rows of odd length): the copies become
// 16-byte accesses, which this GPU serves at any alignment.
__device__ __forceinline__ void ld8(const bf16_t* p, float (&v)[VE]) {
  bf16_t h[VE];
  __builtin_memcpy(h, p, sizeof h);
#pragma unroll
  for (int e = 0; e < VE; ++e) v[e] = bf16_to_f32(h[e]);
}
__device__ __forceinline__ void ld8(const float* p, float (&v)[VE]) { __builtin_memcpy(v, p, sizeof v); }
__device__ __forceinline__ void st8(bf16_t* p, const float (&v)[VE]) {
  bf16_t h[VE];
#pragma unroll
  for (int e = 0; e < VE; ++e) h[e] = f32_to_bf16(v[e]);
  __builtin_memcpy(p, h, sizeof h);
}
__device__ __forceinline__ void st8(float* p, const float (&v)[VE]) { __builtin_memcpy(p, v, sizeof v); }

// Elements c .. c + 7 of a row of d (zeros past its end).
template <typename T>
__device__ __forceinline__ void ld_row(const T* row, int c, int d, float (&v)[VE]) {
  if (c + VE <= d) {
    ld8(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = c + e < d ? to_f32<T>(row[c + e]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void st_row(T* row, int c, int d, const float (&v)[VE]) {
  if (c + VE <= d) {
    st8(row + c, v);
  } else {
#pragma unroll
    for (int e = 0; e < VE; ++e)
      if (c + e < d) row[c + e] = from_f32<T>(v[e]);
  }
}
// One thread's 8 elements c .. c + 7 of rows of d >= 8 elements. Where the row ends inside them the load starts 8
// elements before its end and the values move down (zeros behind the end): every lane loads one whole vector. RAGGED:
// d is no multiple of 8 (else there is nothing to move and to mask).
template <bool RAGGED>
struct Span {
  int c, d, at, move;
  bool in;  // the thread has elements of the row
  __device__ __forceinline__ Span(int c_, int d_) : c(c_), d(d_) {
    in = c < d;
    at = RAGGED ? min(c, d - VE) : c;
    move = c - at;
  }
  // The load in two parts, so that the bits of the next row can be on their way while this one's are used.
  template <typename T>
  struct Raw {
    uint32_t w[VE * sizeof(T) / 4];
  };
  template <typename T>
  __device__ __forceinline__ void fetch(const T* row, Raw<T>& r) const {
    if (in) {
      __builtin_memcpy(r.w, row + at, sizeof r.w);
    } else {
#pragma unroll
      for (uint32_t& x : r.w) x = 0;
    }
  }
  template <typename T>
  __device__ __forceinline__ void use(const Raw<T>& r, float (&v)[VE]) const {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      if constexpr (sizeof(T) == 2) v[e] = __uint_as_float(e & 1 ? r.w[e / 2] & 0xffff0000u : r.w[e / 2] << 16);
      else v[e] = __uint_as_float(r.w[e]);
    }
    if (RAGGED && __any(move)) {  // (only in the wave that holds the row's end)
#pragma unroll
      for (int s = 4; s > 0; s >>= 1) {
        const bool m = move & s;
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = m ? (e + s < VE ? v[e + s] : 0.f) : v[e];
      }
    }
  }
  __device__ __forceinline__ void zero(float (&v)[VE]) const {
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = 0.f;
  }
  template <typename T>
  __device__ __forceinline__ void load(const T* row, float (&v)[VE]) const {
    Raw<T> r;
    fetch(row, r);
    use(r, v);
  }
  __device__ __forceinline__ void load(const Vec& w, long long off, float none, float (&v)[VE]) const {
    if (!w.p) {
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = none;
    } else if (w.dt == 1) {
      load(reinterpret_cast<const bf16_t*>(w.p) + off, v);
    } else {
      load(reinterpret_cast<const float*>(w.p) + off, v);
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(T* row, const float (&v)[VE]) const {
    if (!in) return;
    if constexpr (RAGGED) st_row(row, c, d, v);
    else st8(row + c, v);
  }
  // whether element e is the row's (in a centred sum, the zeros behind its end are not)
  __device__ __forceinline__ bool has(int e) const { return RAGGED ? c + e < d : in; }
};

// Dropout's factors of elements c .. c + 7 (c a multiple of 8) of a row.
__device__ __forceinline__ void drop8(const Drop& dr, long long row, int c, int d, float (&m)[VE]) {
  const unsigned long long blk = (unsigned long long)row * (unsigned)((d + VE - 1) / VE) + (unsigned)(c / VE);
  uint32_t w[4] = {(uint32_t)blk, (uint32_t)(blk >> 32), dr.s0, dr.s1};
  philox4x32_10(w, dr.k0, dr.k1);
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    const uint32_t u = (e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xffffu;
    m[e] = u >= dr.thr ? dr.scale : 0.f;
  }
}

// A dropped element is 0 whatever it holds (an infinity too).
__device__ __forceinline__ float dropped(float v, float m) { return m == 0.f ? 0.f : v * m; }

}  // namespace

// ---------------------------------------------------------------------------------------------------------------
// y = dropout(x): one Philox block of 128 bits serves 8 elements, 16 bits each (drop probabilities in steps of 2^-16), and
// no mask is stored: the backward pass is the same kernel on the gradient. Bound by memory (2 bytes read and 2 written an
// element against about 12 instructions): 16384 x 4096 bf16 forward and backward 104-107 us, 5.0-5.2 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const DropArgs a) {
  const long long per = (a.d + VE - 1) / VE, total = a.rows * per;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
    const long long row = i / per;
    const int c = (int)(i - row * per) * VE;
    float v[VE], m[VE];
    ld_row(reinterpret_cast<const T*>(a.x) + row * a.ldx, c, a.d, v);
    drop8(a.drop, row, c, a.d, m);
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] = dropped(v[e], m[e]);
    st_row(reinterpret_cast<T*>(a.y) + row * a.ldy, c, a.d, v);
  }
}

hipError_t dropout_launch(const DropArgs& a, hipStream_t st) {
  const long long want = (a.rows * ((a.d + VE - 1) / VE) + 255) / 256;
  const int blocks = (int)(want > 4096 ? 4096 : want);
  if (a.dt == 1) hipLaunchKernelGGL(dropout_kernel<bf16_t>, dim3(blocks), dim3(256), 0, st, a);
  else hipLaunchKernelGGL(dropout_kernel<float>, dim3(blocks), dim3(256), 0, st, a);
  return hipGetLastError();
}

// ---------------------------------------------------------------------------------------------------------------
// y = x + scale gate dropout(Npost(f)), h = Npre(y). TPR threads hold a row, 8 elements each; a workgroup of at least
// 256 threads holds 256 / TPR rows. The waves' sums meet in LDS where a row has more than one. The
// variance of a layer norm is the mean of the squared centred values, summed from the registers (no difference of large
// sums). h is made from y before y's rounding. Bound by memory, x and f read once, y and h written once: 16384 rows of 4096
// bf16 with two rms norms 102 us, 5.3 TB/s (as fast as a copy); 33280 rows of 512 fp32 with a layer norm, a gate and dropout
// 48 us, 5.7 TB/s.
namespace {

constexpr int res_threads(int tpr) { return tpr < 256 ? 256 : tpr; }

// Sum over a wave, in all lanes: the 16 lanes of each row by DPP moves, then the four rows' sums read as scalars (six
// shuffles through LDS take several times as long, and a row's time is a chain of these sums).
__device__ __forceinline__ float lanes_sum(float v) {
  v = row16_sum(v);
  const int i = __float_as_int(v);
  return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
         (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}

// Sums over the TPR threads of a row, every thread of the workgroup taking part. red holds one value for each wave; its
// next use has to come after a barrier.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
  v = lanes_sum(v);
  if constexpr (TPR > 64) {
    const int w = threadIdx.x >> 6, w0 = w / (TPR / 64) * (TPR / 64);
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) v += red[w0 + i];
  }
  return v;
}
template <int TPR>
__device__ __forceinline__ float2 row_sum2(float2 v, float2* red) {
  v.x = lanes_sum(v.x);
  v.y = lanes_sum(v.y);
  if constexpr (TPR > 64) {
    const int w = threadIdx.x >> 6, w0 = w / (TPR / 64) * (TPR / 64);
    if ((threadIdx.x & 63) == 0) red[w] = v;
    __syncthreads();
    v = make_float2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) {
      v.x += red[w0 + i].x;
      v.y += red[w0 + i].y;
    }
  }
  return v;
}

// mean and 1 / std of a row held in u; u is centred in place for a layer norm (red: 2 x 16 floats)
template <int TPR, bool RAGGED>
__device__ __forceinline__ float2 row_stats(float (&u)[VE], const Span<RAGGED>& sp, int kind, float eps, float* red) {
  const float inv_d = 1.f / (float)sp.d;
  float mean = 0.f, s = 0.f;
  if (kind == NORM_LAYER) {
#pragma unroll
    for (int e = 0; e < VE; ++e) s += u[e];
    mean = row_sum<TPR>(s, red) * inv_d;
    s = 0.f;
#pragma unroll
    for (int e = 0; e < VE; ++e) u[e] = sp.has(e) ? u[e] - mean : 0.f;
  }
#pragma unroll
  for (int e = 0; e < VE; ++e) s += u[e] * u[e];
  return make_float2(mean, 1.f / sqrtf(row_sum<TPR>(s, red + 16) * inv_d + eps));
}

template <typename T, int TPR, bool RAGGED>
__global__ void __launch_bounds__(res_threads(TPR)) residual_norm_kernel(const ResArgs a) {
  __shared__ float red[2][32];
  const long long want =
      (long long)blockIdx.x * (res_threads(TPR) / TPR) + __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  const bool live = want < a.rows;
  const long long row = live ? want : a.rows - 1;  // a row behind the last one takes part in the barriers only
  const int t = threadIdx.x % TPR;
  const Span<RAGGED> sp(t * VE, a.d);
  float4 st = make_float4(0.f, 0.f, 0.f, 0.f);
  float x[VE];
  sp.load(reinterpret_cast<const T*>(a.x) + row * a.ldx, x);
  if (a.f) {
    float u[VE], g[VE];
    sp.load(reinterpret_cast<const T*>(a.f) + row * a.ldf, u);
    sp.load(a.gate, row / a.gate_every * a.ldg, 1.f, g);
    if (a.post != NORM_NONE) {
      float w[VE], b[VE];
      sp.load(a.post_w, 0, 1.f, w);
      sp.load(a.post_b, 0, 0.f, b);
      const float2 s = row_stats<TPR, RAGGED>(u, sp, a.post, a.eps, red[0]);
      st.z = s.x;
      st.w = s.y;
#pragma unroll
      for (int e = 0; e < VE; ++e) u[e] = u[e] * s.y * w[e] + b[e];
    }
    if (a.drop.thr) {
      float m[VE];
      drop8(a.drop, row, sp.c, a.d, m);
#pragma unroll
      for (int e = 0; e < VE; ++e) u[e] = dropped(u[e], m[e]);
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) x[e] += sp.has(e) ? a.scale * g[e] * u[e] : 0.f;
  }
  if (a.y && live) sp.store(reinterpret_cast<T*>(a.y) + row * a.ldy, x);
  if (a.pre != NORM_NONE) {
    float w[VE], b[VE];
    sp.load(a.pre_w, 0, 1.f, w);
    sp.load(a.pre_b, 0, 0.f, b);
    const float2 s = row_stats<TPR, RAGGED>(x, sp, a.pre, a.eps, red[1]);
    st.x = s.x;
    st.y = s.y;
#pragma unroll
    for (int e = 0; e < VE; ++e) w[e] = x[e] * s.y * w[e] + b[e];
    if (live) sp.store(reinterpret_cast<T*>(a.h) + row * a.ldh, w);
  }
  if (a.stats && t == 0 && live) a.stats[row] = st;
}

// What a thread has of a row in the kernels for the other rows (res_wide, res_backward_wide): the bits of 8 elements of every
// tensor, all loaded before any is looked at. A load that starts inside the last 8 elements of a row starts at the first
// of them, and the values move down (zeros behind the end).
template <typename T>
struct Wide {
  const ResArgs& a;
  long long row;
  float4 st, mean;
  int c, at;
  uint32_t x[VE * sizeof(T) / 4], f[VE * sizeof(T) / 4], dy[VE * sizeof(T) / 4], dh[VE * sizeof(T) / 4];
  uint32_t g[VE], pw[VE], pb[VE], qw[VE], qb[VE];
  __device__ __forceinline__ Wide(const ResArgs& args) : a(args) {}
  __device__ __forceinline__ void place(int col) {
    c = col;
    at = a.d < VE ? 0 : min(c, a.d - VE);
  }
  template <typename U, size_t N>
  __device__ __forceinline__ void bits(const U* p, uint32_t (&w)[N]) const {
    if (a.d >= VE) {
      __builtin_memcpy(w, p + at, VE * sizeof(U));
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const uint32_t b = e >= a.d ? 0 : sizeof(U) == 4 ? reinterpret_cast<const uint32_t*>(p)[e] : (uint32_t)p[e];
        if constexpr (sizeof(U) == 4) w[e] = b;
        else w[e / 2] = e & 1 ? w[e / 2] | b << 16 : b;
      }
    }
  }
  __device__ __forceinline__ void bits(const Vec& v, long long off, uint32_t (&w)[VE]) const {
    if (!v.p) return;
    if (v.dt == 1) bits(reinterpret_cast<const bf16_t*>(v.p) + off, w);
    else bits(reinterpret_cast<const float*>(v.p) + off, w);
  }
  // the row's own tensors (whichever the call has), and the vectors that all rows share
  __device__ __forceinline__ void fetch_row() {
    if (a.x) bits(reinterpret_cast<const T*>(a.x) + row * a.ldx, x);
    if (a.f) bits(reinterpret_cast<const T*>(a.f) + row * a.ldf, f);
    if (a.dy) bits(reinterpret_cast<const T*>(a.dy) + row * a.lddy, dy);
    if (a.dh) bits(reinterpret_cast<const T*>(a.dh) + row * a.lddh, dh);
    bits(a.gate, row / a.gate_every * a.ldg, g);
  }
  __device__ __forceinline__ void fetch_shared(bool bias) {
    bits(a.pre_w, 0, pw);
    if (bias) bits(a.pre_b, 0, pb);
    bits(a.post_w, 0, qw);
    bits(a.post_b, 0, qb);
  }
  __device__ __forceinline__ void move_down(float (&v)[VE]) const {
    if (a.d < VE || !__any(c != at)) return;  // (only in the wave that holds the row's end)
#pragma unroll
    for (int s = 4; s > 0; s >>= 1) {
      const bool m = (c - at) & s;
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = m ? (e + s < VE ? v[e + s] : 0.f) : v[e];
    }
  }
  template <typename U, size_t N>
  __device__ __forceinline__ void values(const uint32_t (&w)[N], float (&v)[VE]) const {
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      if constexpr (sizeof(U) == 2) v[e] = __uint_as_float(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
      else v[e] = __uint_as_float(w[e]);
    }
    move_down(v);
  }
  __device__ __forceinline__ void values(const Vec& q, const uint32_t (&w)[VE], float none, float (&v)[VE]) const {
    if (!q.p) {
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = none;
    } else if (q.dt == 1) {
      values<bf16_t>(w, v);
    } else {
      values<float>(w, v);
    }
  }
  // the branch: f's normalised values, b = dropout(Npost(f)) and the elements kept
  __device__ __forceinline__ unsigned branch(float (&fh)[VE], float (&b)[VE]) const {
    unsigned kept = 255;
    values<T>(f, fh);
    if (a.post != NORM_NONE) {
      float w[VE];
      values(a.post_w, qw, 1.f, w);
      values(a.post_b, qb, 0.f, b);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        fh[e] = (fh[e] - st.z) * st.w;
        b[e] += fh[e] * w[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) b[e] = fh[e];
    }
    if (a.drop.thr) {
      float k[VE];
      drop8(a.drop, row, c, a.d, k);
      kept = 0;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        b[e] = dropped(b[e], k[e]);
        kept |= k[e] != 0.f ? 1u << e : 0u;
      }
    }
    return kept;
  }
  __device__ __forceinline__ void y_of(float (&y)[VE]) const {
    values<T>(x, y);
    if (!a.f) return;
    float fh[VE], b[VE], gate[VE];
    branch(fh, b);
    values(a.gate, g, 1.f, gate);
#pragma unroll
    for (int e = 0; e < VE; ++e) y[e] += a.scale * gate[e] * b[e];
  }
  // y's normalised values, dh and c = dh w
  __device__ __forceinline__ void pre(float (&hat)[VE], float (&dhv)[VE], float (&cw)[VE]) const {
    y_of(hat);
    values<T>(dh, dhv);
    values(a.pre_w, pw, 1.f, cw);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      hat[e] = (hat[e] - st.x) * st.y;
      cw[e] *= dhv[e];
    }
  }
  __device__ __forceinline__ void dyt(float (&v)[VE]) const {
    if (a.dy) values<T>(dy, v);
    else
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] = 0.f;
    if (!a.dh) return;
    float hat[VE], dhv[VE], cw[VE];
    pre(hat, dhv, cw);
#pragma unroll
    for (int e = 0; e < VE; ++e) v[e] += (cw[e] - mean.x - hat[e] * mean.y) * st.y;
  }
  // v = dyt in; out: f's normalised values, du (v), du w (dw) and the gate's gradient
  __device__ __forceinline__ void post(float (&v)[VE], float (&fh)[VE], float (&dw)[VE], float (&dg)[VE]) const {
    float gate[VE];
    const unsigned kept = branch(fh, dg);
    values(a.gate, g, 1.f, gate);
    if (a.post != NORM_NONE) {
      values(a.post_w, qw, 1.f, dw);
    } else {
#pragma unroll
      for (int e = 0; e < VE; ++e) dw[e] = 1.f;
    }
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      float du = a.scale * v[e];
      dg[e] *= du;
      du *= gate[e];
      if (a.drop.thr) du = kept >> e & 1 ? du * a.drop.scale : 0.f;
      v[e] = du;
      dw[e] *= du;
    }
  }
};
// The values made of the bits so far are not kept for later, where they would not fit the registers: an empty asm statement
// makes the bits new ones to the compiler.
template <typename... W>
__device__ __forceinline__ void forget(W&... w) {
  auto one = [](auto& q) __attribute__((always_inline)) {
#pragma unroll
    for (uint32_t& b : q) asm volatile("" : "+v"(b));
  };
  (one(w), ...);
}
// ONE: the rows fit one vector a thread, whose bits stay for all passes. Else every pass reads the row again, from the
// caches (branch: only f is looked at).
template <bool ONE, typename T, typename F>
__device__ __forceinline__ void wide_pass(Wide<T>& t, bool bias, bool branch, F fn) {
  if constexpr (ONE) {
    forget(t.x, t.f, t.dy, t.dh, t.g);
    t.fetch_shared(bias);
    if (t.c < t.a.d) fn();
  } else {
    for (int c = threadIdx.x * VE; c < t.a.d; c += blockDim.x * VE) {
      t.place(c);
      if (branch) {
        t.bits(reinterpret_cast<const T*>(t.a.f) + t.row * t.a.ldf, t.f);
      } else {
        t.fetch_row();
        t.fetch_shared(bias);
      }
      fn();
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) residual_norm_wide_kernel(const ResArgs a) {
  __shared__ float red[16];
  Wide<T> t(a);
  t.row = blockIdx.x;
  t.st = make_float4(0.f, 0.f, 0.f, 0.f);
  t.place(threadIdx.x * VE);
  const float inv_d = 1.f / (float)a.d;
  auto stats = [&](int kind, bool branch, auto at) {
    float mean = 0.f, s = 0.f;
    if (kind == NORM_LAYER) {
      wide_pass<false>(t, false, branch, [&] {
        float v[VE];
        at(v);
#pragma unroll
        for (int e = 0; e < VE; ++e) s += t.c + e < a.d ? v[e] : 0.f;
      });
      mean = block_sum(s, red) * inv_d;
      s = 0.f;
    }
    wide_pass<false>(t, false, branch, [&] {
      float v[VE];
      at(v);
#pragma unroll
      for (int e = 0; e < VE; ++e) s += t.c + e < a.d ? (v[e] - mean) * (v[e] - mean) : 0.f;
    });
    return make_float2(mean, 1.f / sqrtf(block_sum(s, red) * inv_d + a.eps));
  };
  if (a.f && a.post != NORM_NONE) {
    const float2 s = stats(a.post, true, [&](float (&v)[VE]) { t.template values<T>(t.f, v); });
    t.st.z = s.x;
    t.st.w = s.y;
  }
  if (a.pre != NORM_NONE) {
    const float2 s = stats(a.pre, false, [&](float (&v)[VE]) { t.y_of(v); });
    t.st.x = s.x;
    t.st.y = s.y;
  }
  wide_pass<false>(t, true, false, [&] {
    float y[VE];
    t.y_of(y);
    if (a.y) st_row(reinterpret_cast<T*>(a.y) + t.row * a.ldy, t.c, a.d, y);
    if (a.pre != NORM_NONE) {
      float w[VE], b[VE];
      t.values(a.pre_w, t.pw, 1.f, w);
      t.values(a.pre_b, t.pb, 0.f, b);
#pragma unroll
      for (int e = 0; e < VE; ++e) w[e] = (y[e] - t.st.x) * t.st.y * w[e] + b[e];
      st_row(reinterpret_cast<T*>(a.h) + t.row * a.ldh, t.c, a.d, w);
    }
  });
  if (a.stats && threadIdx.x == 0) a.stats[t.row] = t.st;
}

}  // namespace

template <typename T, int TPR>
static void residual_norm_sized(const ResArgs& a, hipStream_t st) {
  constexpr int RW = res_threads(TPR) / TPR;
  const dim3 grid((unsigned)((a.rows + RW - 1) / RW)), block(res_threads(TPR));
  if (a.d % VE) hipLaunchKernelGGL((residual_norm_kernel<T, TPR, true>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((residual_norm_kernel<T, TPR, false>), grid, block, 0, st, a);
}
template <typename T>
static hipError_t residual_norm_t(const ResArgs& a, hipStream_t st) {
  if (res_wide(a.d)) hipLaunchKernelGGL(residual_norm_wide_kernel<T>, dim3((unsigned)a.rows), dim3(1024), 0, st, a);
  else if (a.d <= 512) residual_norm_sized<T, 64>(a, st);
  else if (a.d <= 1024) residual_norm_sized<T, 128>(a, st);
  else if (a.d <= 2048) residual_norm_sized<T, 256>(a, st);
  else if (a.d <= 4096) residual_norm_sized<T, 512>(a, st);
  else residual_norm_sized<T, 1024>(a, st);
  return hipGetLastError();
}
hipError_t residual_norm_launch(const ResArgs& a, hipStream_t st) {
  return a.dt == 1 ? residual_norm_t<bf16_t>(a, st) : residual_norm_t<float>(a, st);
}

// ---------------------------------------------------------------------------------------------------------------
// Backward. y is made again from x and f, as many bytes as the stored y and f and without y's rounding. With
// hat = (y - mean) / std, c = dh w:
//   dyt = dy + (c - [layer] mean(c) - hat mean(c hat)) / std;  dx = dyt
//   dgate = sum over its rows of scale dyt b;  du = scale gate dropout'(dyt);  df from du and f as dyt from dh and y
//   weights: column sums of dh hat and du fhat, biases: of dh and du
// A workgroup takes `chunk` consecutive rows and keeps its column sums in registers; they go to one row of `part` each
// and a second kernel adds those in a fixed order. A gate whose rows all lie in one workgroup has one such row.
// Bound by memory where rows are long enough (16384 rows of 4096 bf16, two rms norms: 180 us, 4.5 TB/s; 33280 rows of 512
// fp32: 86 us, 4.7 TB/s), by the chain of a row's sums on short ragged ones (8481 rows of 770 bf16, everything on: 51 us,
// 1.5 TB/s): a row's two means are each a wave's sum, a barrier and the waves' sums. The next row's loads are under way
// meanwhile (without them, and with one workgroup a CU: 410 us in place of 180).
namespace {

// Stores a workgroup's column sum as a row of the partial sums and starts it again from zero.
template <int TPR, bool RAGGED>
__device__ __forceinline__ void put_sum(float (&s)[VE], float* dst, const Span<RAGGED>& sp, float* lds) {
  if constexpr (TPR < 256) {  // the sums of the workgroup's rows meet in LDS, in order
    const int k = threadIdx.x / TPR, t = threadIdx.x % TPR;
#pragma unroll
    for (int e = 0; e < VE; ++e) lds[(k * VE + e) * TPR + t] = s[e];
    __syncthreads();
    if (k == 0) {
#pragma unroll
      for (int q = 1; q < 256 / TPR; ++q)
#pragma unroll
        for (int e = 0; e < VE; ++e) s[e] += lds[(q * VE + e) * TPR + t];
      sp.store(dst, s);
    }
    __syncthreads();
  } else {
    sp.store(dst, s);
  }
  sp.zero(s);
}

// HAS: what the call may have (kPost: a norm after the block, kGate, kBias: a layer norm's biases); what it cannot have
// holds no registers. SUMS: column sums in registers (1: of the norm before, 2: of the norm after, 4: of the gate).
// Waves a SIMD, by what their registers hold without scratch memory (256, 168 and 128 registers a lane for 2, 3 and 4 of
// them); the rows are cut for so many workgroups at once.
constexpr int res_waves(int tpr, int has, int esize) {
  if (tpr == 1024 || has == 0 || has == kBias || (tpr == 512 && has == kPost && esize == 2)) return 4;
  return tpr == 512 || has == 7 || (has == (kPost | kGate) && esize == 4) ? 2 : 3;
}
template <typename T, int TPR, int HAS, int SUMS, bool RAGGED>
__global__ void __launch_bounds__(res_threads(TPR), res_waves(TPR, HAS, sizeof(T)))
    residual_norm_backward_kernel(const ResArgs a) {
  constexpr int RW = res_threads(TPR) / TPR;  // rows the workgroup has in hand at once
  constexpr bool AHEAD = TPR < 1024;          // 1024 threads have no registers for the next row's bits
  __shared__ float2 red[2][16];
  __shared__ float lds[TPR < 256 ? VE * 256 : 1];
  // a row's waves are whole: its number is a scalar, and so are the addresses of its start
  const int t = threadIdx.x % TPR, w = __builtin_amdgcn_readfirstlane(threadIdx.x / TPR);
  using Sp = Span<RAGGED>;
  const Sp sp(t * VE, a.d);
  // rows r0 .. r1 - 1: `chunk` rows (whole gates), or a part of one gate's
  long long r0, r1;
  if (a.per_gate > 1) {
    const long long gate = (long long)blockIdx.x / a.per_gate;
    r0 = gate * a.gate_every + (long long)blockIdx.x % a.per_gate * a.chunk;
    r1 = min(r0 + a.chunk, (gate + 1) * a.gate_every);
  } else {
    r0 = (long long)blockIdx.x * a.chunk;
    r1 = min(r0 + a.chunk, a.rows);
  }
  float s_pw[VE] = {}, s_pb[VE] = {}, s_qw[VE] = {}, s_qb[VE] = {}, s_g[VE] = {};
  const float inv_d = 1.f / (float)a.d;
  const bool post = (HAS & kPost) && a.post != NORM_NONE, gated = (HAS & kGate) && a.gate.p;
  const bool pre_layer = (HAS & kBias) && a.pre == NORM_LAYER, post_layer = (HAS & kBias) && a.post == NORM_LAYER;

  // The weights of a row, read again for each row where a thread has no registers left to keep them (1024 threads have
  // 128 each): an empty asm statement hides from the compiler that the addresses stay the same.
  auto vec = [&](const Vec& v) {
    Vec q = v;
    if constexpr (TPR == 1024) asm volatile("" : "+s"(q.p));
    return q;
  };
  struct Bits {
    typename Sp::template Raw<T> x, f, dy, dh;
    float4 st;
  };
  auto fetch = [&](long long row, Bits& r) {
    r.st = a.stats ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.dy) sp.fetch(reinterpret_cast<const T*>(a.dy) + row * a.lddy, r.dy);
    if (a.f) sp.fetch(reinterpret_cast<const T*>(a.f) + row * a.ldf, r.f);
    if (a.dh) {
      sp.fetch(reinterpret_cast<const T*>(a.x) + row * a.ldx, r.x);
      sp.fetch(reinterpret_cast<const T*>(a.dh) + row * a.lddh, r.dh);
    }
  };
  auto one_row = [&](long long row, bool live, const Bits& r) {
    const float4 st = r.st;
    float v[VE], fh[VE], b[VE], g[VE], wt[VE];  // v: dyt, then du
    unsigned kept = 0;
    if (a.dy) sp.use(r.dy, v);
    else sp.zero(v);
    if (a.f) {  // the branch again: fh = f's normalised values, b = dropout(Npost(f))
      sp.use(r.f, fh);
      if (gated) sp.load(vec(a.gate), row / a.gate_every * a.ldg, 1.f, g);
      if (post) {
        sp.load(vec(a.post_w), 0, 1.f, wt);
        if (post_layer) sp.load(vec(a.post_b), 0, 0.f, b);
        else sp.zero(b);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          fh[e] = (fh[e] - st.z) * st.w;
          b[e] += fh[e] * wt[e];
        }
      } else {
#pragma unroll
        for (int e = 0; e < VE; ++e) b[e] = fh[e];
      }
      if (a.drop.thr) {
        float m[VE];
        drop8(a.drop, row, sp.c, a.d, m);
#pragma unroll
        for (int e = 0; e < VE; ++e) {
          b[e] = dropped(b[e], m[e]);
          kept |= m[e] != 0.f ? 1u << e : 0u;
        }
      }
    }
    if (a.dh) {
      float hat[VE], c[VE], pw[VE];
      float2 m = make_float2(0.f, 0.f);
      sp.use(r.x, hat);
      sp.use(r.dh, c);
      sp.load(vec(a.pre_w), 0, 1.f, pw);
      if (a.f) {
#pragma unroll
        for (int e = 0; e < VE; ++e) hat[e] += gated ? a.scale * g[e] * b[e] : a.scale * b[e];
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        hat[e] = (hat[e] - st.x) * st.y;
        if constexpr (SUMS & 1) {
          s_pw[e] += live ? c[e] * hat[e] : 0.f;
          if constexpr (HAS & kBias) s_pb[e] += live ? c[e] : 0.f;
        }
        c[e] *= pw[e];
        m.x += c[e];
        m.y += c[e] * hat[e];
      }
      m = row_sum2<TPR>(m, red[0]);
      m.x = pre_layer ? m.x * inv_d : 0.f;
      m.y *= inv_d;
#pragma unroll
      for (int e = 0; e < VE; ++e) v[e] += (c[e] - m.x - hat[e] * m.y) * st.y;
    }
    if (a.dx && live) sp.store(reinterpret_cast<T*>(a.dx) + row * a.lddx, v);
    if (a.f) {
      float2 m = make_float2(0.f, 0.f);
      float dg[VE];
      if constexpr (TPR == 1024) {
        if (gated) sp.load(vec(a.gate), row / a.gate_every * a.ldg, 1.f, g);
        if (post) sp.load(vec(a.post_w), 0, 1.f, wt);
      }
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        float du = sp.has(e) ? a.scale * v[e] : 0.f;
        if (gated) {
          dg[e] = du * b[e];
          du *= g[e];
          if constexpr ((SUMS & 4) && (HAS & kGate)) s_g[e] += live ? dg[e] : 0.f;
        }
        if (a.drop.thr) du = kept >> e & 1 ? du * a.drop.scale : 0.f;
        if (post) {
          if constexpr ((SUMS & 2) && (HAS & kPost)) {
            s_qw[e] += live ? du * fh[e] : 0.f;
            if constexpr (HAS & kBias) s_qb[e] += live ? du : 0.f;
          }
          du *= wt[e];
          m.x += du;
          m.y += du * fh[e];
        }
        v[e] = du;
      }
      if (gated && a.dgate && a.gate_every == 1 && live) {  // a gate for each row: no sum
        if (a.gate.dt == 1) sp.store(reinterpret_cast<bf16_t*>(a.dgate) + row * a.lddg, dg);
        else sp.store(reinterpret_cast<float*>(a.dgate) + row * a.lddg, dg);
      }
      if (post) {
        m = row_sum2<TPR>(m, red[1]);
        m.x = post_layer ? m.x * inv_d : 0.f;
        m.y *= inv_d;
#pragma unroll
        for (int e = 0; e < VE; ++e) v[e] = (v[e] - m.x - fh[e] * m.y) * st.w;
      }
      if (a.df && live) sp.store(reinterpret_cast<T*>(a.df) + row * a.lddf, v);
    }
    if constexpr (TPR > 64) __syncthreads();  // red is free again
  };

  const bool gate_sums = (SUMS & 4) && (HAS & kGate) && a.gpart;
  const bool whole_gates = gate_sums && a.per_gate == 1;
  const long long step = whole_gates ? a.gate_every : r1 - r0;
  for (long long b0 = r0; b0 < r1; b0 += step) {
    const long long b1 = min(b0 + step, r1);
    // a row behind the last one takes part in the barriers only
    auto row_of = [&](long long row) { return row + w < b1 ? row + w : b1 - 1; };
    Bits next;
    if constexpr (AHEAD) fetch(row_of(b0), next);
    for (long long row = b0; row < b1; row += RW) {
      Bits now;
      if constexpr (AHEAD) {
        now = next;
        if (row + RW < b1) fetch(row_of(row + RW), next);
      } else {
        fetch(row_of(row), now);
      }
      one_row(row_of(row), row + w < b1, now);
    }
    if (gate_sums)
      put_sum<TPR, RAGGED>(s_g, a.gpart + (whole_gates ? b0 / a.gate_every : (long long)blockIdx.x) * a.d, sp, lds);
  }
  auto put = [&](float (&s)[VE], int k) {
    if (a.slot[k] >= 0) put_sum<TPR, RAGGED>(s, a.part + ((long long)a.slot[k] * a.parts + blockIdx.x) * a.d, sp, lds);
  };
  if constexpr (SUMS & 1) {
    put(s_pw, kSumPreW);
    if constexpr (HAS & kBias) put(s_pb, kSumPreB);
  }
  if constexpr ((SUMS & 2) && (HAS & kPost)) {
    put(s_qw, kSumPostW);
    if constexpr (HAS & kBias) put(s_qb, kSumPostB);
  }
}

// The other lengths (Wide): the same gradients; the column sums are a second kernel's, from the rows' means kept by this
// one.
constexpr int res_wide_threads(int esize, bool one) { return one || esize == 2 ? 1024 : 512; }  // (registers)
template <typename T, bool ONE>
__global__ void __launch_bounds__(res_wide_threads(sizeof(T), ONE)) residual_norm_backward_wide_kernel(const ResArgs a) {
  constexpr int TH = res_wide_threads(sizeof(T), ONE);
  __shared__ float2 red[2][16];
  Wide<T> t(a);
  t.row = blockIdx.x;
  t.st = a.stats ? a.stats[t.row] : make_float4(0.f, 0.f, 0.f, 0.f);
  t.mean = make_float4(0.f, 0.f, 0.f, 0.f);
  t.place(threadIdx.x * VE);
  if constexpr (ONE) t.fetch_row();
  const float inv_d = 1.f / (float)a.d;
  if (a.dh) {
    float2 m = make_float2(0.f, 0.f);
    wide_pass<ONE>(t, false, false, [&] {
      float hat[VE], dh[VE], cw[VE];
      t.pre(hat, dh, cw);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        m.x += cw[e];
        m.y += t.c + e < a.d ? cw[e] * hat[e] : 0.f;
      }
    });
    m = row_sum2<TH>(m, red[0]);
    t.mean.x = a.pre == NORM_LAYER ? m.x * inv_d : 0.f;
    t.mean.y = m.y * inv_d;
  }
  if (a.f && a.post != NORM_NONE) {
    float2 m = make_float2(0.f, 0.f);
    wide_pass<ONE>(t, false, false, [&] {
      float v[VE], fh[VE], dw[VE], dg[VE];
      t.dyt(v);
      t.post(v, fh, dw, dg);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        m.x += t.c + e < a.d ? dw[e] : 0.f;
        m.y += t.c + e < a.d ? dw[e] * fh[e] : 0.f;
      }
    });
    m = row_sum2<TH>(m, red[1]);
    t.mean.z = a.post == NORM_LAYER ? m.x * inv_d : 0.f;
    t.mean.w = m.y * inv_d;
  }
  wide_pass<ONE>(t, false, false, [&] {
    float v[VE], fh[VE], dw[VE], dg[VE];
    t.dyt(v);
    if (a.dx) st_row(reinterpret_cast<T*>(a.dx) + t.row * a.lddx, t.c, a.d, v);
    if (!a.f) return;
    t.post(v, fh, dw, dg);
    if (a.dgate && a.gate_every == 1) {
      if (a.gate.dt == 1) st_row(reinterpret_cast<bf16_t*>(a.dgate) + t.row * a.lddg, t.c, a.d, dg);
      else st_row(reinterpret_cast<float*>(a.dgate) + t.row * a.lddg, t.c, a.d, dg);
    }
    if (a.post != NORM_NONE) {
#pragma unroll
      for (int e = 0; e < VE; ++e) dw[e] = (dw[e] - t.mean.z - fh[e] * t.mean.w) * t.st.w;
    }
    if (a.df) st_row(reinterpret_cast<T*>(a.df) + t.row * a.lddf, t.c, a.d, dw);
  });
  if (threadIdx.x == 0) a.means[t.row] = t.mean;
}

// one workgroup: 2048 columns of `chunk` rows (the same split of the rows as the register kernel's)
template <typename T>
__global__ void __launch_bounds__(256) residual_norm_columns_kernel(const ResArgs a, int strips) {
  const long long wg = blockIdx.x / strips;
  const int c = ((int)(blockIdx.x % strips) * 256 + threadIdx.x) * VE;
  if (c >= a.d) return;
  long long r0, r1;
  if (a.per_gate > 1) {
    const long long gate = wg / a.per_gate;
    r0 = gate * a.gate_every + wg % a.per_gate * a.chunk;
    r1 = min(r0 + a.chunk, (gate + 1) * a.gate_every);
  } else {
    r0 = wg * a.chunk;
    r1 = min(r0 + a.chunk, a.rows);
  }
  float s[4][VE] = {}, sg[VE] = {};
  Wide<T> t(a);
  t.place(c);
  t.fetch_shared(false);
  for (t.row = r0; t.row < r1; ++t.row) {
    const long long row = t.row;
    t.st = a.stats ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
    t.mean = a.means[row];
    t.fetch_row();
    float v[VE];
    t.dyt(v);
    if (a.dh) {
      float hat[VE], dh[VE], cw[VE];
      t.pre(hat, dh, cw);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        s[kSumPreW][e] += dh[e] * hat[e];
        s[kSumPreB][e] += dh[e];
      }
    }
    if (a.f) {
      float fh[VE], dw[VE], dg[VE];
      t.post(v, fh, dw, dg);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        s[kSumPostW][e] += v[e] * fh[e];
        s[kSumPostB][e] += v[e];
        sg[e] += dg[e];
      }
      if (a.gpart && (row + 1 == r1 || (a.per_gate == 1 && (row + 1) % a.gate_every == 0))) {
        st_row(a.gpart + (a.per_gate == 1 ? row / a.gate_every : wg) * a.d, c, a.d, sg);
#pragma unroll
        for (int e = 0; e < VE; ++e) sg[e] = 0.f;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (a.slot[k] >= 0) st_row(a.part + ((long long)a.slot[k] * a.parts + wg) * a.d, c, a.d, s[k]);
}

// A workgroup adds 64 columns of one output: wave w the rows w, w + 16, ..., then the 16 sums in order. It takes one such
// strip after the other: a gate for every few rows has millions of them, and a launch holds less than 2^32 threads (one of
// exactly that many is accepted and runs nothing).
__global__ void __launch_bounds__(1024) column_sums_kernel(const ColumnSums s, long long total) {
  __shared__ float red[16][64];
  const int strips = (s.d + 63) / 64;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  for (long long at = blockIdx.x; at < total; at += gridDim.x) {
    long long i = at / strips;
    int k = 0;
    while (i >= s.e[k].groups) i -= s.e[k++].groups;
    const int c = (int)(at % strips) * 64 + lane;
    const float* in = s.e[k].in + i * s.e[k].per * s.d;
    float v = 0.f;
    if (c < s.d) {
#pragma unroll 8
      for (long long p = w; p < s.e[k].per; p += 16) v += in[p * s.d + c];
    }
    red[w][lane] = v;
    __syncthreads();
    if (w == 0 && c < s.d) {
      for (int q = 1; q < 16; ++q) v += red[q][lane];
      const long long o = i * s.e[k].ldo + c;
      if (s.e[k].dt == 1) reinterpret_cast<bf16_t*>(s.e[k].out)[o] = f32_to_bf16(v);
      else reinterpret_cast<float*>(s.e[k].out)[o] = v;
    }
    __syncthreads();  // red is free again
  }
}

}  // namespace

void residual_norm_split(ResArgs& a, bool gate_sums) {
  // as many workgroups as are on the GPU's 256 CUs at once: one more would begin when all the others
  // end (1024 of them where 512 or 768 fit: 16384 rows of 1024 bf16 58 us in place of 47, 33280 of 512 fp32 102 / 87)
  const long long at_once = a.d <= 512 ? 4 : a.d <= 1024 ? 2 : 1;
  const int waves = res_waves(a.d <= 2048 ? 256 : a.d <= 4096 ? 512 : 1024, res_has(a), a.dt == 1 ? 2 : 4);
  const long long target = res_backward_wide(a) ? 1024 : a.d <= 2048 ? 256 * waves : a.d <= 4096 ? 128 * waves : 256;
  a.chunk = a.rows > target ? (a.rows + target - 1) / target : 1;
  a.chunk = (a.chunk + at_once - 1) / at_once * at_once;
  a.per_gate = 1;
  if (gate_sums && a.gate_every > 1) {
    if (a.chunk >= a.gate_every) a.chunk = (a.chunk + a.gate_every - 1) / a.gate_every * a.gate_every;
    else {
      const long long parts = std::max(1ll, target / (a.rows / a.gate_every));  // of each gate's rows
      a.chunk = (a.gate_every + parts - 1) / parts;
      a.chunk = std::min((a.chunk + at_once - 1) / at_once * at_once, a.gate_every);
      a.per_gate = (a.gate_every + a.chunk - 1) / a.chunk;
    }
  }
  a.parts = a.per_gate > 1 ? a.rows / a.gate_every * a.per_gate : (a.rows + a.chunk - 1) / a.chunk;
}

template <typename T, int TPR, int HAS, bool RAGGED>
static void residual_norm_backward_has(const ResArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.parts), block(res_threads(TPR));
#define PSGDK_RES(SUMS, args) \
  hipLaunchKernelGGL((residual_norm_backward_kernel<T, TPR, HAS, SUMS, RAGGED>), grid, block, 0, st, args)
  if constexpr (TPR < 1024) {
    PSGDK_RES(7, a);
  } else {  // no registers for all sums: the branch's come from a second pass
    PSGDK_RES(1, a);
    if constexpr ((HAS & (kPost | kGate)) != 0) {
      ResArgs q = a;
      q.dx = q.df = q.dgate = nullptr;
      q.slot[kSumPreW] = q.slot[kSumPreB] = -1;
      if (a.gpart || a.slot[kSumPostW] >= 0 || a.slot[kSumPostB] >= 0) PSGDK_RES(6, q);
    }
  }
#undef PSGDK_RES
}
template <typename T, int TPR, bool RAGGED>
static void residual_norm_backward_sized(const ResArgs& a, hipStream_t st) {
  switch (res_has(a)) {
    case 0: return residual_norm_backward_has<T, TPR, 0, RAGGED>(a, st);
    case 1: return residual_norm_backward_has<T, TPR, 1, RAGGED>(a, st);
    case 2:
      if constexpr (TPR < 1024 || !RAGGED || sizeof(T) == 2) return residual_norm_backward_has<T, TPR, 2, RAGGED>(a, st);
      break;
    case 4: return residual_norm_backward_has<T, TPR, 4, RAGGED>(a, st);
  }
  if constexpr (TPR < 1024) {
    switch (res_has(a)) {
      case 3: return residual_norm_backward_has<T, TPR, 3, RAGGED>(a, st);
      case 5: return residual_norm_backward_has<T, TPR, 5, RAGGED>(a, st);
      case 6: return residual_norm_backward_has<T, TPR, 6, RAGGED>(a, st);
      default: return residual_norm_backward_has<T, TPR, 7, RAGGED>(a, st);
    }
  }
}
template <typename T, int TPR>
static void residual_norm_backward_sized(const ResArgs& a, hipStream_t st) {
  return a.d % VE ? residual_norm_backward_sized<T, TPR, true>(a, st) : residual_norm_backward_sized<T, TPR, false>(a, st);
}
template <typename T>
static hipError_t residual_norm_backward_t(const ResArgs& a, hipStream_t st) {
  if (!res_backward_wide(a)) {
    if (a.d <= 512) residual_norm_backward_sized<T, 64>(a, st);
    else if (a.d <= 1024) residual_norm_backward_sized<T, 128>(a, st);
    else if (a.d <= 2048) residual_norm_backward_sized<T, 256>(a, st);
    else if (a.d <= 4096) residual_norm_backward_sized<T, 512>(a, st);
    else residual_norm_backward_sized<T, 1024>(a, st);
  } else {
    if (a.d <= 1024 * VE)
      hipLaunchKernelGGL((residual_norm_backward_wide_kernel<T, true>), dim3((unsigned)a.rows), dim3(1024), 0, st, a);
    else
      hipLaunchKernelGGL((residual_norm_backward_wide_kernel<T, false>), dim3((unsigned)a.rows),
                         dim3(res_wide_threads(sizeof(T), false)), 0, st, a);
    bool any = a.gpart != nullptr;
    for (int k = 0; k < 4; ++k) any = any || a.slot[k] >= 0;
    const int strips = (a.d + 256 * VE - 1) / (256 * VE);
    if (any)
      hipLaunchKernelGGL(residual_norm_columns_kernel<T>, dim3((unsigned)(a.parts * strips)), dim3(256), 0, st, a, strips);
  }
  return hipGetLastError();
}
hipError_t residual_norm_backward_launch(const ResArgs& a, hipStream_t st) {
  return a.dt == 1 ? residual_norm_backward_t<bf16_t>(a, st) : residual_norm_backward_t<float>(a, st);
}

hipError_t column_sums_launch(const ColumnSums& s, hipStream_t st) {
  long long groups = 0;
  for (int k = 0; k < s.n; ++k) groups += s.e[k].groups;
  if (!groups) return hipSuccess;
  const long long total = groups * ((s.d + 63) / 64);
  hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)std::min(total, 1ll << 16)), dim3(1024), 0, st, s, total);
  return hipGetLastError();
}

}  // namespace psgdk
