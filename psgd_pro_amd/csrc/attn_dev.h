// What the forward and backward attention kernels share: fragments, tiles in LDS, masks.
#pragma once
#include <type_traits>

#include "attn.h"
#include "lds.h"

namespace psgdk {

// Products are 32 x 32 blocks, C[m][n] += sum_k A[m][k] B[n][k], 16 k at a time. A lane holds 8 k of row m (or n) lane % 32,
// those of half h = lane / 32. Of C it holds column n = lane % 32 and rows 8 (r / 4) + 4 h + r % 4, r = 0 .. 15.
// Which 8 of the 16 k belong to a half is free as long as A and B agree:
//   straight: 8 h .. 8 h + 7                       (operands read along k)
//   crossed:  4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3  (a C block of the product before is an operand as it lies)
template <typename T>
struct Frag {
  typedef float type __attribute__((ext_vector_type(8)));
};
template <>
struct Frag<bf16_t> {
  typedef bf16x8_t type;
};
template <typename T>
using frag_t = typename Frag<T>::type;

__device__ __forceinline__ f32x16_t mma(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
// fp32: eight products of two k, one of each half (157 TFLOP/s at most)
__device__ __forceinline__ f32x16_t mma(Frag<float>::type a, Frag<float>::type b, f32x16_t c) {
#pragma unroll
  for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
  return c;
}

// 8 values of a C block (r = 8 u .. 8 u + 7) as a crossed operand: k = 16 u + ...
template <typename T>
__device__ __forceinline__ frag_t<T> crossed(const f32x16_t& c, int u) {
  if constexpr (std::is_same_v<T, float>) {
    return frag_t<T>{c[8 * u], c[8 * u + 1], c[8 * u + 2], c[8 * u + 3], c[8 * u + 4], c[8 * u + 5], c[8 * u + 6], c[8 * u + 7]};
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack2_bf16(c[8 * u + 2 * i], c[8 * u + 2 * i + 1]);
    frag_t<T> f;
    __builtin_memcpy(&f, w, 16);
    return f;
  }
}

// what rounding took from those 8 values, f being crossed's
__device__ __forceinline__ bf16x8_t crossed_rest(const f32x16_t& c, int u, bf16x8_t f) {
  f32x16_t r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = c[8 * u + i] - (float)f[i];
  return crossed<bf16_t>(r, 0);
}

// sum + the 8 values
__device__ __forceinline__ float sum_of(bf16x8_t f, float sum) {
  typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
  const bf16x2_t one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2_t{f[2 * i], f[2 * i + 1]}, one, sum, false);
  return sum;
}
__device__ __forceinline__ float sum_of(Frag<float>::type f, float sum) {
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += f[i];
  return sum;
}

// R rows of DP elements in LDS, each row's 16-byte chunks XORed by a function of the row. With bf16: the 16 rows of a quarter
// wave's fragment read lie in 16 different 16-byte bank groups, and so do the 4 rows x 64 bytes of half a transposed read
// (its low two bits from row / 4, the others, which choose among a 64-byte block's places, from row % 4). With fp32 the same
// for fragment reads; a transposed read is 32 columns of two rows that lie 4 apart (rows of 256 bytes and more).
template <typename T, int DP>
struct Rows {
  static constexpr int E = sizeof(T), PER = 16 / E, CPR = DP / PER, PITCH = DP * E;
  static __device__ __forceinline__ int swz(int row) {
    if constexpr (E == 2) {
      const int low = row >> 2 & 3;
      return DP == 128 ? low | (row & 3) << 2 : DP == 64 ? low | (row >> 1 & 1) << 2 : low;
    } else {
      return DP % 64 == 0 ? (row & 3) | (row >> 3 & 1) << 2 | (row >> 2 & 1) << 3 : row >> 1 & 7;
    }
  }
  static __device__ __forceinline__ unsigned at(int row, int chunk) { return row * PITCH + ((chunk ^ swz(row)) << 4); }
  // loads of 1 KB of each of W waves for R rows
  static constexpr int loads(int R, int W) { return R * PITCH / 1024 / W; }
  // row and chunk that lane `lane` of load j of a tile fetches
  static __device__ __forceinline__ void where(int j, int lane, int& row, int& chunk) {
    const int c = j * 64 + lane;
    row = c / CPR;
    chunk = (c % CPR) ^ swz(row);
  }
};

// Fragments of Rows tiles: a tile's address with the lane's part once, then constants. What the swizzle lets pass as an XOR of
// the address where rows are a power of two long (tiles begin at multiples of 1024) is one there; else the chunk's upper bits,
// which the swizzle leaves alone, are added.
// k along the row: row 32 block + lane % 32, k = 16 c + 8 h ..
template <typename T, int DP>
struct Straight {
  using R = Rows<T, DP>;
  unsigned at;
  __device__ __forceinline__ Straight(unsigned base, int lane)
      : at(base + (lane & 31) * R::PITCH + (((R::E == 2 ? 1 : 2) * (lane >> 5) ^ R::swz(lane & 31)) << 4)) {}
  __device__ __forceinline__ frag_t<T> operator()(int block, int c) const {
    constexpr bool POW2 = (DP & (DP - 1)) == 0;
    if constexpr (R::E == 2) {
      const unsigned p = POW2 ? at ^ c << 5 : (at ^ (c & 1) << 5) + (c >> 1) * 64;
      return *(LDS_AS frag_t<T>*)(uintptr_t)(p + block * 32 * R::PITCH);
    } else {
      const unsigned p = POW2 ? at ^ c << 6 : (at ^ (c & 1) << 6) + (c >> 1) * 128, q = p + block * 32 * R::PITCH;
      const f32x4_t x = *(LDS_AS f32x4_t*)(uintptr_t)q, y = *(LDS_AS f32x4_t*)(uintptr_t)(q ^ 16);
      return frag_t<T>{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
    }
  }
};
// k along the column: column 32 t + lane % 32, rows 16 u + 4 h .. and 16 u + 8 + 4 h ..
template <typename T, int DP>
struct Transposed {
  using R = Rows<T, DP>;
  unsigned at, sw;
  __device__ __forceinline__ Transposed(unsigned base, int lane) {
    const int h = lane >> 5;
    if constexpr (R::E == 2) {
      // of 16 lanes lane i names the 8 bytes of row i / 4, columns 4 (i % 4) .., and receives column i of the 4 rows
      const int i = lane & 15, row = 4 * h + (i >> 2);
      at = base + row * R::PITCH + ((((lane >> 3 & 2) + (i >> 1 & 1)) ^ R::swz(row)) << 4) + (i & 1) * 8;
    } else {
      at = base + 4 * h * R::PITCH + (lane & 3) * 4;
      sw = (lane >> 2 & 7) ^ R::swz(4 * h);
    }
  }
  __device__ __forceinline__ frag_t<T> operator()(int u, int t) const {
    constexpr bool XOR = DP == 64 || DP == 128;
    if constexpr (R::E == 2) {
      union {
        s16x4_t v[2];
        frag_t<T> f;
      } w;
#pragma unroll
      for (int x = 0; x < 2; ++x) {  // (8 rows on, row / 4 differs by 2)
        const unsigned p = XOR ? at ^ (t << 6 | x << 5) : (at ^ x << 5) + t * 64;
        w.v[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4_t*)(uintptr_t)(p + (16 * u + 8 * x) * R::PITCH));
      }
      return w.f;
    } else {
      frag_t<T> f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {  // (the swizzle is linear: a row's is the XOR of its parts')
        const int row = (e & 4) * 2 + (e & 3);
        f[e] = *(LDS_AS float*)(uintptr_t)(at + (16 * u + row) * R::PITCH + ((sw ^ R::swz(row) ^ 8 * t) << 4));
      }
      return f;
    }
  }
};

// N steps of load(i) and use(i, fragment), each load D steps ahead of its use (left to itself the compiler loads, waits and
// multiplies one after the other)
template <typename T, int N, int D, typename Load, typename Use>
__device__ __forceinline__ void ahead(frag_t<T> (&f)[D], Load load, Use use) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    use(i, f[i % D]);
    if (i + D < N) f[i % D] = load(i + D);
    __builtin_amdgcn_sched_barrier(0);
  }
}
template <typename T, int D, typename Load>
__device__ __forceinline__ void first_loads(frag_t<T> (&f)[D], Load load) {
#pragma unroll
  for (int i = 0; i < D; ++i) f[i] = load(i);
  __builtin_amdgcn_sched_barrier(0);
}

// 8 elements at p + k for k = 16 c + 8 h, zeros from d on (d a multiple of 8) or where !ok; `some` is what is read then (no
// branch: the loads of a row are on their way together)
template <typename T>
__device__ __forceinline__ frag_t<T> row_frag(const T* p, int k, int d, bool ok, const T* some) {
  ok = ok & (k < d);
  const T* const at = ok ? p + k : some;
  frag_t<T> f;
  if constexpr (sizeof(T) == 2) {
    f = *reinterpret_cast<const frag_t<T>*>(at);
  } else {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(at), y = *reinterpret_cast<const f32x4_t*>(at + 4);
    f = frag_t<T>{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
  }
  uint32_t w[sizeof f / 4];
  __builtin_memcpy(w, &f, sizeof f);
#pragma unroll
  for (uint32_t& v : w) v = ok ? v : 0;
  __builtin_memcpy(&f, w, sizeof f);
  return f;
}

// Waits for what loads x: in front of a loop whose loads into LDS are on their way, where a wait for x would wait for those too.
template <typename X>
__device__ __forceinline__ void arrived(X& x) {
  asm volatile("" : "+v"(x));
}

__device__ __forceinline__ f32x16_t zero16() {
  f32x16_t z;
#pragma unroll
  for (int i = 0; i < 16; ++i) z[i] = 0.f;
  return z;
}

__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
// part `part` of `parts` of n begins here
__device__ __forceinline__ int part_begin(int n, int part, int parts) { return uniform((int)((long long)n * part / parts)); }

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// over both halves, each lane of which gets it
__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// a sequence: its tokens and the position of its first query
struct Seq {
  int len, start;
};
__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
  Seq s;
  long long len = a.lengths ? a.lengths[b] : a.m, start = a.starts ? a.starts[b] : (long long)a.m - a.n;
  len = len < 0 ? 0 : len > a.m ? a.m : len;
  // (positions behind the last key see nothing, wherever they are)
  start = start < -(1ll << 30) ? -(1ll << 30) : start > (1ll << 30) ? 1ll << 30 : start;
  s.len = __builtin_amdgcn_readfirstlane((int)len);
  s.start = __builtin_amdgcn_readfirstlane((int)start);
  return s;
}
__device__ __forceinline__ int row_token(const AttnArgs& a, int r) { return (int)((uint64_t)(uint32_t)r * a.div >> a.div_shift); }

// Key tiles of BK that rows at positions lo .. hi see: first those that hold sinks, then those of the window.
struct KeyTiles {
  int sinks, first, count;
  __device__ __forceinline__ int tile(int t) const { return t < sinks ? t : first + t - sinks; }
};
template <int BK>
__device__ __forceinline__ KeyTiles key_tiles(const AttnArgs& a, const Seq& s, int lo, int hi) {
  KeyTiles k{0, 0, 0};
  const int end = min(hi + 1, s.len);  // of the keys that any of them sees
  if (end <= 0 || lo >= s.len) return k;
  k.sinks = (min(a.sinks, end) + BK - 1) / BK;
  k.first = max(max(max(lo, 0) - a.window + 1, 0) / BK, k.sinks);
  k.count = k.sinks + max((end + BK - 1) / BK - k.first, 0);
  return k;
}

}  // namespace psgdk
