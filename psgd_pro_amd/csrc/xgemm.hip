// The bf16 products of the cross entropy on v_mfma_f32_32x32x16_bf16, operands moved from HBM straight into LDS.
#include "xgemm.h"

namespace psgdk {

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
#define LDS_AS __attribute__((address_space(3)))

// One operand's tile of R rows (m or n) x BK k in LDS, filled by loads that write LDS directly (16 bytes a lane, 1 KB a
// wave in lane order), so any reordering against bank conflicts is in which global chunk a lane asks for.
//   k-contiguous (MC false): rows of BK k, their 16-byte chunks XORed by the row so that the 16 rows of a quarter wave's
//     fragment read lie in 16 different 16-byte bank groups.
//   mn-contiguous (MC true): rows of R m or n for each k, read transposed (ds_read_b64_tr_b16: of 16 lanes lane i names
//     the 8 bytes of k row i / 4, columns 4 (i % 4) .., and receives column i of 4 k rows). A fragment read touches 8 k
//     rows of 64 bytes; their 64-byte blocks are XORed by the k row so that these lie in different banks.
template <int R, int BK, bool MC>
struct Tile {
  static constexpr int BYTES = R * BK * 2;
  static constexpr int LOADS = BYTES / 4096;  // of each of the four waves
  static __device__ __forceinline__ int swk(int row) { return BK == 64 ? (row >> 1) & 7 : (row >> 2) & 3; }
  static __device__ __forceinline__ int swm(int k) { return R == 256 ? (k & 3) | (k >> 1 & 4) : k & 3; }

  // chunk of 8 elements (along the contiguous direction) and row that a lane's load i of a wave fetches
  static __device__ __forceinline__ void where(int wave, int lane, int i, int& row, int& chunk) {
    const int j = wave * LOADS + i;
    if constexpr (!MC) {
      constexpr int CPR = BK / 8;
      row = j * (64 / CPR) + lane / CPR;
      chunk = (lane % CPR) ^ swk(row);
    } else {
      constexpr int CPR = R / 8;
      row = j * (64 / CPR) + lane / CPR;
      chunk = (lane % CPR) ^ (swm(row) << 2);
    }
  }
};

// make_rsrc's words, in scalar registers
__device__ __forceinline__ i32x4_t rsrc_words(const void* p, long long bytes) {
  const uint64_t at = (uint64_t)(uintptr_t)p;
  const int n = bytes > 0x7fffffffLL ? 0x7fffffff : bytes < 0 ? 0 : (int)bytes;
  return i32x4_t{__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane(n), 0x00020000};
}
// 16 bytes a lane from the buffer to LDS at `lds` (wave-uniform) + 16 lane; lanes beyond the buffer write zeros. Not the
// builtin: with it the compiler waits for every such load before any LDS read. The waits are load_wait's.
__device__ __forceinline__ void load_lds(i32x4_t rs, int voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "s"(lds)
               : "memory");
}
// all but the newest N loads into LDS of this wave have arrived, its LDS reads are done, and so for the whole workgroup
template <int N>
__device__ __forceinline__ void load_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// The order of one k step: the next step's READS LDS reads spread evenly behind this step's MM MFMAs.
template <int MM, int READS, int G = 0>
__device__ __forceinline__ void interleave() {
  if constexpr (G < MM) {
    constexpr int N = (G + 1) * READS / MM - G * READS / MM;
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    if constexpr (N > 0) __builtin_amdgcn_sched_group_barrier(0x100, N, 0);
    interleave<MM, READS, G + 1>();
  }
}

}  // namespace

// Four waves, 2 x 2, each WTM x WTN of the output. ST stages of BK k in LDS.
template <int WTM, int WTN, int BK, int ST, bool MCA, bool MCB, int KIND, bool OUTF>
__global__ void __launch_bounds__(256, WTM * WTN > 128 * 64 ? 1 : 2) xgemm_kernel(const XgArgs p) {
  constexpr int BM = 2 * WTM, BN = 2 * WTN, FM = WTM / 32, FN = WTN / 32, KS = BK / 16;
  using TA = Tile<BM, BK, MCA>;
  using TB = Tile<BN, BK, MCB>;
  constexpr int STAGE = TA::BYTES + TB::BYTES, LOADS = TA::LOADS + TB::LOADS;
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned lds0 = (unsigned)(uintptr_t)(LDS_AS unsigned char*)smem;

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave >> 1, wn = wave & 1;
  const int ntiles = p.redo ? p.redo[0] * p.tiles_m : p.tiles_m * p.tiles_n * p.splits;
  for (int w = blockIdx.x; w < ntiles; w += gridDim.x) {
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // what follows from it is made again for each tile, not kept through the epilogue
  const int c = lane & 31, hh = lane >> 5;
  int ti, tj, split = 0;
  if (p.redo) {
    ti = w % p.tiles_m;
    tj = p.redo[1 + w / p.tiles_m];
  } else {
    // each XCD a contiguous run of tiles, 4 tiles of m by n after n, so that the tiles it runs at once share panels
    constexpr int GM = 4;
    int tile = xcd_run(w, ntiles);
    split = tile / (p.tiles_m * p.tiles_n);
    tile -= split * (p.tiles_m * p.tiles_n);
    const int grp = tile / (GM * p.tiles_n), r0 = grp * GM, gm = min(GM, p.tiles_m - r0), idx = tile - r0 * p.tiles_n;
    ti = r0 + idx % gm;
    tj = idx / gm;
  }
  const int m0 = ti * BM, n0 = tj * BN;
  const int kb = split * p.kchunk, ke = min(p.K, kb + p.kchunk);
  const int nk = (ke - kb + BK - 1) / BK;

  // byte offsets of this lane's loads inside a tile
  int va[TA::LOADS], vb[TB::LOADS];
#pragma unroll
  for (int i = 0; i < TA::LOADS; ++i) {
    int row, ch;
    TA::where(wave, lane, i, row, ch);
    va[i] = (int)((long long)row * p.lda + ch * 8) * 2;
  }
#pragma unroll
  for (int i = 0; i < TB::LOADS; ++i) {
    int row, ch;
    TB::where(wave, lane, i, row, ch);
    vb[i] = (int)((long long)row * p.ldb + ch * 8) * 2;
  }
  auto issue = [&](int t) {
    const int k0 = kb + t * BK;
    const bool live = t < nk;
    unsigned base = lds0 + (unsigned)(t % ST) * STAGE;
    const bf16_t* pa = p.A + (MCA ? (long long)k0 * p.lda + m0 : (long long)m0 * p.lda + k0);
    const bf16_t* pb = p.B + (MCB ? (long long)k0 * p.ldb + n0 : (long long)n0 * p.ldb + k0);
    i32x4_t ra = rsrc_words(pa, !live ? 0 : 2 * (MCA ? (long long)(min(ke, p.kreal) - k0 - 1) * p.lda + ((p.M - m0 + 7) & ~7)
                                                           : (long long)(p.M - m0 - 1) * p.lda + (ke - k0)));
    i32x4_t rb = rsrc_words(pb, !live ? 0 : 2 * (MCB ? (long long)(ke - k0 - 1) * p.ldb + ((p.N - n0 + 7) & ~7)
                                                           : (long long)(p.N - n0 - 1) * p.ldb + (ke - k0)));
    // a scalar register that a vector instruction wrote may be read by a load 5 wait states later at the earliest, which
    // the compiler does not see to inside asm statements
    asm volatile("s_nop 4" : "+s"(ra), "+s"(rb), "+s"(base));
    const bool whole = k0 + BK <= ke;
#pragma unroll
    for (int i = 0; i < TA::LOADS; ++i) {
      int v = va[i];
      if (!MCA && !whole) {
        int row, ch;
        TA::where(wave, lane, i, row, ch);
        v = k0 + ch * 8 < ke ? v : kOob;
      }
      load_lds(ra, v, base + (unsigned)(wave * TA::LOADS + i) * 1024);
    }
#pragma unroll
    for (int i = 0; i < TB::LOADS; ++i) {
      int v = vb[i];
      if (!MCB && !whole) {
        int row, ch;
        TB::where(wave, lane, i, row, ch);
        v = k0 + ch * 8 < ke ? v : kOob;
      }
      load_lds(rb, v, base + TA::BYTES + (unsigned)(wave * TB::LOADS + i) * 1024);
    }
  };

  // LDS offsets of this lane's fragment reads inside a stage: k-contiguous operands by k step, others by 32-block
  unsigned oa[MCA ? FM : KS], ob[MCB ? FN : KS];
  const int rr = (lane & 15) >> 2;
#pragma unroll
  for (int i = 0; i < (MCA ? FM : KS); ++i)
    oa[i] = MCA ? (8 * hh + rr) * BM * 2 + ((((wm * WTM + 32 * i) >> 5) ^ TA::swm(8 * hh + rr)) << 6) + (lane >> 4 & 1) * 32 +
                      (lane & 3) * 8
                : (wm * WTM + c) * BK * 2 + (((2 * i + hh) ^ TA::swk(c)) << 4);
#pragma unroll
  for (int i = 0; i < (MCB ? FN : KS); ++i)
    ob[i] = TA::BYTES +
            (MCB ? (8 * hh + rr) * BN * 2 + ((((wn * WTN + 32 * i) >> 5) ^ TB::swm(8 * hh + rr)) << 6) + (lane >> 4 & 1) * 32 +
                       (lane & 3) * 8
                 : (wn * WTN + c) * BK * 2 + (((2 * i + hh) ^ TB::swk(c)) << 4));

  auto tr = [](unsigned at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4_t*)(uintptr_t)at);
  };
  auto pair = [&](unsigned at, int pitch4) {
    union {
      s16x4_t h[2];
      bf16x8_t v;
    } u;
    u.h[0] = tr(at);
    u.h[1] = tr(at + pitch4);
    return u.v;
  };
  bf16x8_t fa[2][FM], fb[2][FN];
  auto frags = [&](int set, unsigned base, int ks) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      if constexpr (MCB) fb[set][j] = pair(base + ob[j] + ks * 16 * BN * 2, 4 * BN * 2);
      else fb[set][j] = *(LDS_AS bf16x8_t*)(uintptr_t)(base + ob[ks] + j * 32 * BK * 2);
    }
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      if constexpr (MCA) fa[set][i] = pair(base + oa[i] + ks * 16 * BM * 2, 4 * BM * 2);
      else fa[set][i] = *(LDS_AS bf16x8_t*)(uintptr_t)(base + oa[ks] + i * 32 * BK * 2);
    }
  };

  f32x16_t acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

#pragma unroll
  for (int t = 0; t < ST; ++t) issue(t);
  load_wait<(ST - 1) * LOADS>();
  frags(0, lds0, 0);
  static_assert(KS % 2 == 0, "fragment sets alternate over whole tiles");
  constexpr int READS = FM * (MCA ? 2 : 1) + FN * (MCB ? 2 : 1), MM = FM * FN;
  for (int kt = 0; kt < nk; ++kt) {
    const unsigned base = lds0 + (unsigned)(kt % ST) * STAGE, next = lds0 + (unsigned)((kt + 1) % ST) * STAGE;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int cur = ks & 1;
      if (ks + 1 < KS) {
        frags(cur ^ 1, base, ks + 1);
      } else {
        load_wait<(ST - 2) * LOADS>();
        issue(kt + ST);
        frags(cur ^ 1, next, 0);
      }
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[cur][i], fb[cur][j], acc[i][j], 0, 0, 0);
      interleave<MM, READS>();
    }
  }
  load_wait<0>();  // LDS is the epilogue's now

  // Element e of acc[i][j]: m = 32 i + 8 (e / 4) + 4 hh + e % 4, n = 32 j + c of the wave's block: 4 consecutive m a
  // lane. The block is put together in LDS (rows n of WTM 16-bit values, 16-byte chunks XORed by n) and leaves in rows of
  // 16-byte stores.
  const int mw = m0 + wm * WTM, nw = n0 + wn * WTN;
  if constexpr (OUTF) {
    float* const o = p.outf + (long long)split * p.N * p.ldo;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = nw + 32 * j + c;
      if (n >= p.N) continue;
      float* const q = o + (long long)n * p.ldo + mw + 4 * hh;
#pragma unroll
      for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int m = 32 * i + 8 * g;
          if (mw + 4 * hh + m >= p.M) continue;
          f32x4_t v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
          if (p.accumulate) v += *reinterpret_cast<const f32x4_t*>(q + m);
          *reinterpret_cast<f32x4_t*>(q + m) = v;
        }
    }
    return;
  }
  unsigned char* const ep = smem + wave * WTN * WTM * 2;
  constexpr int CH = WTM / 8;
  auto slot = [&](int n, int ch) { return ep + n * WTM * 2 + ((ch ^ (n & (CH - 1))) << 4); };
  if constexpr (KIND == XG_LOGITS) {
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = nw + 32 * j + c;
      const bool row = n < p.N;
      const float r = row ? p.ref[n] : 0.f;
      const int t = row ? p.target[n] : -1;
      const int tl = t - mw - 4 * hh;  // the target as a column of this lane's first group
      const bool inside = mw + WTM <= p.M && !__any(tl >= -4 && tl < WTM + 4);
      constexpr float L2E = 1.4426950408889634f;
      // pknorm: x 32767 to the nearest, clamped; x = ((z - r) - low - 64) / (64 32767 / 32768)
      constexpr float QS = 32768.f / 32767.f / 64.f;
      const float e0 = -r * L2E, q0 = (-r - kLogitLow - 64.f) * QS;
      float s = 0.f, top = -INFINITY;
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        asm volatile("" : "+a"(acc[i][j]));  // accumulators leave their registers tile by tile, not all at once
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float z[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) z[e] = acc[i][j][4 * g + e];
          const int m = 32 * i + 8 * g + 4 * hh;
          if (p.max_only) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (mw + m + e < p.M) top = fmaxf(top, z[e]);
          } else if (inside) {
#pragma unroll
            for (int e = 0; e < 4; ++e) s += __builtin_amdgcn_exp2f(__builtin_fmaf(z[e], L2E, e0));
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const bool other = mw + m + e < p.M && mw + m + e != t;
              s += other ? __builtin_amdgcn_exp2f(__builtin_fmaf(z[e], L2E, e0)) : 0.f;
            }
          }
          if (p.q) {
            const auto lo = __builtin_amdgcn_cvt_pknorm_i16(__builtin_fmaf(z[0], QS, q0), __builtin_fmaf(z[1], QS, q0));
            const auto hi = __builtin_amdgcn_cvt_pknorm_i16(__builtin_fmaf(z[2], QS, q0), __builtin_fmaf(z[3], QS, q0));
            uint2 w;
            __builtin_memcpy(&w.x, &lo, 4);
            __builtin_memcpy(&w.y, &hi, 4);
            *reinterpret_cast<uint2*>(slot(32 * j + c, 4 * i + g) + hh * 8) = w;
          }
        }
      }
      if (p.max_only) {
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (row && hh == 0) p.tops[(long long)n * 2 * p.tiles_m + 2 * ti + wm] = top;
      } else {
        s += __shfl_xor(s, 32, 64);
        if (row && hh == 0) p.sums[(long long)n * 2 * p.tiles_m + 2 * ti + wm] = t < 0 ? 0.f : s;
      }
    }
    if (!p.q) continue;
  } else {
    const float al = p.alpha ? p.alpha[0] : 1.f;
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int i = 0; i < FM; ++i) {
        asm volatile("" : "+a"(acc[i][j]));  // accumulators leave their registers tile by tile, not all at once
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<uint2*>(slot(32 * j + c, 4 * i + g) + hh * 8) =
              make_uint2(pack2_bf16(al * acc[i][j][4 * g], al * acc[i][j][4 * g + 1]),
                         pack2_bf16(al * acc[i][j][4 * g + 2], al * acc[i][j][4 * g + 3]));
      }
  }
  __syncthreads();
  uint16_t* const out = KIND == XG_LOGITS ? reinterpret_cast<uint16_t*>(p.q) : p.out;
#pragma unroll 4
  for (int it = 0; it < WTN * CH / 64; ++it) {
    const int idx = it * 64 + lane, n = idx / CH, ch = idx % CH, m = mw + 8 * ch;
    if (nw + n >= p.N || m >= p.M) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(slot(n, ch));
    uint16_t* o = out + (long long)(nw + n) * p.ldo + m;
    if (m + 8 <= p.M) {
      __builtin_memcpy(o, &v, 16);
    } else {
      uint16_t h[8];
      __builtin_memcpy(h, &v, 16);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (m + e < p.M) o[e] = h[e];
    }
  }
  if constexpr (KIND != XG_LOGITS) return;
  __syncthreads();  // LDS is the next tile's
  }
}

template <int WTM, int WTN, int BK, int ST, bool MCA, bool MCB, int KIND, bool OUTF = false>
static hipError_t launch_x(XgArgs& a, hipStream_t st) {
  constexpr int smem_main = ST * (Tile<2 * WTM, BK, MCA>::BYTES + Tile<2 * WTN, BK, MCB>::BYTES), smem_epi = 4 * WTM * WTN * 2;
  constexpr int smem = smem_main > smem_epi ? smem_main : smem_epi;
  void (*fn)(XgArgs) = xgemm_kernel<WTM, WTN, BK, ST, MCA, MCB, KIND, OUTF>;
  static const hipError_t attr =
      hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (attr != hipSuccess) return attr;
  a.tiles_m = (a.M + 2 * WTM - 1) / (2 * WTM);
  a.tiles_n = (a.N + 2 * WTN - 1) / (2 * WTN);
  if (!a.kreal) a.kreal = a.K;
  a.kchunk = a.splits > 1 ? ((a.K + a.splits - 1) / a.splits + BK - 1) / BK * BK : a.K;
  const long long tiles = (long long)a.tiles_m * a.tiles_n * a.splits;
  // tiles to be done again are not known here: one workgroup a CU takes them in turn, and ends at once without any
  hipLaunchKernelGGL(fn, dim3((unsigned)(a.redo && tiles > 256 ? 256 : tiles)), dim3(256), smem, st, a);
  return hipGetLastError();
}

int xgemm_splits(long long M, long long N, long long K) {
  const long long tiles = ((M + 255) / 256) * ((N + 255) / 256);
  long long s = 1;
  while (s < 16 && tiles * s < 256 && K / (s * 2) >= 512) s *= 2;
  return (int)s;
}

hipError_t xgemm_launch(XgArgs& a, int kind, hipStream_t st) {
  if (kind == XG_LOGITS) return launch_x<128, 128, 64, 2, false, false, XG_LOGITS>(a, st);
  if (kind == XG_DX)
    return a.outf ? launch_x<128, 128, 64, 2, true, false, XG_DX, true>(a, st)
                  : launch_x<128, 128, 64, 2, true, false, XG_DX>(a, st);
  return a.outf ? launch_x<128, 128, 64, 2, true, true, XG_DW, true>(a, st)
                : launch_x<128, 128, 64, 2, true, true, XG_DW>(a, st);
}

}  // namespace psgdk
