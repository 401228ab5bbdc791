// The bf16 products of the cross entropy on v_mfma_f32_32x32x16_bf16, operands moved from HBM straight into LDS.
#include <cmath>
#include <type_traits>

#include "xgemm.h"

namespace psgdk {

namespace {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
// A wave's way out holds one after the other what its loads wrote, 16-bit results and rows of them: its numbers are read by
// types that may alias all of those, so that no read moves past a write of another type to the same bytes.
typedef float lds_float __attribute__((may_alias));
typedef int lds_int __attribute__((may_alias));
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
// the same with 4 bytes a lane
__device__ __forceinline__ void load_lds4(i32x4_t rs, int voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "s"(lds)
               : "memory");
}
// all but the newest N loads into LDS of this wave have arrived, its LDS reads are done, and so for the whole workgroup
template <int N>
__device__ __forceinline__ void load_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace

// Four waves, 2 x 2, each WTM x WTN of the output; ST stages of BK k in LDS, and a block of 32 x WTM 16-bit values for
// each wave's way out. A workgroup takes one tile after the other; the loads of the next tile's first stages are on their
// way before a tile's results leave. No load that a register waits for may come between: its wait would be for all of them,
// and for the last tile's stores. (REDO, the listed blocks alone, is an instance of its own for its list's loads.)
// Bound by the matrix cores at the clock that their power leaves (1.7-1.8 GHz): 4096 x 4096 x 131072 (4.4 TFLOP a product),
// logits 3.70 ms (1190 TFLOP/s), dx 3.26 (1350), dw 3.35 (1310), the MFMA pipe busy 64, 75 and 72% of the cycles; the
// logits' exponentials and stores are the rest of theirs. Why one workgroup of four 128 x 128 waves a CU: two of 128 x 256
// (logits / dx / dw) 4.60 / 4.09 / 3.53 ms, eight waves of 128 x 64 4.02 / 3.32 / 3.44, k tiles of 32 in four stages
// 4.06 / 3.32 / 3.61.
template <int WTM, int WTN, int BK, int ST, bool MCA, bool MCB, int KIND, bool OUTF, bool REDO>
__global__ void __launch_bounds__(256, 1) xgemm_kernel(const XgArgs p) {
  constexpr int BM = 2 * WTM, BN = 2 * WTN, FM = WTM / 32, FN = WTN / 32, KS = BK / 16;
  using TA = Tile<BM, BK, MCA>;
  using TB = Tile<BN, BK, MCB>;
  constexpr int STAGE = TA::BYTES + TB::BYTES, LOADS = TA::LOADS + TB::LOADS;
  extern __shared__ __align__(1024) unsigned char smem[];
  const unsigned lds0 = (unsigned)(uintptr_t)(LDS_AS unsigned char*)smem;

  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 31, hh = lane >> 5, wm = wave >> 1, wn = wave & 1;

  static_assert(BN == kXgRows, "a listed block is a tile of n");
  const int live = __builtin_amdgcn_readfirstlane(min(max(p.count[0] - p.first, 0), KIND == XG_DW ? p.K : p.N));
  const int N = KIND == XG_DW ? p.N : live, K = KIND == XG_DW ? live : p.K, tiles_n = (N + BN - 1) / BN;
  const int ntiles = REDO ? p.redo[0] * p.tiles_m : p.tiles_m * tiles_n * p.splits;
  if ((int)blockIdx.x >= ntiles || (KIND == XG_DW && p.accumulate && K == 0)) return;
  // tile w of the workgroups' order: its m and n tile and its part of k
  auto where = [&](int w, int& ti, int& tj, int& split) __attribute__((always_inline)) {
    split = 0;
    if constexpr (REDO) {
      ti = w % p.tiles_m;
      tj = p.redo[1 + w / p.tiles_m];
      return;
    }
    // each XCD a contiguous run of tiles, 4 tiles of m by n after n, so that the tiles it runs at once share panels
    constexpr int GM = 4;
    int tile = xcd_run(w, ntiles);
    split = tile / (p.tiles_m * tiles_n);
    tile -= split * (p.tiles_m * tiles_n);
    const int grp = tile / (GM * tiles_n), r0 = grp * GM, gm = min(GM, p.tiles_m - r0), idx = tile - r0 * tiles_n;
    ti = r0 + (gm == GM ? idx % GM : idx % gm);
    tj = gm == GM ? idx / GM : idx / gm;
  };

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
  // The loads, one k tile after the other and on into the next output tile: plan() moves on to the next (and its stage),
  // load(i) issues its load i. The buffers begin at the tile and end with the operand: rows behind it read zeros (k behind
  // the end of a k-contiguous row is the lanes' own check), and behind the last output tile there are only zeros.
  const bf16_t *pa, *pb;
  const long long da = MCA ? (long long)BK * p.lda : BK, db = MCB ? (long long)BK * p.ldb : BK;
  long long ea, eb;
  int wl = blockIdx.x, kp, kl;
  unsigned to = lds0;
  i32x4_t ra, rb;
  int v[LOADS];
  auto begin = [&]() __attribute__((always_inline)) {
    int ti, tj, split;
    where(wl, ti, tj, split);
    const int m0 = ti * BM, n0 = tj * BN;
    kp = split * p.kchunk;
    kl = min(K, kp + p.kchunk);
    pa = p.A + (MCA ? (long long)kp * p.lda + m0 : (long long)m0 * p.lda + kp);
    pb = p.B + (MCB ? (long long)kp * p.ldb + n0 : (long long)n0 * p.ldb + kp);
    ea = MCA ? (long long)(min(kl, p.kreal) - kp - 1) * p.lda + ((p.M - m0 + 7) & ~7)
             : (long long)(p.M - m0 - 1) * p.lda + (kl - kp);
    eb = MCB ? (long long)(kl - kp - 1) * p.ldb + ((N - n0 + 7) & ~7)
             : (long long)(N - n0 - 1) * p.ldb + (kl - kp);
  };
  auto plan = [&](bool first) __attribute__((always_inline)) {
    if (!first) {
      to = to + STAGE == lds0 + ST * STAGE ? lds0 : to + STAGE;
      pa += da;
      pb += db;
      ea -= da;
      eb -= db;
      kp += BK;
      if (kp >= kl) {
        wl += gridDim.x;
        if (wl < ntiles) {
          begin();
        } else {
          ea = eb = 0;
          kl = 0;
        }
      }
    }
    ra = rsrc_words(pa, 2 * ea);
    rb = rsrc_words(pb, 2 * eb);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const bool isa = i < TA::LOADS;
      v[i] = isa ? va[i < TA::LOADS ? i : 0] : vb[i < TA::LOADS ? 0 : i - TA::LOADS];
      if (isa ? !MCA : !MCB) {
        int row, ch;
        if (isa) TA::where(wave, lane, i, row, ch);
        else TB::where(wave, lane, i - TA::LOADS, row, ch);
        v[i] = kp + ch * 8 < kl ? v[i] : kOob;
      }
    }
    // a scalar register that a vector instruction wrote may be read by a load 5 wait states later at the earliest, which
    // the compiler does not see to inside asm statements
    asm volatile("s_nop 4" : "+s"(ra), "+s"(rb), "+s"(to));
  };
  auto load = [&](int i) __attribute__((always_inline)) {
    if (i < TA::LOADS) load_lds(ra, v[i], to + (unsigned)(wave * TA::LOADS + i) * 1024);
    else load_lds(rb, v[i], to + TA::BYTES + (unsigned)(wave * TB::LOADS + i - TA::LOADS) * 1024);
  };

  // LDS offset of this lane's first fragment read inside a stage. The others differ by a constant, and by an XOR of the
  // k step (k-contiguous: chunk 2 ks + hh of the row) or of the 32-block (mn-contiguous), which the swizzles let pass.
  const int rr = (lane & 15) >> 2;
  static_assert((FM & (FM - 1)) == 0 && (FN & (FN - 1)) == 0, "a wave's 32-blocks differ in the lowest bits of their number");
  const unsigned oa = MCA ? (8 * hh + rr) * BM * 2 + (((wm * WTM >> 5) ^ TA::swm(8 * hh + rr)) << 6) + (lane >> 4 & 1) * 32 +
                                (lane & 3) * 8
                          : (wm * WTM + c) * BK * 2 + ((hh ^ TA::swk(c)) << 4);
  const unsigned ob = TA::BYTES +
                      (MCB ? (8 * hh + rr) * BN * 2 + (((wn * WTN >> 5) ^ TB::swm(8 * hh + rr)) << 6) + (lane >> 4 & 1) * 32 +
                                 (lane & 3) * 8
                           : (wn * WTN + c) * BK * 2 + ((hh ^ TB::swk(c)) << 4));

  auto tr = [](unsigned at) __attribute__((always_inline)) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((LDS_AS s16x4_t*)(uintptr_t)at);
  };
  auto pair = [&](unsigned at, int pitch4) __attribute__((always_inline)) {
    union {
      s16x4_t h[2];
      bf16x8_t v;
    } u;
    u.h[0] = tr(at);
    u.h[1] = tr(at + pitch4);
    return u.v;
  };
  bf16x8_t fa[2][FM], fb[2][FN];
  // fragment f of k step ks: B's FN, then A's FM
  auto frag = [&](int set, unsigned base, int ks, int f) __attribute__((always_inline)) {
    if (f < FN) {
      if constexpr (MCB) fb[set][f] = pair(((base + ob) ^ (f << 6)) + ks * 16 * BN * 2, 4 * BN * 2);
      else fb[set][f] = *(LDS_AS bf16x8_t*)(uintptr_t)(((base + ob) ^ (ks << 5)) + f * 32 * BK * 2);
    } else {
      const int i = f - FN;
      if constexpr (MCA) fa[set][i] = pair(((base + oa) ^ (i << 6)) + ks * 16 * BM * 2, 4 * BM * 2);
      else fa[set][i] = *(LDS_AS bf16x8_t*)(uintptr_t)(((base + oa) ^ (ks << 5)) + i * 32 * BK * 2);
    }
  };

  // the state in front of a tile's first step: its ST - 1 first k tiles and the first share of the next are on their way
  constexpr int MM = FM * FN, FR = FM + FN, PER = KS > 2 ? (LOADS + KS - 2) / (KS - 1) : (LOADS + KS - 1) / KS;
  begin();
  for (int t = 0; t < ST; ++t) {
    plan(t == 0);
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      if (i < PER || t + 1 < ST) load(i);
  }
  load_wait<(ST - 2) * LOADS + PER>();
#pragma unroll
  for (int f = 0; f < FM + FN; ++f) frag(0, lds0, 0, f);
  unsigned base = lds0;
  unsigned char* const ep0 = smem + ST * STAGE + wave * 32 * WTM * 2;  // the wave's way out
  const unsigned ep = lds0 + ST * STAGE + wave * 32 * WTM * 2;
  const float al = KIND != XG_LOGITS && !OUTF && p.alpha ? p.alpha[0] : 1.f;

  for (int w = blockIdx.x; w < ntiles; w += gridDim.x) {
    int ti, tj, split;
    where(w, ti, tj, split);
    int nk = max((min(K - split * p.kchunk, p.kchunk) + BK - 1) / BK, 1);  // (of no rows at all: zeros)
    asm("" : "+s"(nk));  // known to be at least 1, the loop's registers spill
    const int mw = ti * BM + wm * WTM, nw = tj * BN + wn * WTN;  // this wave's block
    if constexpr (KIND == XG_LOGITS) {  // r and target of the wave's rows, into its way out, for when the products are done
      i32x4_t rs = rsrc_words(p.ref, 4ll * N), ts = rsrc_words(p.target, 4ll * N);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_nop 4" : "+s"(rs), "+s"(ts)::"memory");
#pragma unroll
      for (int i = 0; i < WTN; i += 64) {
        load_lds4(rs, (nw + i + lane) * 4, ep + i * 4);
        load_lds4(ts, (nw + i + lane) * 4, ep + (WTN + i) * 4);
      }
    }
    f32x16_t acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

    static_assert(KS % 2 == 0, "fragment sets alternate over whole tiles");
    // One k step: its MFMAs, and between them, in an order that the compiler keeps, the reads of the next step's fragments
    // (early, so that they are there when the step ends) and a share of the loads. The last step of a k tile waits for the
    // next one before, and begins the loads of the tile that takes this one's stage; the next tile's first steps issue the
    // rest, all before its last but one. (The loads one after the other kept the MFMAs waiting for half of the time.)
    constexpr int EARLY = MM * 3 / 4;  // MFMAs over which the reads are spread
    for (int kt = 0; kt < nk; ++kt) {
      const unsigned next = base + STAGE == lds0 + ST * STAGE ? lds0 : base + STAGE;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int cur = ks & 1;
        const bool last = ks + 1 == KS;
        if (last) load_wait<(ST - 2) * LOADS>();
#pragma unroll
        for (int g = 0; g < MM; ++g) {
          const int i = g / FN, j = g % FN;
          acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[cur][i], fb[cur][j], acc[i][j], 0, 0, 0);
#pragma unroll
          for (int f = 0; f < FR; ++f)
            if (f * EARLY / FR == g) frag(cur ^ 1, last ? next : base, last ? 0 : ks + 1, f);
#pragma unroll
          for (int l = 0; l < PER; ++l) {
            const int n = (last ? 0 : ks + 1) * PER + l;
            if (l * MM / PER == g && n < LOADS) load(n);
          }
          if (ks + 2 == KS && g == MM - 2) plan(false);  // for the loads that begin with the last step
          if (g < MM - 2) __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      base = next;
    }

    // Element e of acc[i][j]: m = 32 i + 8 (e / 4) + 4 hh + e % 4, n = 32 j + c of the wave's block: 4 consecutive m a
    // lane. 32 n at a time are put together in the wave's own part of LDS (rows n of WTM 16-bit values, 16-byte chunks
    // XORed by n) and leave in rows of 16-byte stores.
    if constexpr (OUTF) {
      float* const o = p.outf + (long long)split * p.N * p.ldo;
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        const int n = nw + 32 * j + c;
        if (n >= N) continue;
        float* const q = o + (long long)n * p.ldo + mw + 4 * hh;
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int m = 32 * i + 8 * g;
            if (mw + 4 * hh + m >= p.M) continue;
            f32x4_t x = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            if (p.accumulate) x += *reinterpret_cast<const f32x4_t*>(q + m);
            *reinterpret_cast<f32x4_t*>(q + m) = x;
          }
      }
      continue;
    }
    float ref[FN];
    int tgt[FN];
    if constexpr (KIND == XG_LOGITS) {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        ref[j] = *(LDS_AS lds_float*)(uintptr_t)(ep + (32 * j + c) * 4);
        tgt[j] = *(LDS_AS lds_int*)(uintptr_t)(ep + (WTN + 32 * j + c) * 4);
      }
    }
    constexpr int CH = WTM / 8;
    auto slot = [&](int n, int ch) __attribute__((always_inline)) { return ep0 + n * WTM * 2 + ((ch ^ (n & (CH - 1))) << 4); };
    int to_lo = 0, to_hi = 0;  // where rows nw + lane and nw + 64 + lane go
    if constexpr (KIND == XG_DX) {
      static_assert(WTN == 128, "two rows a lane");
      to_lo = nw + lane;
      to_hi = nw + 64 + lane;
      if (p.order) {
        to_lo = p.order[min(to_lo, N - 1)];
        to_hi = p.order[min(to_hi, N - 1)];
      }
    }
    uint16_t* const out = KIND == XG_LOGITS ? reinterpret_cast<uint16_t*>(p.q) : p.out;
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int n = nw + 32 * j + c;
      const bool row = n < N;
      if constexpr (KIND == XG_LOGITS) {
        const float r = ref[j];
        const int t = tgt[j];
        const int tl = t - mw - 4 * hh;  // the target as a column of this lane's first group
        const bool inside = mw + WTM <= p.M && !__any(tl >= -4 && tl < WTM + 4);
        constexpr float L2E = 1.4426950408889634f;
        // pknorm: x 32767 to the nearest, clamped; x = ((z - r) - low - 64) / (64 32767 / 32768)
        constexpr float QS = 32768.f / 32767.f / 64.f;
        const float e0 = -r * L2E, q0 = (-r - kLogitLow - 64.f) * QS;
        float s = 0.f, top = -INFINITY;
        auto code = [&](int i, int g, const float* z) __attribute__((always_inline)) {
          const auto lo = __builtin_amdgcn_cvt_pknorm_i16(__builtin_fmaf(z[0], QS, q0), __builtin_fmaf(z[1], QS, q0));
          const auto hi = __builtin_amdgcn_cvt_pknorm_i16(__builtin_fmaf(z[2], QS, q0), __builtin_fmaf(z[3], QS, q0));
          uint2 x;
          __builtin_memcpy(&x.x, &lo, 4);
          __builtin_memcpy(&x.y, &hi, 4);
          *reinterpret_cast<uint2*>(slot(c, 4 * i + g) + hh * 8) = x;
        };
        auto usual = [&](auto keep) __attribute__((always_inline)) {  // no branches between the 64 exponentials
          float s1 = 0.f, s2 = 0.f, s3 = 0.f;
#pragma unroll
          for (int i = 0; i < FM; ++i) {
            asm volatile("" : "+a"(acc[i][j]));  // accumulators leave their registers tile by tile, not all at once
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float z[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
              s += __builtin_amdgcn_exp2f(__builtin_fmaf(z[0], L2E, e0));
              s1 += __builtin_amdgcn_exp2f(__builtin_fmaf(z[1], L2E, e0));
              s2 += __builtin_amdgcn_exp2f(__builtin_fmaf(z[2], L2E, e0));
              s3 += __builtin_amdgcn_exp2f(__builtin_fmaf(z[3], L2E, e0));
              if constexpr (decltype(keep)::value) code(i, g, z);
            }
          }
          s = (s + s1) + (s2 + s3);
        };
        const bool max_only = REDO && p.max_only;
        if (inside && !max_only) {
          if (p.q) usual(std::true_type{});
          else usual(std::false_type{});
        } else {
#pragma unroll
          for (int i = 0; i < FM; ++i) {
            asm volatile("" : "+a"(acc[i][j]));
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              const float z[4] = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
              const int m = mw + 32 * i + 8 * g + 4 * hh;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if (max_only) top = fmaxf(top, m + e < p.M ? z[e] : -INFINITY);
                else s += m + e < p.M && m + e != t ? __builtin_amdgcn_exp2f(__builtin_fmaf(z[e], L2E, e0)) : 0.f;
              }
              if (p.q) code(i, g, z);
            }
          }
        }
        if (max_only) {
          top = fmaxf(top, __shfl_xor(top, 32, 64));
          if (row && hh == 0) p.tops[(long long)n * 2 * p.tiles_m + 2 * ti + wm] = top;
        } else {
          s += __shfl_xor(s, 32, 64);
          if (row && hh == 0) p.sums[(long long)n * 2 * p.tiles_m + 2 * ti + wm] = s;
        }
        if (!p.q) continue;
      } else {
#pragma unroll
        for (int i = 0; i < FM; ++i) {
          asm volatile("" : "+a"(acc[i][j]));  // accumulators leave their registers tile by tile, not all at once
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<uint2*>(slot(c, 4 * i + g) + hh * 8) =
                make_uint2(pack2_bf16(al * acc[i][j][4 * g], al * acc[i][j][4 * g + 1]),
                           pack2_bf16(al * acc[i][j][4 * g + 2], al * acc[i][j][4 * g + 3]));
        }
      }
#pragma unroll
      for (int it = 0; it < 32 * CH / 64; ++it) {
        const int idx = it * 64 + lane, q = idx / CH, ch = idx % CH, m = mw + 8 * ch, no = nw + 32 * j + q;
        const uint4 x = *reinterpret_cast<const uint4*>(slot(q, ch));
        const int to = KIND == XG_DX ? __shfl(j < 2 ? to_lo : to_hi, (32 * j + q) & 63, 64) : no;
        if (no >= N || m >= p.M) continue;
        uint16_t* o = out + (long long)to * p.ldo + m;
        if (m + 8 <= p.M) {
          __builtin_memcpy(o, &x, 16);
        } else {
          uint16_t h[8];
          __builtin_memcpy(h, &x, 16);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (m + e < p.M) o[e] = h[e];
        }
      }
    }
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load may reach LDS after the workgroup
}

template <int WTM, int WTN, int BK, int ST, bool MCA, bool MCB, int KIND, bool OUTF = false, bool REDO = false>
static hipError_t launch_x(XgArgs& a, hipStream_t st) {
  constexpr int smem = ST * (Tile<2 * WTM, BK, MCA>::BYTES + Tile<2 * WTN, BK, MCB>::BYTES) + 4 * 32 * WTM * 2;
  void (*fn)(XgArgs) = xgemm_kernel<WTM, WTN, BK, ST, MCA, MCB, KIND, OUTF, REDO>;
  static const hipError_t attr =
      hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (attr != hipSuccess) return attr;
  a.tiles_m = (a.M + 2 * WTM - 1) / (2 * WTM);
  a.tiles_n = (a.N + 2 * WTN - 1) / (2 * WTN);
  if (!a.kreal) a.kreal = a.K;
  if (a.splits == 1) a.kchunk = a.K;
  const long long tiles = (long long)a.tiles_m * a.tiles_n * a.splits;
  hipLaunchKernelGGL(fn, dim3((unsigned)(tiles > 256 ? 256 : tiles)), dim3(256), smem, st, a);  // one a CU
  return hipGetLastError();
}

// The time of whole rounds of one workgroup a CU: a CU multiplies a 256 x 256 tile at 5.3 TFLOP/s (4096 x 4096 x 131072:
// 1360 TFLOP/s) and a 128 x 256 one, whose fragments are read 1.5 times as often, at 4.2 (1080). Small tiles win where
// large ones fill half a round or pad m: 1531 x 770 x 50021 dw 188 -> 160 us, dx 164 -> 154. A further part of k costs
// fp32 sums written and read.
XgPlan xgemm_plan(long long M, long long N, long long K, bool can_split) {
  XgPlan best{256, 1, (int)K};
  double least = 1e30;
  for (int bm : {256, 128}) {
    const double tiles = (double)((M + bm - 1) / bm) * (double)((N + 255) / 256);
    const double tile = 2. * bm * 256 / (bm == 256 ? 5.3e12 : 4.2e12);  // a k
    for (int s = 1; s <= (can_split ? 32 : 1) && (s == 1 || K / s >= 512); ++s) {
      const double rounds = std::ceil(tiles * s / 256), t = rounds * tile * (double)((K + s - 1) / s) +
                            (s > 1 ? 8. * s * (double)M * (double)N / 5e12 + 3e-6 : 0.);
      if (t < least) {
        least = t;
        const long long chunk = ((K + s - 1) / s + 63) / 64 * 64;  // whole k tiles: the last part may not be there
        best = XgPlan{bm, (int)((K + chunk - 1) / chunk), s == 1 ? (int)K : (int)chunk};
      }
    }
  }
  return best;
}

hipError_t xgemm_launch(XgArgs& a, int kind, int bm, hipStream_t st) {
  if (kind == XG_LOGITS)
    return a.redo ? launch_x<128, 128, 64, 2, false, false, XG_LOGITS, false, true>(a, st)
                  : launch_x<128, 128, 64, 2, false, false, XG_LOGITS>(a, st);
  if (kind == XG_Z)
    return bm == 128 ? launch_x<64, 128, 64, 3, false, false, XG_Z, true>(a, st)
                     : launch_x<128, 128, 64, 2, false, false, XG_Z, true>(a, st);
  if (kind == XG_DX) {
    if (bm == 128)
      return a.outf ? launch_x<64, 128, 64, 3, true, false, XG_DX, true>(a, st)
                    : launch_x<64, 128, 64, 3, true, false, XG_DX>(a, st);
    return a.outf ? launch_x<128, 128, 64, 2, true, false, XG_DX, true>(a, st)
                  : launch_x<128, 128, 64, 2, true, false, XG_DX>(a, st);
  }
  if (bm == 128)
    return a.outf ? launch_x<64, 128, 64, 3, true, true, XG_DW, true>(a, st)
                  : launch_x<64, 128, 64, 3, true, true, XG_DW>(a, st);
  return a.outf ? launch_x<128, 128, 64, 2, true, true, XG_DW, true>(a, st)
                : launch_x<128, 128, 64, 2, true, true, XG_DW>(a, st);
}

}  // namespace psgdk
