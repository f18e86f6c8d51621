// e4m3 projection of many rows: out[m][n] = X W^T over blocks of 128 columns,
// each with its own scales (the definition is in starkv.h).
//
// A workgroup computes a tile of the output, k block by k block: the block's
// rows of 128 bytes go to LDS by direct loads (16 bytes a lane), NST stages
// ahead of the matrix instructions.  Instructions are 32 x 32 x 64, so a block
// is two halves:
//   * power-of-two scales ride in the instruction itself (its operands carry
//     an exponent byte each), so the accumulators take the sums directly;
//   * with fp32 scales both halves' sums p are formed first, acc += p (sx sw).
// The weight rows are the instruction's A operand and the activations its B
// operand: a lane then holds four consecutive columns of one output row, and
// one activation scale.
//
// LDS rows are 128 bytes; 16-byte piece c of row r lies at piece
// c ^ swz(r), swz(r) = (r & 7) ^ ((r >> 3) & 1): the 16 rows that one operand
// read touches at the same piece fall on distinct banks, taken 8 or 16 lanes
// at a time.
//
// The loop overlaps its three resources: half 0's products run while half 1's
// operands are read; then, behind the block's one barrier, half 1's products
// run while the next block's half 0 is read and another block is loaded into
// the stage just consumed.  (One after the other - load, read, multiply -
// each 128 x 128 block took 1850 cycles, the sum of the three, where the
// products take 512.)
#include <algorithm>
#include <type_traits>

#include "fp8.hpp"

namespace starkv {

namespace {
typedef __attribute__((address_space(3))) void lds_void;
__device__ inline int swz(int r) { return (r & 7) ^ ((r >> 3) & 1); }

// 1 KB to LDS byte address `lds` (16 bytes a lane) from base + the lane's
// offset.  In inline assembly, so that the compiler, which then does not see
// it write LDS, adds no wait of its own before reads of the other stage: one
// loop body serves both stages.  Volatile statements keep their order, so the
// loads stay between the barriers; nothing else in these kernels uses m0.  A
// wait state separates the scalar write of m0 from the load that takes it.
__device__ inline void dma_1k(const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "m0");
}

// one dword a lane from its own address to LDS byte address `lds` + 4 * lane
__device__ inline void dma_dword(const void* src, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "s"(lds) : "m0");
}
// The same where go is not 0: the branch stands inside the statement, so that a loop stays one block of code, within
// which the compiler keeps the order given (it moved products over a branch of its own, away from the reads that
// they are to cover).
__device__ inline void dma_1k_if(int go, const uint8_t* base, uint32_t off, uint32_t lds) {
  asm volatile("s_cmp_eq_u32 %3, 0\n\ts_cbranch_scc1 1f\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1\n1:"
               ::"v"(off), "s"(base), "s"(lds), "s"(go) : "m0", "scc");
}
__device__ inline void dma_dword_if(int go, const void* src, uint32_t lds) {
  asm volatile("s_cmp_eq_u32 %2, 0\n\ts_cbranch_scc1 1f\n\ts_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off\n1:"
               ::"v"(src), "s"(lds), "s"(go) : "m0", "scc");
}
// Wait for LDS reads, and until at most LOADS loads are on their way (go not 0) or none.
template <int LOADS> __device__ inline void wait_one_stage(int go) {
  asm volatile("s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 1f\n\ts_waitcnt vmcnt(0)\n1:\ts_waitcnt vmcnt(%1) lgkmcnt(0)"
               ::"s"(go), "n"(LOADS) : "scc", "memory");
}
// the aligned dword with the byte at base + the lane's offset
__device__ inline void dma_dword_at(const uint8_t* base, uint32_t off, uint32_t lds) {
  const uint32_t low = (uint32_t)(uintptr_t)base & 3;
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"((off + low) & ~3u), "s"(base - low), "s"(lds) : "m0");
}
// s_waitcnt vmcnt(v) lgkmcnt(l)
__device__ constexpr int vm_lgkm(int v, int l) { return 0x0070 | (v & 15) | ((v >> 4) << 14) | l << 8; }
__device__ constexpr int vm_lgkm0(int v) { return vm_lgkm(v, 0); }
// Tile number -> (tm, tn): down eight row tiles before the next column, so that an XCD's L2 serves most reads of a
// contiguous run of tiles.
__device__ inline void tile_at(const Fp8GemmArgs& a, int tl, int& tm, int& tn) {
  constexpr int GROUP = 8;
  const int grp = tl / (GROUP * a.tiles_n), rem = tl - grp * GROUP * a.tiles_n;
  const int gm = min(GROUP, a.tiles_m - grp * GROUP);
  tm = grp * GROUP + rem % gm;
  tn = rem / gm;
}
}  // namespace

// Zero the bytes past column k of a stage that holds the row's last, short
// block (nv < 128 columns): they are any value, also NaN.
template <int ROWS, int THREADS> __device__ inline void zero_tail(uint8_t* st, int nv, int tid) {
  const int p0 = nv >> 4, np = 8 - p0;             // pieces from the first short one on
  for (int i = tid; i < ROWS * np; i += THREADS) {
    const int r = i / np, p = p0 + i - r * np;
    uint4* q = (uint4*)(st + r * 128 + ((p ^ swz(r & 15)) << 4));
    *q = keep_bytes(*q, nv - 16 * p);
  }
}

__device__ inline floatx16 mfma8_32(intx8 a, intx8 b, floatx16 c, int scale_a, int scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, scale_a, 0, scale_b);
}

// The results of 32 rows and 32 G columns from (row0, col0) on: lane (c, g) holds columns 32 j + 8 q + 4 g .. + 3 of row
// c in v[j] (SILU: gate columns, then the same up columns).  They are finished and rounded there and go through the
// wave's own part of LDS, so that whole rows of 64 bytes and more leave (8 bytes of each of 32 rows at a time, as the
// accumulators hold them, 128 x 128 tiles spent 8 us of a round on it); a residual comes the same way.  16-byte
// piece p of row r lies at p ^ r (of the row's pieces).  quick: all columns are inside the row; whole: the rows, too.
template <typename O, int G, bool SILU, bool NONTEMPORAL>
__device__ inline void finish_chunk(const Fp8GemmArgs& a, uint8_t* ob, int row0, int col0, const floatx16 (&v)[SILU ? 2 * G : G],
                                    float r, bool quick, bool whole) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  typedef u32x4 __attribute__((aligned(2))) u32x4_any;
  constexpr int RB = 32 * G * sizeof(O), PP = RB / 16, PC = 16 / sizeof(O);     // bytes and pieces of a row, columns of a piece
  constexpr int RPI = 64 / PP, NR = 32 / RPI;      // rows at a time
  const int lane = threadIdx.x & 63, g = lane >> 5;
  int c = lane & 31;
  asm volatile("" : "+v"(c));                      // addresses are formed here, not kept over a tile
  const int ncol = SILU ? a.half : a.n, lr0 = lane / PP, rc = lane % PP, col = col0 + PC * rc;
  auto slot = [&](int row, int p) __attribute__((always_inline)) { return ob + row * RB + ((p ^ (row & (PP - 1))) << 4); };
  if (!SILU && a.res) {
    if (quick) {
      u32x4 t[NR];
#pragma unroll
      for (int i = 0; i < NR; ++i)
        t[i] = *(const u32x4_any*)((const O*)a.res + (int64_t)min(row0 + lr0 + RPI * i, a.m - 1) * a.rs + col);
#pragma unroll
      for (int i = 0; i < NR; ++i) *(u32x4*)slot(lr0 + RPI * i, rc) = t[i];
    } else {
#pragma unroll 1
      for (int lr = lr0; lr < 32; lr += RPI) {
        O e[PC];
#pragma unroll
        for (int i = 0; i < PC; ++i)
          e[i] = row0 + lr < a.m && col + i < ncol ? ((const O*)a.res)[(int64_t)(row0 + lr) * a.rs + col + i] : (O)0.f;
        u32x4 u;
        __builtin_memcpy(&u, e, 16);
        *(u32x4*)slot(lr, rc) = u;
      }
    }
  }
  asm volatile("" ::: "memory");                   // other lanes read what this one wrote
#pragma unroll
  for (int j = 0; j < G; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint8_t* const p = sizeof(O) == 2 ? slot(c, 4 * j + q) + 8 * g : slot(c, 8 * j + 2 * q + g);
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        f[e] = SILU ? silu_mul_f32(r * v[j][4 * q + e], r * v[SILU ? j + G : j][4 * q + e]) : r * v[j][4 * q + e];
      O w[4];
      if (!SILU && a.res) {
        __builtin_memcpy(w, __builtin_assume_aligned(p, 4 * sizeof(O)), sizeof(w));
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] += (float)w[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] = (O)f[e];
      __builtin_memcpy(__builtin_assume_aligned(p, 4 * sizeof(O)), w, sizeof(w));
    }
  asm volatile("" ::: "memory");
  if (quick) {
    u32x4 o[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) o[i] = *(const u32x4*)slot(lr0 + RPI * i, rc);
    O* const out = (O*)a.out + (int64_t)(row0 + lr0) * a.os + col;
#pragma unroll
    for (int i = 0; i < NR; ++i)
      if (whole || row0 + lr0 + RPI * i < a.m) {
        u32x4_any* const to = (u32x4_any*)(out + (int64_t)(RPI * i) * a.os);
        if (NONTEMPORAL) __builtin_nontemporal_store(o[i], to);
        else *to = o[i];
      }
  } else {
#pragma unroll 1
    for (int lr = lr0; lr < 32; lr += RPI) {
      const u32x4 u = *(const u32x4*)slot(lr, rc);
      O e[PC];
      __builtin_memcpy(e, &u, 16);
#pragma unroll
      for (int i = 0; i < PC; ++i)
        if (row0 + lr < a.m && col + i < ncol) ((O*)a.out)[(int64_t)(row0 + lr) * a.os + col + i] = e[i];
    }
  }
  asm volatile("" ::: "memory");
}

// WM x WN waves of 32 I x 32 J, NST stages; KS such groups of waves take every KS-th block, each with stages of its
// own, and meet in LDS at the end; SILU: a wave's columns are half gate columns and half the same up columns
template <int WM, int WN, int I, int J, int KS, int NST, typename S, typename O, bool SILU>
__global__ __launch_bounds__(64 * WM * WN * KS, (WM * WN * KS + 3) / 4 * (KS * NST * (WM * I + WN * J) * 4096 <= 78000 ? 2 : 1))
void fp8_gemm_kernel(const Fp8GemmArgs a) {
  constexpr int NW = WM * WN, TM = 32 * I, TN = 32 * J, BM = WM * TM, BN = WN * TN;
  constexpr int LOADS = (BM + BN) / 8 / NW;         // 1 KB loads per wave and stage
  static_assert(LOADS * 8 * NW == BM + BN, "whole loads");
  static_assert(!SILU || J % 2 == 0, "gate and up halves");
  constexpr bool EXACT = __is_same(O, float);      // 16-bit instructions (see half_of)
  constexpr bool PART = EXACT || !S::pow2;         // a block's sums are scaled afterwards
  // a stage: rows, then a dword with the scale of each activation row and of two weight blocks
  constexpr int SLOTS = (BM + 2 + 63) / 64 * 64, ROWS = (BM + BN) * 128, STAGE = ROWS + SLOTS * 4;
  constexpr int SLW = SLOTS / 64, SL = (SLW + NW - 1) / NW, LW = LOADS + SL;       // loads that fill those slots, a wave's of them
  static_assert(NST == 2 || (NST == 3 && LW < 32), "waits");
  __shared__ __attribute__((aligned(16))) uint8_t lds_all[KS * NST * STAGE];
  static_assert((KS - 1) * NW * I * J * 4096 <= KS * NST * STAGE, "the groups' sums fit");

  const int lane = threadIdx.x & 63;
  const int kg = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / NW;     // group of waves
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) - kg * NW;
  const int wm = wave % WM, wn = wave / WM;
  const int c = lane & 31, g = lane >> 5;
  uint8_t* const lds = lds_all + kg * NST * STAGE;

  // workgroup i runs on XCD i % 8; each XCD takes a contiguous run of tiles
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (idx >= total) return;
  int tm, tn;
  tile_at(a, idx, tm, tn);
  const int m0 = tm * BM, n0 = tn * (SILU ? BN / 2 : BN);

  // weight row of tile row j (wave-contiguous: wave wn owns rows wn TN ..; with SILU
  // its first half are gate rows, its second half the up rows of the same columns)
  auto wrow_of = [&](int j) {
    if constexpr (SILU) {
      const int q = j / TN, r = j % TN;
      return (r < TN / 2 ? 0 : a.half - TN / 2) + n0 + q * (TN / 2) + r;
    }
    return n0 + j;
  };

  // this lane's source of each of the wave's loads (8 rows x 8 pieces), from the tile's first row
  const int rs = lane >> 3, q8 = lane & 7;
  const uint8_t* const xbase = (const uint8_t*)a.x + (int64_t)m0 * a.xs;
  const uint8_t* const wbase = a.w + (int64_t)n0 * a.ws;
  uint32_t off[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (wave * LOADS + i) * 8 + rs;
    const int64_t r = row < BM ? min(m0 + row, a.m - 1) - m0 : min(wrow_of(row - BM), a.n - 1) - n0;
    off[i] = (uint32_t)(r * (row < BM ? a.xs : a.ws));
  }
  // Scales go the same way, a dword a lane: this wave's loads take 64 slots each, which hold the scale of activation
  // row slot, then of the tile's two weight blocks (the gate and the up rows', or 128 rows each).
  // (Power-of-two scales are bytes: the aligned dword that holds it is loaded, and the byte taken from it at the end.)
  typedef typename S::T ST;
  auto wblock = [&](int u) { return min(SILU ? n0 + u * a.half : n0 + u * FP8_BLOCK, a.n - 1) >> 7; };
  const ST* sptr[SL];
  int64_t sstep[SL];
  int slot0[SL];
#pragma unroll
  for (int u = 0; u < SL; ++u) {
    slot0[u] = (wave + u * NW) % SLW * 64;
    const int slot = slot0[u] + lane;
    const bool xslot = slot < BM;
    sptr[u] = xslot ? (const ST*)a.sx + (int64_t)min(m0 + slot, a.m - 1) * a.sxr
                    : (const ST*)a.sw + (int64_t)wblock(slot == BM + 1) * a.swr;
    sstep[u] = xslot ? a.sxb : a.swb;
  }
  const int last = (a.k - 1) >> 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds_all + kg * NST * STAGE;
  // load number i < LW of a stage for block kb, where go is not 0
  auto issue1 = [&](int stage, int kb, int i, int go) __attribute__((always_inline)) {
    if (i < LOADS) {
      const int row = (wave * LOADS + i) * 8;      // uniform; the lane's piece of its row is q8 ^ swz(row + rs)
      const int p = min(kb * 8 + (q8 ^ rs ^ ((row >> 3) & 1)), last);
      dma_1k_if(go, row < BM ? xbase : wbase, off[i] + (uint32_t)p * 16, lds0 + stage + row * 128);
    } else {
      const int u = i - LOADS;
      dma_dword_if(go, (const void*)((uintptr_t)(sptr[u] + kb * sstep[u]) & ~(uintptr_t)3), lds0 + stage + ROWS + slot0[u] * 4);
    }
  };
  // the scale in slot `s` of a stage, p its address: as the instruction takes it (its byte in a register) or in fp32
  auto scale_of = [&](const uint8_t* st, int s, const ST* p) __attribute__((always_inline)) {
    const uint32_t v = *(const uint32_t*)(st + ROWS + s * 4);
    if constexpr (S::pow2) return (int)(v >> (8 * ((uint32_t)(uintptr_t)p & 3)) & 0xffu);
    else return __uint_as_float(v);
  };
  typedef std::conditional_t<S::pow2, int, float> SR;
  struct Sc { SR x[I], w[SILU ? 2 : 1]; };
  const ST* sxp[I];
#pragma unroll
  for (int i = 0; i < I; ++i) sxp[i] = (const ST*)a.sx + (int64_t)min(m0 + wm * TM + 32 * i + c, a.m - 1) * a.sxr;
  auto scales = [&](Sc& sc, const uint8_t* st, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < I; ++i) sc.x[i] = scale_of(st, wm * TM + 32 * i + c, sxp[i] + kb * a.sxb);
#pragma unroll
    for (int u = 0; u < (SILU ? 2 : 1); ++u) {
      const int v = SILU ? u : wn * TN / FP8_BLOCK;
      sc.w[u] = scale_of(st, BM + v, (const ST*)a.sw + (int64_t)wblock(v) * a.swr + kb * a.swb);
    }
  };

  // operand reads: lane (c, g) takes pieces 4 h + 2 g and + 1 of row c
  const int f = (c & 7) ^ ((c >> 3) & 1);
  int rd[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int t = 0; t < 2; ++t) rd[h][t] = c * 128 + (((4 * h + 2 * g + t) ^ f) << 4);
  struct Half { intx8 x[I], w[J]; };
  auto get = [&](const uint8_t* st, int h, int row) __attribute__((always_inline)) {
    return frag8(*(const uint4*)(st + row * 128 + rd[h][0]), *(const uint4*)(st + row * 128 + rd[h][1]));
  };
  // operand e of a half: activations and weights in turn, as the products ask for them
  constexpr int NR = I + J, NP = I * J;
  auto read1 = [&](Half& o, const uint8_t* st, int h, int e) __attribute__((always_inline)) {
    constexpr int L = 2 * (I < J ? I : J);
    const bool isx = e < L ? (e & 1) == 0 : I > J;
    const int k = e < L ? e >> 1 : e - L / 2;
    if (isx) o.x[k] = get(st, h, wm * TM + 32 * k);
    else o.w[k] = get(st, h, BM + wn * TN + 32 * k);
  };

  floatx16 acc[J][I], part[PART ? J : 1][PART ? I : 1];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int i = 0; i < I; ++i) acc[j][i] = floatx16{};
  auto product = [&](const Half& o, const Sc& sc, auto h, int q) __attribute__((always_inline)) {
    constexpr bool FIRST = decltype(h)::value == 0;
    const int j = q % J, i = q / J;
    if constexpr (EXACT) {
      floatx16 p = FIRST ? floatx16{} : part[j][i];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        p = __builtin_amdgcn_mfma_f32_32x32x16_f16(half_of(o.w[j], u), half_of(o.x[i], u), p, 0, 0, 0);
      part[j][i] = p;
    } else if constexpr (PART) {
      part[j][i] = mfma8_32(o.w[j], o.x[i], FIRST ? floatx16{} : part[j][i], E8_ONE, E8_ONE);
    } else {
      acc[j][i] = mfma8_32(o.w[j], o.x[i], acc[j][i], sc.w[SILU ? 2 * j / J : 0], sc.x[i]);
    }
  };
  auto rescale = [&](const Sc& sc, int q) __attribute__((always_inline)) {
    if constexpr (PART) {
      const int j = q % J, i = q / J;
      const float s = scale_f32((ST)sc.x[i]) * scale_f32((ST)sc.w[SILU ? 2 * j / J : 0]);
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[j][i][e] = fmaf(part[j][i][e], s, acc[j][i][e]);
    }
  };

  // The blocks in the order last, first, second ..: the row's last one may be
  // short, and what lies behind it is zeroed before the loop starts.  Group kg
  // takes the blocks kg, kg + KS .. of that order, n of them.
  const int n = (a.kb - kg + KS - 1) / KS, most = (a.kb + KS - 1) / KS;
  auto block = [&](int t) { return t == 0 && kg == 0 ? a.kb - 1 : kg + KS * t - 1; };
#pragma unroll 1
  for (int t = 0; t < min(n, NST); ++t)
#pragma unroll
    for (int i = 0; i < LW; ++i) issue1(t * STAGE, block(t), i, 1);
  // the first stage landed
  if (n >= NST) __builtin_amdgcn_s_waitcnt(vm_lgkm0((NST - 1) * LW));
  else if (NST > 2 && n > 1) __builtin_amdgcn_s_waitcnt(vm_lgkm0(LW));
  else __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
  asm volatile("s_barrier" ::: "memory");
  if (a.k & (FP8_BLOCK - 1)) {
    if (kg == 0) zero_tail<BM + BN, 64 * NW>(lds, a.k & (FP8_BLOCK - 1), wave * 64 + lane);
    __builtin_amdgcn_s_waitcnt(0xC07F);            // LDS writes done; the loads in flight are not waited for
    asm volatile("s_barrier" ::: "memory");
  }
  const std::integral_constant<int, 0> first{};
  const std::integral_constant<int, 1> second{};
  Half h0, h1;
  Sc sc, sn;
#pragma unroll
  for (int e = 0; e < NR; ++e) read1(h0, lds, 0, e);
  scales(sc, lds, block(0));
  int cur = 0;
  for (int t = 0; t < n; ++t) {                    // block(t) in stage `cur`, its half 0 in h0, its scales in sc
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      product(h0, sc, first, q);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = q * NR / NP; e < (q + 1) * NR / NP; ++e) read1(h1, lds + cur, 1, e);
      __builtin_amdgcn_sched_barrier(0);
    }
    // half 1 read; this wave's part of the next stage landed (with three stages, that of one more may be on its way)
    if constexpr (NST == 2) __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
    else wait_one_stage<LW>(max(0, n - 2 - t));
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    const int nxt = cur == (NST - 1) * STAGE ? 0 : cur + STAGE;
    // (behind the last block: reads of what is there, for nobody)
    scales(sn, lds + nxt, block(t + 1));
    const int more = max(0, n - NST - t), kn = block(t + NST);
#pragma unroll
    for (int q = 0; q < NP; ++q) {
      product(h1, sc, second, q);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = q * LW / NP; i < (q + 1) * LW / NP; ++i) issue1(cur, kn, i, more);
#pragma unroll
      for (int e = q * NR / NP; e < (q + 1) * NR / NP; ++e) read1(h0, lds + nxt, 0, e);
      if (q) rescale(sc, q - 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    rescale(sc, NP - 1);
    sc = sn;
    cur = nxt;
  }
  if constexpr (KS > 1) {
    if (n < most) asm volatile("s_barrier" ::: "memory");      // as many as the other groups' loops
    // the groups' sums, in group order
    __syncthreads();
    floatx4* const red = (floatx4*)lds_all;        // [group - 1][wave][j][i][q][lane]
    if (kg > 0) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            red[(((((kg - 1) * NW + wave) * J + j) * I + i) * 4 + q) * 64 + lane] =
                floatx4{acc[j][i][4 * q], acc[j][i][4 * q + 1], acc[j][i][4 * q + 2], acc[j][i][4 * q + 3]};
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int v = 0; v < KS - 1; ++v)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < I; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const floatx4 t = red[((((v * NW + wave) * J + j) * I + i) * 4 + q) * 64 + lane];
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][i][4 * q + e] += t[e];
          }
  }

  // results by way of LDS, behind what the groups' sums take
  constexpr int G = SILU ? J / 2 : J, OB = 32 * 32 * G * sizeof(O), SUMS = (KS - 1) * NW * I * J * 4096;
  static_assert(SUMS + NW * OB <= KS * NST * STAGE, "the results fit");
  if constexpr (KS == 1) __syncthreads();          // the other waves' operands
  const int col0 = n0 + wn * 32 * G;
  const bool quick = col0 + 32 * G <= (SILU ? a.half : a.n);
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int row0 = m0 + wm * TM + 32 * i;
    floatx16 v[J];
#pragma unroll
    for (int j = 0; j < J; ++j) v[j] = acc[j][i];
    finish_chunk<O, G, SILU, false>(a, lds_all + SUMS + wave * OB, row0, col0, v,
                                    a.rscale ? a.rscale[min(row0 + c, a.m - 1)] : 1.f, quick, row0 + 32 <= a.m);
  }
}

// ---------------------------------------------------------------------------
// Power-of-two scales, 256 x 256 tiles: four waves of 128 x 128 (one per SIMD,
// 256 accumulators each), 32 x 32 x 64 instructions.  The matrix cores need
// 2048 cycles for a block; the operands of four 128 x 128 wave tiles take
// 128 KB of LDS reads and 64 KB of writes per block, 1536 cycles at 128
// bytes, where eight waves of 64 x 128 would take all of the 2048.
//
// A block is two halves of 64 columns, each with operand registers of its own,
// 16 products to a half:
//   * half 0's products run while half 1's operands are read, those of the
//     first two row groups first;
//   * behind product 12 these have been read: all waves meet, and the first
//     half of the stage's rows is loaded anew, for the block after next;
//   * behind product 20 (the fourth of half 1) the rest has been read: they
//     meet again, and the other half is loaded;
//   * half 1's products run while the next block's half 0 is read.
// At each meeting a wave waits for the loads it issued 24 products ago, not for
// the last ones, and for all but its last four reads: nothing is waited for
// with the matrix cores idle unless memory is late.  (One meeting, after half
// 0: loads in a burst of 16 products, 16 products to land: 2 % slower.)
// Measured: 1.4 us a block on all CUs, where products alone take 1.0; without
// the loads 1.2, without the reads 1.24.  8192 x 22016 x 4096 with SiLU: 565 to
// 600 us by the card, 2610 to 2460 TFLOP/s.
//
// A workgroup takes tile after tile: the next tile's first two blocks load
// while this one's results are stored, and the stores drain behind the next
// tile's first block.
// ---------------------------------------------------------------------------
constexpr int WT = 256;                            // tile rows and columns
constexpr int WSTAGE = 2 * WT * 128;               // bytes of a stage
constexpr int WSC = 256 * 4 + 4 * 64 * 4;           // bytes of a stage's scales: the activation rows' and, per wave, the weights'
constexpr int WOUT = 32 * 64 * 2;                  // bytes a wave stages of its results: 32 rows x 64 columns
constexpr int WLOADS = 18;                         // a wave's loads of a block: 16 of rows, two of scales

template <typename O, bool SILU>
__global__ __launch_bounds__(256, 1) void fp8_gemm_wide_kernel(const Fp8GemmArgs a) {
  static_assert(sizeof(O) == 2, "16-bit outputs");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * WSTAGE + 2 * WSC + 2 * WT * 4 + 4 * WOUT];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave & 1, wn = wave >> 1;
  const int c = lane & 31, g = lane >> 5;
  const int end = a.kb - 1;

  // Loads: 512 rows of 128 bytes, X then W; this wave takes rows 128 wave .. (X: waves 0, 1), eight rows and
  // their eight pieces at a time.  Offsets from the tile's first row fit 32 bits.
  const int rs = lane >> 3, q8 = lane & 7;
  const bool isx = wave < 2;
  const int last = (a.k - 1) >> 4;
  const int piece0 = q8 ^ rs;                      // piece of row r at slot q8: q8 ^ swz(r), swz(8 i + rs) = rs ^ (i & 1)
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds + wave * 16 * 1024;

  // the tile in hand
  int m0, n0;
  const uint8_t* base;
  uint32_t off[16];                                // of the wave's loads' lane: row and piece
  const uint32_t po[2] = {(uint32_t)min(piece0, last) * 16, (uint32_t)min(piece0 ^ 1, last) * 16};
  const uint8_t *sxp, *swp;                        // scales of block 0: the tile's first activation row's and weight rows'
  uint32_t sxo, swo;                               // from there: of the scales this lane loads
  uint32_t xlow[4], wlow[2];                       // low address bits of the scales this lane reads
  // W rows of the tile: with SILU, wave column wn owns 64 gate rows and the same 64 up rows
  auto wrow = [&](int j) {
    if constexpr (SILU) return ((j & 64) ? a.half : 0) + n0 + (j >> 7) * 64 + (j & 63);
    return n0 + j;
  };
  auto take = [&](int idx) __attribute__((always_inline)) {
    int tm, tn;
    tile_at(a, idx, tm, tn);
    m0 = tm * WT;
    n0 = tn * (SILU ? WT / 2 : WT);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = (wave & 1) * 128 + 8 * i + rs;
      const int64_t row = isx ? min(m0 + r, a.m - 1) - m0 : min(wrow(r), a.n - 1) - n0;
      off[i] = (uint32_t)(row * (isx ? a.xs : a.ws)) + po[i & 1];
    }
    base = isx ? (const uint8_t*)a.x + (int64_t)m0 * a.xs : a.w + (int64_t)n0 * a.ws;
    sxp = (const uint8_t*)a.sx + (int64_t)m0 * a.sxr;
    sxo = (uint32_t)((min(m0 + wave * 64 + lane, a.m - 1) - m0) * a.sxr);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      xlow[i] = (uint32_t)(uintptr_t)a.sx + (uint32_t)min(m0 + wm * 128 + 32 * i + c, a.m - 1) * (uint32_t)a.sxr;
    const auto wsc = [&](int t) { return (int64_t)(min(wrow(wn * 128 + 64 * t), a.n - 1) >> 7) * a.swr; };
    swp = (const uint8_t*)a.sw + wsc(0);
    swo = lane & 1 ? (uint32_t)(wsc(1) - wsc(0)) : 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) wlow[t] = (uint32_t)(uintptr_t)a.sw + (uint32_t)wsc(t);
  };
  // Scales go to LDS as the rows do (the aligned dword that holds the byte): loads into registers would bring the
  // compiler's waits, which know nothing of the loads in flight, into the loop.
  constexpr int SCALES = 2 * WSTAGE;
  auto issue_scales = [&](int stage, int kb) __attribute__((always_inline)) {    // stage: 0 or WSTAGE
    const uint32_t to = (uint32_t)(uintptr_t)(lds_void*)lds + SCALES + (stage ? WSC : 0);
    dma_dword_at(sxp + (int64_t)kb * a.sxb, sxo, to + wave * 256);
    dma_dword_at(swp + (int64_t)kb * a.swb, swo, to + 1024 + wave * 256);
  };
  struct Sc { uint32_t x[4], w[2]; };
  auto scales = [&](Sc& sc, int stage) __attribute__((always_inline)) {
    const uint8_t* const st = lds + SCALES + (stage ? WSC : 0);
#pragma unroll
    for (int i = 0; i < 4; ++i) sc.x[i] = *(const uint32_t*)(st + (wm * 128 + 32 * i + c) * 4);
#pragma unroll
    for (int t = 0; t < (SILU ? 2 : 1); ++t) sc.w[t] = *(const uint32_t*)(st + 1024 + wave * 256 + t * 4);
  };
  auto bytes_of = [&](Sc& sc, int kb) __attribute__((always_inline)) {           // the bytes in those dwords
#pragma unroll
    for (int i = 0; i < 4; ++i) sc.x[i] = __builtin_amdgcn_ubfe(sc.x[i], (xlow[i] + (uint32_t)kb * (uint32_t)a.sxb) << 3 & 24, 8);
#pragma unroll
    for (int t = 0; t < (SILU ? 2 : 1); ++t)
      sc.w[t] = __builtin_amdgcn_ubfe(sc.w[t], (wlow[t] + (uint32_t)kb * (uint32_t)a.swb) << 3 & 24, 8);
  };
  // The blocks in the order last, first, second .. (the last may be short:
  // what lies behind it is zeroed before the loop starts).  A full block's
  // pieces need no check against the row's end.
  auto block = [&](int t) { return t == 0 ? end : t > end ? 0 : t - 1; };
  auto issue1 = [&](int stage, int kb, int i) __attribute__((always_inline)) {
    dma_1k(base + (int64_t)kb * FP8_BLOCK, off[i], lds0 + stage + i * 1024);
  };
  auto issue_last = [&]() __attribute__((always_inline)) {
    const int left = last - end * 8;
    const uint32_t d[2] = {(uint32_t)min(piece0, left) * 16 - po[0], (uint32_t)min(piece0 ^ 1, left) * 16 - po[1]};
#pragma unroll
    for (int i = 0; i < 16; ++i) dma_1k(base + (int64_t)end * FP8_BLOCK, off[i] + d[i & 1], lds0 + i * 1024);
  };

  // operand reads: lane (c, g) takes pieces 4 h + 2 g and + 1 of row c
  const int f = (c & 7) ^ ((c >> 3) & 1);
  int rd[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int t = 0; t < 2; ++t) rd[h][t] = c * 128 + (((4 * h + 2 * g + t) ^ f) << 4);
  struct Half { uint4 x[4][2], w[4][2]; };
  // the q-th of the half's 16 reads: activations and weights of row group 0, then 1 ..
  auto read1 = [&](Half& o, const uint8_t* st, int h, int q) __attribute__((always_inline)) {
    const int i = q >> 2, t = q & 1;
    if (q & 2) o.w[i][t] = *(const uint4*)(st + (WT + wn * 128 + 32 * i) * 128 + rd[h][t]);
    else o.x[i][t] = *(const uint4*)(st + (wm * 128 + 32 * i) * 128 + rd[h][t]);
  };

  // tiles of this XCD (workgroup i runs on XCD i % 8), one after the other
  const int total = a.tiles_m * a.tiles_n, per = (total + 7) >> 3;
  const int first = (blockIdx.x & 7) * per, stop = min(total, first + per), stride = gridDim.x >> 3;
  int idx = first + (blockIdx.x >> 3);
  if (idx >= stop) return;
  take(idx);
  Sc sc, sn;
  // a tile's first two blocks
  constexpr int FACTORS = 2 * WSTAGE + 2 * WSC;    // row factors of this tile and the next
  int par = 0;
  auto start = [&](int to) __attribute__((always_inline)) {
    if (a.rscale)
      dma_dword(a.rscale + min(m0 + wave * 64 + lane, a.m - 1), (uint32_t)(uintptr_t)(lds_void*)lds + FACTORS + to * WT * 4 + wave * 256);
    issue_last();
    issue_scales(0, end);
#pragma unroll
    for (int i = 0; i < 8; ++i) issue1(WSTAGE, block(1), i);
    issue_scales(WSTAGE, block(1));
#pragma unroll
    for (int i = 8; i < 16; ++i) issue1(WSTAGE, block(1), i);
  };
  start(par);
  // vmcnt counts in order: behind the start's loads stand the stores of the last tile, NSTORE of them if it was
  // whole, which need not have ended for the loads to be there
  constexpr int NSTORE = SILU ? 16 : 32;
  bool drain = true;                               // another number of stores: wait for everything
  while (true) {
    floatx16 acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = floatx16{};
    if (drain) __builtin_amdgcn_s_waitcnt(vm_lgkm0(0));
    else __builtin_amdgcn_s_waitcnt(vm_lgkm0(WLOADS + NSTORE));
    asm volatile("s_barrier" ::: "memory");
    if (a.k & (FP8_BLOCK - 1)) {
      zero_tail<2 * WT, 256>(lds, a.k & (FP8_BLOCK - 1), threadIdx.x);
      __builtin_amdgcn_s_waitcnt(0xC07F);            // LDS writes done
      asm volatile("s_barrier" ::: "memory");
    }
    Half h0, h1;
#pragma unroll
    for (int q = 0; q < 16; ++q) read1(h0, lds, 0, q);
    scales(sc, 0);
    int cur = 0;
    auto product = [&](const Half& o, int q) __attribute__((always_inline)) {
      // row groups in the order in which the reads bring them
      constexpr int ORDER[16] = {0, 1, 4, 5, 2, 6, 8, 9, 10, 3, 7, 11, 12, 13, 14, 15};
      const int j = ORDER[q] >> 2, i = ORDER[q] & 3;
      acc[j][i] = mfma8_32(frag8(o.w[j][0], o.w[j][1]), frag8(o.x[i][0], o.x[i][1]), acc[j][i],
                           (int)sc.w[SILU ? j >> 1 : 0], (int)sc.x[i]);
    };
    // block(t) in stage `cur`, its half 0 in h0, its scales in sc
    auto step = [&](int t, auto firstc) __attribute__((always_inline)) {
      constexpr bool FIRST = decltype(firstc)::value;
      bytes_of(sc, block(t));
      const int kn = block(t + 2);
      // a wait that leaves v loads on their way (and the first block's: the last tile's stores), and four reads
      auto sync = [&](auto vc) __attribute__((always_inline)) {
        constexpr int V = decltype(vc)::value;
        if (FIRST && !drain) __builtin_amdgcn_s_waitcnt(vm_lgkm(V + NSTORE, 4));
        else __builtin_amdgcn_s_waitcnt(vm_lgkm(V, 4));
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
      };
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        product(h0, q);
        if (q == 12) issue_scales(cur, kn);
        if (q >= 12) issue1(cur, kn, q - 12);
        read1(h1, lds + cur, 1, q);
        __builtin_amdgcn_sched_barrier(0);
        if (q == 11) sync(std::integral_constant<int, 8>{});
      }
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        product(h1, q);
        if (q < 12) issue1(cur, kn, q + 4);
        read1(h0, lds + (cur ^ WSTAGE), 0, q);
        if (q == 8) scales(sn, cur ^ WSTAGE);
        __builtin_amdgcn_sched_barrier(0);
        if (q == 3) sync(std::integral_constant<int, 10>{});
      }
      sc = sn;
      cur ^= WSTAGE;
    };
    step(0, std::true_type{});
    for (int t = 1; t <= end; ++t) step(t, std::false_type{});
    // after the last blocks the loads repeated one and the reads took what was there, for nobody
    __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("s_barrier" ::: "memory");
    const int om = m0 + wm * 128, on = n0 + wn * (SILU ? 64 : 128);
    idx += stride;
    const bool more = idx < stop;
    if (more) {
      take(idx);
      start(par ^ 1);
    }

    // Results, 32 rows x 64 columns at a time.  One copy of the code serves all chunks: unrolled it came from memory
    // instruction by instruction (48 KB of code: 25 us a tile).  Stores are non-temporal: results of this many bytes
    // would push operands out of L2 (8192 x 8192, k 16384: 890 -> 785 us).
    uint8_t* const ob = lds + FACTORS + 2 * WT * 4 + wave * WOUT;
    const bool quick = on + (SILU ? 64 : 128) <= (SILU ? a.half : a.n), whole = quick && om + 128 <= a.m;
    drain = !whole;
#pragma unroll 1
    for (int ch = 0; ch < (SILU ? 4 : 8); ++ch) {
      const int row0 = om + 32 * (SILU ? ch : ch >> 1), col0 = on + (SILU ? 0 : 64 * (ch & 1));
      floatx16 v[SILU ? 4 : 2];
      auto pick = [&](auto chc) __attribute__((always_inline)) {
        constexpr int C = decltype(chc)::value;
#pragma unroll
        for (int j = 0; j < (SILU ? 4 : 2); ++j) v[j] = SILU ? acc[j][C & 3] : acc[2 * (C & 1) + j][C >> 1];
      };
      switch (ch) {
        case 0: pick(std::integral_constant<int, 0>{}); break;
        case 1: pick(std::integral_constant<int, 1>{}); break;
        case 2: pick(std::integral_constant<int, 2>{}); break;
        case 3: pick(std::integral_constant<int, 3>{}); break;
        case 4: pick(std::integral_constant<int, SILU ? 0 : 4>{}); break;
        case 5: pick(std::integral_constant<int, SILU ? 0 : 5>{}); break;
        case 6: pick(std::integral_constant<int, SILU ? 0 : 6>{}); break;
        default: pick(std::integral_constant<int, SILU ? 0 : 7>{}); break;
      }
      const float r = a.rscale ? *(const float*)(lds + FACTORS + par * WT * 4 + (row0 - om + wm * 128 + c) * 4) : 1.f;
      finish_chunk<O, 2, SILU, true>(a, ob, row0, col0, v, r, quick, whole);
    }
    par ^= 1;
    if (!more) break;
  }
}

// Which kernel and tile, by modelled time: for each round of resident
// workgroups a fixed part and a part for each k block (microseconds).  Tiles
// of 64 and 128 columns run with one workgroup on a CU or two, the larger ones
// alone, and their blocks go the faster the more CUs idle.  Fitted to the
// times of every tile in 252 products of n 1640 to 22016, k 320 to 11008, 48
// to 8192 rows, all with bf16 outputs: the tile picked is the fastest or within
// 8 % of it in all but three (10 to 16 %).  (fp32 outputs, whose blocks take 16-bit
// instructions, go by the table of sums scaled apart; their tiles have not been
// timed one against the other.)  Small tiles fill the chip with few rows, large ones
// read less per product: powers of two, 2048 x 4096, k 4096 takes 89, 62, 47,
// 38, 37 and 49 us on the tiles below, 256 rows of it 15, 14, 17, 21, 27 and
// 43, 4096 rows 59 on the last and 70 on the one before it.
//   few rows   16 weight rows a workgroup, no LDS (m <= 16; to 32 rows while a
//              second group of rows costs less than the tiles' start: 32 rows,
//              n 1640, k 1024: 4.7 against 5.4 us; n 2048, k 4096: 8.6 against
//              8.5; n 7376, k 2048: 8.9 against 7.0)
//   64 x 32    4 k groups of waves, one workgroup a CU; 2 k groups, two
//   64 x 64    2 k groups      64 x 128, 128 x 128   one
//   128 x 256  eight waves, three stages (fp32 scales, 2048 x 4096, k 11008:
//              100 us on 128 x 128, 90 on these)
//   256 x 256  power-of-two scales and 16-bit outputs
Fp8Plan plan_fp8_gemm(int m, int n, int kb, bool silu, bool exact, bool pow2, int cus) {
  Fp8Plan p = {};
  p.cus = cus;
  if (m <= 16 || (m <= 32 && (int64_t)m * n * kb <= 1 << 21)) {
    p.few = true;
    p.bm = m <= 16 ? 16 : 32;
    p.bn = silu ? 32 : 16;
    return p;
  }
  struct Shape { int bm, bn; float one, two, fix1, fix2; };        // 256 columns: one of the only CU in use, two of all
  static const Shape fast[] = {{64, 32, 0.15f, 0.26f, 1.3f, 2.1f},  {64, 64, 0.29f, 0.34f, 1.4f, 3.0f},
                               {64, 128, 0.37f, 0.55f, 1.0f, 3.2f}, {128, 128, 0.55f, 0.87f, 3.2f, 4.2f},
                               {128, 256, 0.59f, 0.81f, 2.9f, 6.2f}, {256, 256, 0.87f, 1.28f, 9.6f, 12.9f}};
  // the sums of a block scaled apart
  static const Shape part[] = {{64, 32, 0.14f, 0.26f, 1.7f, 2.3f},  {64, 64, 0.29f, 0.34f, 1.3f, 2.8f},
                               {64, 128, 0.38f, 0.57f, 2.2f, 3.3f}, {128, 128, 0.58f, 0.99f, 3.3f, 5.1f},
                               {128, 256, 0.80f, 0.80f, 2.7f, 7.9f}};
  const bool scaled = exact || !pow2;
  float best = 0.f;
  for (int i = 0; i < (scaled ? 5 : 6); ++i) {
    const Shape& h = scaled ? part[i] : fast[i];
    if (h.bn == 32 && silu) continue;
    const bool alone = h.bn == 256;
    const int64_t tiles = ceil_div(m, h.bm) * ceil_div(n, h.bn), slots = alone ? cus : 2 * cus;
    const int64_t rounds = tiles / slots, rest = tiles - rounds * slots;
    float t = rounds * (kb * h.two + h.fix2);
    if (rest && alone) t += kb * (h.one + (h.two - h.one) * rest / cus) + h.fix1;
    else if (rest) t += rest <= cus ? kb * h.one + h.fix1 : kb * h.two + h.fix2;
    if (p.bm == 0 || t < best) {
      best = t;
      p.bm = h.bm;
      p.bn = h.bn;
      p.ks = h.bm == 64 && h.bn == 32 && tiles <= cus ? 4 : 2;
    }
  }
  return p;
}

template <int WM, int WN, int I, int J, int KS, int NST, typename S, typename O, bool SILU>
static int launch_tile(Fp8GemmArgs a, hipStream_t st) {
  a.tiles_m = (int)ceil_div(a.m, 32 * WM * I);
  a.tiles_n = (int)ceil_div(a.n, 32 * WN * J);
  const dim3 grid((unsigned)(8 * ceil_div((int64_t)a.tiles_m * a.tiles_n, 8))), block(64 * WM * WN * KS);
  hipLaunchKernelGGL((fp8_gemm_kernel<WM, WN, I, J, KS, NST, S, O, SILU>), grid, block, 0, st, a);
  return (int)hipGetLastError();
}
template <typename O, bool SILU> static int launch_wide(Fp8GemmArgs a, int cus, hipStream_t st) {
  a.tiles_m = (int)ceil_div(a.m, WT);
  a.tiles_n = (int)ceil_div(a.n, WT);
  const int64_t per = ceil_div((int64_t)a.tiles_m * a.tiles_n, 8);        // tiles of an XCD
  const dim3 grid((unsigned)(8 * std::min<int64_t>(per, std::max(1, cus / 8))));
  hipLaunchKernelGGL((fp8_gemm_wide_kernel<O, SILU>), grid, dim3(256), 0, st, a);
  return (int)hipGetLastError();
}
template <typename S, typename O, bool SILU> static int launch_shape(const Fp8GemmArgs& a, const Fp8Plan& p, hipStream_t st) {
  if constexpr (!__is_same(O, float) && S::pow2)
    if (p.bm == 256) return launch_wide<O, SILU>(a, p.cus, st);
  if (p.bn == 256) return launch_tile<2, 4, 2, 2, 1, 3, S, O, SILU>(a, st);
  if (p.bm == 128) return launch_tile<2, 2, 2, 2, 1, 2, S, O, SILU>(a, st);
  if (p.bn == 128) return launch_tile<2, 2, 1, 2, 1, 3, S, O, SILU>(a, st);
  if constexpr (!SILU)
    if (p.bn == 32) return p.ks == 4 ? launch_tile<2, 1, 1, 1, 4, 3, S, O, SILU>(a, st) : launch_tile<2, 1, 1, 1, 2, 3, S, O, SILU>(a, st);
  return launch_tile<2, 1, 1, 2, 2, 2, S, O, SILU>(a, st);
}
template <typename S, typename O> static int launch_silu(const Fp8GemmArgs& a, const Fp8Plan& p, bool silu, hipStream_t st) {
  return silu ? launch_shape<S, O, true>(a, p, st) : launch_shape<S, O, false>(a, p, st);
}
template <typename S> static int launch_out(const Fp8GemmArgs& a, const Fp8Plan& p, int od, bool silu, hipStream_t st) {
  if (od == STARKV_F16) return launch_silu<S, _Float16>(a, p, silu, st);
  if (od == STARKV_BF16) return launch_silu<S, __bf16>(a, p, silu, st);
  return launch_silu<S, float>(a, p, silu, st);
}
int launch_fp8_gemm(const Fp8GemmArgs& a, const Fp8Plan& p, int out_dtype, int scale_dtype, bool silu, hipStream_t st) {
  return scale_dtype == STARKV_E8M0 ? launch_out<ScaleE8>(a, p, out_dtype, silu, st)
                                    : launch_out<ScaleF32>(a, p, out_dtype, silu, st);
}

}  // namespace starkv
