// e4m3 projection of many rows: out[m][n] = X W^T over blocks of 128 columns,
// each with its own scales (the definition is in starkv.h).
//
// A workgroup computes a BM x BN tile of the output, k block by k block: the
// block's BM + BN rows of 128 bytes go to LDS by direct loads (16 bytes a
// lane), one stage ahead of the matrix instructions.  One 16 x 16 x 128
// instruction is one block's partial sum:
//   * power-of-two scales ride in the instruction itself (its operands carry
//     an exponent byte each), so the accumulators take the sums directly;
//   * fp32 scales multiply each partial sum, acc += p * (sx sw).
// The weight rows are the instruction's A operand and the activations its B
// operand: a lane then holds four consecutive columns of one output row, and
// one activation scale.
//
// LDS rows are 128 bytes; 16-byte piece c of row r lies at piece
// c ^ swz(r), swz(r) = (r & 7) ^ ((r >> 3) & 1): the 16 rows that one operand
// read touches at the same piece fall on distinct banks, taken 8 or 16 lanes
// at a time.
//
// Two stages, each an array of its own, the loop unrolled over them (the
// compiler then sees that reading one cannot alias the loads in flight into
// the other), and one barrier per block.
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

// Workgroup -> tile (tm, tn) and 1 + its split of k; 0: none.  Workgroup i
// runs on XCD i % 8; each XCD takes a contiguous run of tiles, which go down
// eight row tiles before the next column, so that its L2 serves most reads.
__device__ inline void tile_at(const Fp8GemmArgs& a, int tl, int& tm, int& tn) {
  constexpr int GROUP = 8;
  const int grp = tl / (GROUP * a.tiles_n), rem = tl - grp * GROUP * a.tiles_n;
  const int gm = min(GROUP, a.tiles_m - grp * GROUP);
  tm = grp * GROUP + rem % gm;
  tn = rem / gm;
}
__device__ inline int tile_of(const Fp8GemmArgs& a, int wg, int& tm, int& tn) {
  const int tiles = a.tiles_m * a.tiles_n, total = tiles * a.splits;
  const int per = (total + 7) >> 3;
  const int idx = (wg & 7) * per + (wg >> 3);
  if (idx >= total) return 0;
  const int split = idx / tiles;
  tile_at(a, idx - split * tiles, tm, tn);
  return split + 1;
}

// eight consecutive results (16-bit, and the residual added) from column col on, nv of them inside the row
template <typename O> __device__ inline void store8(const Fp8GemmArgs& a, int row, int col, int nv, float (&v)[8]) {
  O* o = (O*)a.out + (int64_t)row * a.os + col;
  const O* rp = (const O*)a.res + (int64_t)row * a.rs + col;
  if (a.vec_out >= 2 && nv >= 8) {
    if (a.res) {
      const uint4 t = *(const uint4*)rp;
      O r[8];
      __builtin_memcpy(r, &t, 16);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += (float)r[e];
    }
    O t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (O)v[e];
    uint4 u;
    __builtin_memcpy(&u, t, 16);
    *(uint4*)o = u;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < nv) {
        if (a.res) v[e] += (float)rp[e];
        o[e] = (O)v[e];
      }
  }
}
}  // namespace

// Zero the bytes past column k of a stage that holds the row's last, short
// block (nv < 128 columns): they are any value, also NaN.
template <int ROWS, int THREADS> __device__ inline void zero_tail(uint8_t* st, int nv) {
  const int p0 = nv >> 4, np = 8 - p0;             // pieces from the first short one on
  for (int i = threadIdx.x; i < ROWS * np; i += THREADS) {
    const int r = i / np, p = p0 + i - r * np;
    uint4* q = (uint4*)(st + r * 128 + ((p ^ swz(r & 15)) << 4));
    *q = keep_bytes(*q, nv - 16 * p);
  }
}

// WM x WN waves; SILU: the tile's columns are BN / 2 gate columns and the same up columns
template <int BM, int BN, int WM, int WN, typename S, typename O, bool SILU, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN, BM * BN >= 32768 ? 2 : 1) void fp8_gemm_kernel(const Fp8GemmArgs a) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN;    // wave tile
  constexpr int MF = TM / 16, NF = TN / 16;
  constexpr int LOADS = (BM + BN) / 8 / NW;                  // 1 KB loads per wave and stage
  static_assert(LOADS * 8 * NW == BM + BN && BM % 8 == 0, "whole loads");
  static_assert(!SILU || NF % 2 == 0, "gate and up halves");
  constexpr bool EXACT = __is_same(O, float);      // 16-bit instructions (see half_of)
  constexpr int STAGE = (BM + BN) * 128;
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int c = lane & 15, g = lane >> 4;

  int tm, tn;
  const int split = tile_of(a, blockIdx.x, tm, tn) - 1;
  if (split < 0) return;
  const int m0 = tm * BM, n0 = tn * (SILU ? BN / 2 : BN);
  const int kb0 = split * a.kb_per, kb1 = min(a.kb, kb0 + a.kb_per);

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
  const int last = (a.k - 1) >> 4;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void*)lds;
  auto issue = [&](int stage, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int row = (wave * LOADS + i) * 8;      // uniform; the lane's piece of its row is q8 ^ swz(row + rs)
      const int p = min(kb * 8 + (q8 ^ rs ^ ((row >> 3) & 1)), last);
      dma_1k(row < BM ? xbase : wbase, off[i] + (uint32_t)p * 16, lds0 + stage + row * 128);
    }
  };

  // scales: activation row m0 + wm TM + 16 i + c, weight block of the wave's (gate / up) rows
  typedef typename S::T ST;
  constexpr int NS = SILU ? 2 : 1;
  const ST* const sxp = (const ST*)a.sx + (int64_t)m0 * a.sxr;
  uint32_t sxo[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) sxo[i] = (uint32_t)((min(m0 + wm * TM + 16 * i + c, a.m - 1) - m0) * a.sxr);
  const ST* swp[NS];
#pragma unroll
  for (int t = 0; t < NS; ++t)
    swp[t] = (const ST*)a.sw + (int64_t)(min(wrow_of(wn * TN + t * (TN / 2)), a.n - 1) >> 7) * a.swr;

  floatx4 acc[NF][MF];
#pragma unroll
  for (int j = 0; j < NF; ++j)
#pragma unroll
    for (int i = 0; i < MF; ++i) acc[j][i] = floatx4{0.f, 0.f, 0.f, 0.f};

  const int rd0 = c * 128 + ((g ^ swz(c)) << 4);            // piece g of row c; piece g + 4 lies 64 bytes off (xor)
  struct Sc { ST x[MF], w[NS]; };
  auto scales = [&](Sc& sc, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MF; ++i) sc.x[i] = (sxp + (int64_t)kb * a.sxb)[sxo[i]];
#pragma unroll
    for (int t = 0; t < NS; ++t) sc.w[t] = swp[t][(int64_t)kb * a.swb];
  };
  // The blocks in the order last, first, second ..: the row's last one may be
  // short, and what lies behind it is zeroed before the loop starts.
  const int n = kb1 - kb0;
  auto block = [&](int t) { return t == 0 || t >= n ? kb1 - 1 : kb0 + t - 1; };
  Sc sc, sn;
  issue(0, block(0));
  scales(sc, block(0));
  if (kb1 == a.kb && (a.k & (FP8_BLOCK - 1))) {
    __builtin_amdgcn_s_waitcnt(0x0070);
    __syncthreads();
    zero_tail<BM + BN, 64 * NW>(lds, a.k & (FP8_BLOCK - 1));
  }
  int at = 0;
  for (int t = 0; t < n; ++t, at ^= STAGE) {
    // this wave's loads of block t (issued a block ago) landed, and its reads of the other stage are done ...
    __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("s_barrier" ::: "memory");        // ... and everyone's
    issue(at ^ STAGE, block(t + 1));               // (after the last block: one of them again, for nobody)
    scales(sn, block(t + 1));
    const uint8_t* const cur = lds + at;
    auto frag = [&](int row16) __attribute__((always_inline)) {
      const uint8_t* p = cur + row16 * 128;
      return frag8(*(const uint4*)(p + rd0), *(const uint4*)(p + (rd0 ^ 64)));
    };
    intx8 xf[MF];
#pragma unroll
    for (int i = 0; i < MF; ++i) xf[i] = frag(wm * TM + 16 * i);
    if constexpr (EXACT) {
      intx8 wf[NF];
      floatx4 p[NF][MF];
#pragma unroll
      for (int j = 0; j < NF; ++j) wf[j] = frag(BM + wn * TN + 16 * j);
#pragma unroll
      for (int j = 0; j < NF; ++j)
#pragma unroll
        for (int i = 0; i < MF; ++i) p[j][i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        half8 wh[NF], xh[MF];
#pragma unroll
        for (int j = 0; j < NF; ++j) wh[j] = half_of(wf[j], q);
#pragma unroll
        for (int i = 0; i < MF; ++i) xh[i] = half_of(xf[i], q);
#pragma unroll
        for (int j = 0; j < NF; ++j)
#pragma unroll
          for (int i = 0; i < MF; ++i) p[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(wh[j], xh[i], p[j][i], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) {
          const float s = scale_f32(sc.x[i]) * scale_f32(sc.w[SILU ? j / (NF / 2) : 0]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(p[j][i][e], s, acc[j][i][e]);
        }
    } else {
#pragma unroll
      for (int j = 0; j < NF; ++j) {
        const intx8 wf = frag(BM + wn * TN + 16 * j);
        const ST sw = sc.w[SILU ? j / (NF / 2) : 0];
#pragma unroll
        for (int i = 0; i < MF; ++i) {
          if constexpr (S::pow2) {
            acc[j][i] = mfma8(wf, xf[i], acc[j][i], sw, sc.x[i]);
          } else {
            const float s = sc.x[i] * sw;
            const floatx4 p = mfma8(wf, xf[i], floatx4{0.f, 0.f, 0.f, 0.f}, E8_ONE, E8_ONE);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(p[e], s, acc[j][i][e]);
          }
        }
      }
    }
    sc = sn;
  }
  __builtin_amdgcn_s_waitcnt(0x0070);              // the last loads, before the workgroup gives up its LDS

  // lane (c, g): columns 16 j + 4 g .. + 3 of row 16 i + c of the wave's tile
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int row = m0 + wm * TM + 16 * i + c;
    if (row >= a.m) continue;
    const float r = !SPLIT && a.rscale ? a.rscale[row] : 1.f;
#pragma unroll
    for (int j = 0; j < (SILU && !SPLIT ? NF / 2 : NF); ++j) {
      float v[4];
      if constexpr (SPLIT) {
        const int col = wrow_of(wn * TN + 16 * j) + 4 * g, nv = a.n - col;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[j][i][e];
        // the row pitch of the partial sums is a whole number of 4 columns
        const int np = (a.n + 3) & ~3;
        if (nv > 0) *(float4*)(a.part + ((int64_t)split * a.m + row) * np + col) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
        const int col = (SILU ? n0 + wn * (TN / 2) + 16 * j : n0 + wn * TN + 16 * j) + 4 * g;
        const int nv = (SILU ? a.half : a.n) - col;
        if (nv <= 0) continue;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = SILU ? silu_mul_f32(r * acc[j][i][e], r * acc[SILU ? j + NF / 2 : j][i][e]) : r * acc[j][i][e];
        if (!SILU && a.res) {
          float t[4];
          load4<O>((const O*)a.res + (int64_t)row * a.rs + col, t, nv, a.vec_out != 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] += t[e];
        }
        store4<O>((O*)a.out + (int64_t)row * a.os + col, v, nv, a.vec_out != 0);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Power-of-two scales, 256 x 256 tiles: four waves of 128 x 128 (one per SIMD,
// 256 accumulators each), 32 x 32 x 64 instructions.  The matrix cores need
// 2048 cycles for a block; the operands of four 128 x 128 wave tiles take
// 128 KB of LDS reads and 64 KB of writes per block, 1536 cycles at 128
// bytes, where eight waves of 64 x 128 would take all of the 2048.
//
// A block is two halves of 64 columns, each with operand registers of its own:
//   * half 0's products run while half 1's operands are read;
//   * then every wave has read this stage and (its loads have landed and) the
//     next stage is whole: the one barrier of the block;
//   * half 1's products run while the next block's half 0 is read, and the
//     block after that is loaded into the stage just freed.
// So neither the barrier nor an LDS read is waited for with the matrix cores
// idle.  A workgroup takes tile after tile: the next tile's first blocks load
// while this one's results are stored, by way of LDS so that whole 128-byte
// lines leave (straight from the accumulators' layout, 16 bytes a row, the
// stores of a tile took as long as 1600 columns of products).
// ---------------------------------------------------------------------------
constexpr int WT = 256;                            // tile rows and columns
constexpr int WSTAGE = 2 * WT * 128;               // bytes of a stage
constexpr int WOUT = 32 * 64 * 4;                  // bytes a wave stages of its results: 32 rows x 64 columns, fp32

__device__ inline floatx16 mfma8_32(intx8 a, intx8 b, floatx16 c, int scale_a, int scale_b) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, 0, scale_a, 0, scale_b);
}

template <typename O, bool SILU>
__global__ __launch_bounds__(256, 1) void fp8_gemm_wide_kernel(const Fp8GemmArgs a) {
  static_assert(sizeof(O) == 2, "16-bit outputs");
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * WSTAGE + 4 * WOUT];
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
  const uint8_t *sxp, *swp[2];
  uint32_t sxo[4];
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
      off[i] = (uint32_t)(row * (isx ? a.xs : a.ws));
    }
    base = isx ? (const uint8_t*)a.x + (int64_t)m0 * a.xs : a.w + (int64_t)n0 * a.ws;
    sxp = (const uint8_t*)a.sx + (int64_t)m0 * a.sxr;
#pragma unroll
    for (int i = 0; i < 4; ++i) sxo[i] = (uint32_t)((min(m0 + wm * 128 + 32 * i + c, a.m - 1) - m0) * a.sxr);
#pragma unroll
    for (int t = 0; t < 2; ++t)
      swp[t] = (const uint8_t*)a.sw + (int64_t)(min(wrow(wn * 128 + 64 * t), a.n - 1) >> 7) * a.swr;
  };
  struct Sc { uint8_t x[4], w[2]; };
  auto scales = [&](Sc& sc, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sc.x[i] = (sxp + (int64_t)kb * a.sxb)[sxo[i]];
#pragma unroll
    for (int t = 0; t < (SILU ? 2 : 1); ++t) sc.w[t] = swp[t][(int64_t)kb * a.swb];
  };
  // The blocks in the order last, first, second .. (the last may be short:
  // what lies behind it is zeroed before the loop starts).  A full block's
  // pieces need no check against the row's end.
  auto block = [&](int t) { return t == 0 ? end : t > end ? 0 : t - 1; };
  auto issue_last = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      dma_1k(base, off[i] + (uint32_t)min(end * 8 + (piece0 ^ (i & 1)), last) * 16, lds0 + i * 1024);
  };
  const uint32_t po[2] = {(uint32_t)min(piece0, last) * 16, (uint32_t)min(piece0 ^ 1, last) * 16};
  auto issue1 = [&](int stage, int kb, int i) __attribute__((always_inline)) {
    dma_1k(base + (int64_t)kb * FP8_BLOCK, off[i] + po[i & 1], lds0 + stage + i * 1024);
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
  issue_last();
  scales(sc, end);
  while (true) {
    floatx16 acc[4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[j][i] = floatx16{};
    __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("s_barrier" ::: "memory");
    if (a.k & (FP8_BLOCK - 1)) {
      zero_tail<2 * WT, 256>(lds, a.k & (FP8_BLOCK - 1));
      __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) issue1(WSTAGE, block(1), i);
    Half h0, h1;
#pragma unroll
    for (int q = 0; q < 16; ++q) read1(h0, lds, 0, q);
    int cur = 0;
    auto product = [&](const Half& o, int q) __attribute__((always_inline)) {
      // row groups in the order in which the reads bring them
      constexpr int ORDER[16] = {0, 1, 4, 5, 2, 6, 8, 9, 10, 3, 7, 11, 12, 13, 14, 15};
      const int j = ORDER[q] >> 2, i = ORDER[q] & 3;
      acc[j][i] = mfma8_32(frag8(o.w[j][0], o.w[j][1]), frag8(o.x[i][0], o.x[i][1]), acc[j][i], sc.w[SILU ? j >> 1 : 0],
                           sc.x[i]);
    };
    for (int t = 0; t <= end; ++t, cur ^= WSTAGE) {    // block(t) in stage `cur`, its half 0 in h0, its scales in sc
      scales(sn, block(t + 1));
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        product(h0, q);
        read1(h1, lds + cur, 1, q);
        __builtin_amdgcn_sched_barrier(0);
      }
      // half 1 read; this wave's part of the next stage landed
      __builtin_amdgcn_s_waitcnt(0x0070);
      asm volatile("s_barrier" ::: "memory");
      __builtin_amdgcn_sched_barrier(0);
      const int kn = block(t + 2);
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        product(h1, q);
        issue1(cur, kn, q);
        read1(h0, lds + (cur ^ WSTAGE), 0, q);
        __builtin_amdgcn_sched_barrier(0);
      }
      sc = sn;
    }
    // after the last blocks the loads repeated one and the reads took what was there, for nobody
    __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("s_barrier" ::: "memory");
    const int om = m0 + wm * 128, on = n0 + wn * (SILU ? 64 : 128);
    idx += stride;
    const bool more = idx < stop;
    if (more) {
      take(idx);
      issue_last();
      scales(sc, end);
    }

    // Results: lane (c, g) holds columns 32 j + 8 q + 4 g .. + 3 of row 32 i + c of acc[j][i].  Two accumulators
    // (SILU: gate and up) go through the wave's own part of LDS at a time, 32 rows of 256 bytes, 16-byte piece p of
    // row r at p ^ (r & 15).  One copy of the code that finishes and stores them serves all: a tile's stores are run
    // once, and unrolled they came from memory instruction by instruction (48 KB of code: 25 us a tile).
    uint8_t* const ob = lds + 2 * WSTAGE + wave * WOUT;
    const int ncol = SILU ? a.half : a.n;
#pragma unroll 1
    for (int ch = 0; ch < 8; ++ch) {
      auto put = [&](auto chc) __attribute__((always_inline)) {
        constexpr int C = decltype(chc)::value, I = C >> 1, J = C & 1;
#pragma unroll
        for (int jj = 0; jj < 2; ++jj)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const floatx16& v = acc[SILU ? J + 2 * jj : 2 * J + jj][I];
            *(floatx4*)(ob + c * 256 + (((8 * jj + 2 * q + g) ^ (c & 15)) << 4)) =
                floatx4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
          }
      };
      switch (ch) {
        case 0: put(std::integral_constant<int, 0>{}); break;
        case 1: put(std::integral_constant<int, 1>{}); break;
        case 2: put(std::integral_constant<int, 2>{}); break;
        case 3: put(std::integral_constant<int, 3>{}); break;
        case 4: put(std::integral_constant<int, 4>{}); break;
        case 5: put(std::integral_constant<int, 5>{}); break;
        case 6: put(std::integral_constant<int, 6>{}); break;
        default: put(std::integral_constant<int, 7>{}); break;
      }
      // eight columns a lane: 8 lanes to a row of 64 columns, or 4 to a row of 32 gate and 32 up columns
      constexpr int LPR = SILU ? 4 : 8, RPI = 64 / LPR;
      const int rc = lane & (LPR - 1);
      const int col = on + (ch & 1) * (SILU ? 32 : 64) + 8 * rc;
#pragma unroll 1
      for (int lr = lane / LPR; lr < 32; lr += RPI) {
        const int row = om + 32 * (ch >> 1) + lr;
        const uint8_t* p = ob + lr * 256;
        const int sw = lr & 15;
        const floatx4 u0 = *(const floatx4*)(p + (((2 * rc) ^ sw) << 4)), u1 = *(const floatx4*)(p + (((2 * rc + 1) ^ sw) << 4));
        if (row >= a.m || col >= ncol) continue;
        const float r = a.rscale ? a.rscale[row] : 1.f;
        float v[8];
        if constexpr (SILU) {
          const floatx4 w0 = *(const floatx4*)(p + (((2 * rc + 8) ^ sw) << 4)), w1 = *(const floatx4*)(p + (((2 * rc + 9) ^ sw) << 4));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[e] = silu_mul_f32(r * u0[e], r * w0[e]);
            v[4 + e] = silu_mul_f32(r * u1[e], r * w1[e]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) { v[e] = r * u0[e]; v[4 + e] = r * u1[e]; }
        }
        store8<O>(a, row, col, ncol - col, v);
      }
    }
    if (!more) break;
  }
}

// out = epilogue of the splits' partial sums, added in split order
template <typename O, bool SILU> __global__ __launch_bounds__(256) void fp8_join_kernel(const Fp8GemmArgs a) {
  const int np = (a.n + 3) & ~3, cols = SILU ? a.half : a.n;
  const int c4 = (cols + 3) >> 2;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= (int64_t)a.m * c4) return;
  const int64_t row = id / c4;
  const int col = (int)(id - row * c4) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f), u = s;
  for (int z = 0; z < a.splits; ++z) {
    const float* p = a.part + ((int64_t)z * a.m + row) * np + col;
    const float4 t = *(const float4*)p;
    s.x += t.x; s.y += t.y; s.z += t.z; s.w += t.w;
    if constexpr (SILU) {
      const float4 t2 = *(const float4*)(p + a.half);
      u.x += t2.x; u.y += t2.y; u.z += t2.z; u.w += t2.w;
    }
  }
  const float r = a.rscale ? a.rscale[row] : 1.f;
  float v[4] = {r * s.x, r * s.y, r * s.z, r * s.w};
  if constexpr (SILU) {
    const float w[4] = {r * u.x, r * u.y, r * u.z, r * u.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = silu_mul_f32(v[e], w[e]);
  }
  const int nv = cols - col;
  if (!SILU && a.res) {
    float t[4];
    load4<O>((const O*)a.res + row * a.rs + col, t, nv, a.vec_out != 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += t[e];
  }
  store4<O>((O*)a.out + row * a.os + col, v, nv, a.vec_out != 0);
}

Fp8Plan plan_fp8_gemm(int m, int n, int kb, bool exact, int cus) {
  Fp8Plan p = {};
  p.cus = cus;
  const bool big = !exact && (int64_t)ceil_div(m, 256) * ceil_div(n, 256) >= cus;
  p.bm = big ? 256 : m <= 64 ? 64 : 128;
  p.bn = big ? 256 : 128;
  const int64_t tiles = ceil_div(m, p.bm) * ceil_div(n, p.bn);
  int splits = 1;
  while (splits < 16 && tiles * splits * 2 <= 2 * cus && kb / (splits * 2) >= 4) splits *= 2;
  p.kb_per = (int)ceil_div(kb, splits);
  p.splits = (int)ceil_div(kb, p.kb_per);
  p.part_bytes = p.splits > 1 ? (size_t)p.splits * m * (size_t)round_up(n, 4) * 4 : 0;
  return p;
}

template <int BM, int BN, int WM, int WN, typename S, typename O, bool SILU>
static int launch_tile(Fp8GemmArgs a, hipStream_t st) {
  a.tiles_m = (int)ceil_div(a.m, BM);
  a.tiles_n = (int)ceil_div(a.n, BN);
  const int64_t total = (int64_t)a.tiles_m * a.tiles_n * a.splits;
  const dim3 grid((unsigned)(8 * ceil_div(total, 8))), block(64 * WM * WN);
  if (a.splits > 1) {
    hipLaunchKernelGGL((fp8_gemm_kernel<BM, BN, WM, WN, S, O, SILU, true>), grid, block, 0, st, a);
    const int64_t ids = (int64_t)a.m * ceil_div(SILU ? a.half : a.n, 4);
    hipLaunchKernelGGL((fp8_join_kernel<O, SILU>), dim3((unsigned)ceil_div(ids, 256)), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((fp8_gemm_kernel<BM, BN, WM, WN, S, O, SILU, false>), grid, block, 0, st, a);
  }
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
  if constexpr (!__is_same(O, float))
    if (p.bm == 256) {
      if constexpr (S::pow2) return launch_wide<O, SILU>(a, p.cus, st);
      else return launch_tile<256, 256, 4, 2, S, O, SILU>(a, st);
    }
  if (p.bm == 128) return launch_tile<128, 128, 2, 2, S, O, SILU>(a, st);
  return launch_tile<64, 128, 1, 4, S, O, SILU>(a, st);
}
template <typename S, typename O> static int launch_silu(const Fp8GemmArgs& a, const Fp8Plan& p, bool silu, hipStream_t st) {
  return silu ? launch_shape<S, O, true>(a, p, st) : launch_shape<S, O, false>(a, p, st);
}
template <typename S> static int launch_out(const Fp8GemmArgs& a, const Fp8Plan& p, int od, bool silu, hipStream_t st) {
  if (od == STARKV_F16) return launch_silu<S, _Float16>(a, p, silu, st);
  if (od == STARKV_BF16) return launch_silu<S, __bf16>(a, p, silu, st);
  return launch_silu<S, float>(a, p, silu, st);
}
int launch_fp8_gemm(const Fp8GemmArgs& a0, const Fp8Plan& p, int out_dtype, int scale_dtype, bool silu, hipStream_t st) {
  Fp8GemmArgs a = a0;
  a.splits = p.splits;
  a.kb_per = p.kb_per;
  return scale_dtype == STARKV_E8M0 ? launch_out<ScaleE8>(a, p, out_dtype, silu, st)
                                    : launch_out<ScaleF32>(a, p, out_dtype, silu, st);
}

}  // namespace starkv
