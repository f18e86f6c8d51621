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
}  // namespace

// WM x WN waves; SILU: the tile's columns are BN / 2 gate columns and the same up columns
template <int BM, int BN, int WM, int WN, typename S, typename O, bool SILU, bool SPLIT>
__global__ __launch_bounds__(64 * WM * WN, BM * BN >= 32768 ? 2 : 1) void fp8_gemm_kernel(const Fp8GemmArgs a) {
  constexpr int NW = WM * WN, TM = BM / WM, TN = BN / WN;    // wave tile
  constexpr int MF = TM / 16, NF = TN / 16;
  constexpr int LOADS = (BM + BN) / 8 / NW;                  // 1 KB loads per wave and stage
  static_assert(LOADS * 8 * NW == BM + BN && BM % 8 == 0, "whole loads");
  static_assert(!SILU || NF % 2 == 0, "gate and up halves");
  constexpr bool EXACT = __is_same(O, float);      // 16-bit instructions (see half_of)
  __shared__ __attribute__((aligned(16))) uint8_t st0[(BM + BN) * 128];
  __shared__ __attribute__((aligned(16))) uint8_t st1[(BM + BN) * 128];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % WM, wn = wave / WM;
  const int c = lane & 15, g = lane >> 4;

  // workgroup -> tile: workgroup i runs on XCD i % 8; each XCD takes a
  // contiguous run of tiles, which go down eight row tiles before the next column
  const int tiles = a.tiles_m * a.tiles_n;
  const int total = tiles * a.splits;
  const int per = (total + 7) >> 3;
  const int idx = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || idx >= total) return;
  const int split = idx / tiles, tl = idx - split * tiles;
  constexpr int GROUP = 8;
  const int grp = tl / (GROUP * a.tiles_n), rem = tl - grp * GROUP * a.tiles_n;
  const int gm = min(GROUP, a.tiles_m - grp * GROUP);
  const int tm = grp * GROUP + rem % gm, tn = rem / gm;
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

  // this lane's source of each of the wave's loads: 8 rows x 8 pieces
  const int rs = lane >> 3, q8 = lane & 7;
  const uint8_t* src[LOADS];
  int piece[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) {
    const int row = (wave * LOADS + i) * 8 + rs;
    piece[i] = q8 ^ swz(row & 15);
    src[i] = row < BM ? (const uint8_t*)a.x + (int64_t)min(m0 + row, a.m - 1) * a.xs
                      : a.w + (int64_t)min(wrow_of(row - BM), a.n - 1) * a.ws;
  }
  const int last = (a.k - 1) >> 4;
  auto issue = [&](uint8_t* st, int kb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i)
      __builtin_amdgcn_global_load_lds((const void*)(src[i] + (int64_t)min(kb * 8 + piece[i], last) * 16),
                                       (lds_void*)(st + (wave * LOADS + i) * 1024), 16, 0, 0);
  };

  // scales: activation row m0 + wm TM + 16 i + c, weight block of the wave's (gate / up) rows
  typedef typename S::T ST;
  constexpr int NS = SILU ? 2 : 1;
  const ST* sxp[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i)
    sxp[i] = (const ST*)a.sx + (int64_t)min(m0 + wm * TM + 16 * i + c, a.m - 1) * a.sxr;
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
    for (int i = 0; i < MF; ++i) sc.x[i] = sxp[i][(int64_t)kb * a.sxb];
#pragma unroll
    for (int t = 0; t < NS; ++t) sc.w[t] = swp[t][(int64_t)kb * a.swb];
  };
  // block kb from stage `cur` with the scales `sc`, the next one's loads into
  // `nxt` and `sn` issued first; LAST: none follows, and it may end before 128 columns
  auto step = [&](auto last_c, const uint8_t* cur, uint8_t* nxt, int kb, const Sc& sc, Sc& sn) __attribute__((always_inline)) {
    constexpr bool LAST = decltype(last_c)::value;
    // this wave's loads of block kb (issued a block ago) landed, and its reads of the other stage are done ...
    __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("s_barrier" ::: "memory");        // ... and everyone's
    if constexpr (!LAST) {
      issue(nxt, kb + 1);
      scales(sn, kb + 1);
    }
    const int nv = a.k - kb * FP8_BLOCK - 16 * g;
    auto frag = [&](int row16) __attribute__((always_inline)) {
      const uint8_t* p = cur + row16 * 128;
      uint4 lo = *(const uint4*)(p + rd0), hi = *(const uint4*)(p + (rd0 ^ 64));
      if constexpr (LAST) {                        // bytes past column k: any value in either operand
        lo = keep_bytes(lo, nv);
        hi = keep_bytes(hi, nv - 64);
      }
      return frag8(lo, hi);
    };
    intx8 wf[NF];
#pragma unroll
    for (int j = 0; j < NF; ++j) wf[j] = frag(BM + wn * TN + 16 * j);
    if constexpr (EXACT) {
      intx8 xf[MF];
      floatx4 p[NF][MF];
#pragma unroll
      for (int i = 0; i < MF; ++i) xf[i] = frag(wm * TM + 16 * i);
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
      return;
    }
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const intx8 xf = frag(wm * TM + 16 * i);
      if constexpr (S::pow2) {
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[j][i] = mfma8(wf[j], xf, acc[j][i], sc.w[SILU ? j / (NF / 2) : 0], sc.x[i]);
      } else {
#pragma unroll
        for (int j = 0; j < NF; ++j) {
          const float s = sc.x[i] * sc.w[SILU ? j / (NF / 2) : 0];
          const floatx4 p = mfma8(wf[j], xf, floatx4{0.f, 0.f, 0.f, 0.f}, E8_ONE, E8_ONE);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(p[e], s, acc[j][i][e]);
        }
      }
    }
  };
  const std::false_type more{};
  const std::true_type end{};
  Sc s0, s1;
  issue(st0, kb0);
  scales(s0, kb0);
  int kb = kb0;
  for (; kb + 2 < kb1; kb += 2) {
    step(more, st0, st1, kb, s0, s1);
    step(more, st1, st0, kb + 1, s1, s0);
  }
  if (kb + 1 < kb1) {
    step(more, st0, st1, kb, s0, s1);
    step(end, st1, st0, kb + 1, s1, s0);
  } else {
    step(end, st0, st1, kb, s0, s1);
  }

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
template <typename S, typename O, bool SILU> static int launch_shape(const Fp8GemmArgs& a, const Fp8Plan& p, hipStream_t st) {
  if constexpr (!__is_same(O, float))
    if (p.bm == 256) return launch_tile<256, 256, 4, 2, S, O, SILU>(a, st);
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
