// e4m3 projection of up to 32 rows: out = X W^T as a stream of the
// weight (the definition is in starkv.h).
//
// One matrix instruction (16 x 16 x 128) is one block of 128 columns of 16
// weight rows against 16 activation rows, added up in fp32.  Power-of-two
// scales ride in the instruction, exactly; fp32 scales, and any of fp32
// outputs, multiply a block's sums as sx sw, formed in fp32.  (Formed so for
// power-of-two scales too, a product of scales past 2^127 made NaN of blocks of
// zeros, which the tiles of fp8_gemm.hip add as zeros.)  A workgroup owns NT
// groups of 16 weight rows (SiLU-multiply: 16 gate rows and their 16 up rows)
// and MT groups of 16 activation rows; its waves split the blocks of k and meet
// in LDS at the end.  Weight and activation bytes go from memory to the matrix
// operand registers directly, without LDS: a block or two in flight per wave
// and as many waves as fit.
//
// Bound by the weight stream for few rows (6.5 TB/s beside 3.4 us of launch
// and first loads: m 1, n 22016, k 4096 in 17.3 us), by the reads of the
// activations from L2 for more.
//
// 16-bit activations come quantised by a launch of their own (2.1 to 2.5 us
// for up to 16 rows): quantising them in here, by every workgroup again, cost
// more than that from two rows on (m 8, n 7376, k 4096: 13.5 against 12.0 us,
// m 16: 15.9 against 13.2; m 1: 11.5 against 10.5).
#include <algorithm>
#include <type_traits>

#include "fp8.hpp"

namespace starkv {

namespace {
constexpr int FW_PART = 2;                         // k blocks a wave loads at a time, sums scaled apart (1: the same; 4: 5 to 15 % slower)
}  // namespace

// O: output type; NT: groups of weight rows (SILU: 2, gate and up); MT: groups of activation rows
template <typename S, typename O, int NT, int MT, bool SILU>
__global__ __launch_bounds__(512) void fp8_few_kernel(const Fp8GemmArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  // workgroup i runs on XCD i % 8: the row groups of one weight tile follow each other on one XCD, whose L2 then
  // holds the tile's bytes for all of them
  const int mc = (a.m + 16 * MT - 1) / (16 * MT), at8 = blockIdx.x >> 3;
  const int tile = (at8 / mc) * 8 + (blockIdx.x & 7);
  const int n0 = tile * (SILU ? 16 : 16 * NT), m0 = (at8 % mc) * (16 * MT);
  if (n0 >= (SILU ? a.half : a.n)) return;
  const int last = (a.k - 1) >> 4;                 // the last 16-byte piece that holds a column

  // lane (c, g): pieces g and g + 4 of each block of row c; rows past the end repeat the last one, for nobody
  const uint8_t* wrow[NT];
  const typename S::T* wsc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r0 = n0 + t * (SILU ? a.half : 16);
    wrow[t] = a.w + (int64_t)min(r0 + c, a.n - 1) * a.ws + 16 * g;
    wsc[t] = (const typename S::T*)a.sw + (int64_t)(min(r0, a.n - 1) >> 7) * a.swr;
  }
  const uint8_t* xrow[MT];
  const typename S::T* xsc[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = min(m0 + 16 * i + c, a.m - 1);
    xrow[i] = (const uint8_t*)a.x + (int64_t)r * a.xs + 16 * g;
    xsc[i] = (const typename S::T*)a.sx + (int64_t)r * a.sxr;
  }

  // Scales that the instruction takes are asked for before the bytes they go with: behind them, or behind the first
  // product (where the compiler put one, or two blocks at a time), m 8, n 22016, k 4096 with SiLU took 2 % more.
  constexpr bool SCALED = S::pow2 && !__is_same(O, float);
  constexpr int FW = SCALED ? 1 : FW_PART;
  floatx4 acc[NT][MT];
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[t][i] = floatx4{0.f, 0.f, 0.f, 0.f};
  struct Block {
    uint4 x[MT][2], w[NT][2];
    typename S::T sx[MT], sw[NT];
  };
  auto scales = [&](Block& d, int bb) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < MT; ++i) d.sx[i] = xsc[i][(int64_t)bb * a.sxb];
#pragma unroll
    for (int t = 0; t < NT; ++t) d.sw[t] = wsc[t][(int64_t)bb * a.swb];
  };
  // block bb's bytes; SHORT: pieces behind column k repeat the last one
  auto load = [&](auto short_c, Block& d, int bb) __attribute__((always_inline)) {
    if constexpr (SCALED) {
      scales(d, bb);
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int64_t at = (int64_t)bb * FP8_BLOCK + 64 * h;
      if constexpr (decltype(short_c)::value) at = min(at, (int64_t)(last - g) * 16);
#pragma unroll
      for (int t = 0; t < NT; ++t) d.w[t][h] = *(const uint4*)(wrow[t] + at);
#pragma unroll
      for (int i = 0; i < MT; ++i) d.x[i][h] = *(const uint4*)(xrow[i] + at);
    }
    if constexpr (!SCALED) scales(d, bb);
  };
  auto use = [&](auto short_c, Block& d, int bb) __attribute__((always_inline)) {
    if constexpr (SCALED) __builtin_amdgcn_sched_barrier(0);       // all that a block needs is asked for first
    if constexpr (decltype(short_c)::value) {      // columns past k: any value in either operand
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int nv = a.k - bb * FP8_BLOCK - 16 * (g + 4 * h);
#pragma unroll
        for (int i = 0; i < MT; ++i) d.x[i][h] = keep_bytes(d.x[i][h], nv);
#pragma unroll
        for (int t = 0; t < NT; ++t) d.w[t][h] = keep_bytes(d.w[t][h], nv);
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const intx8 xf = frag8(d.x[i][0], d.x[i][1]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const intx8 wf = frag8(d.w[t][0], d.w[t][1]);
        if constexpr (SCALED) {
          acc[t][i] += mfma8(wf, xf, floatx4{0.f, 0.f, 0.f, 0.f}, d.sw[t], d.sx[i]);
        } else {
          const floatx4 p = __is_same(O, float) ? mfma8_exact(wf, xf)
                                                : mfma8(wf, xf, floatx4{0.f, 0.f, 0.f, 0.f}, E8_ONE, E8_ONE);
          const float sc = scale_f32(d.sx[i]) * scale_f32(d.sw[t]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[t][i][e] = fmaf(p[e], sc, acc[t][i][e]);
        }
      }
    }
  };
  const std::false_type whole{};
  const std::true_type part{};
  // whole blocks; all that a round of FW needs is asked for before any of it is used: one wait for memory a round
  const int kf = a.k / FP8_BLOCK;
  const int b0 = (int)((int64_t)kf * w / nw), b1 = (int)((int64_t)kf * (w + 1) / nw);
  for (int b = b0; b < b1; b += FW) {
    Block d[FW];
#pragma unroll
    for (int u = 0; u < FW; ++u) load(whole, d[u], min(b + u, b1 - 1));
#pragma unroll
    for (int u = 0; u < FW; ++u)
      if (b + u < b1) use(whole, d[u], b + u);
  }
  if (kf < a.kb && w == nw - 1) {                  // the row's last, short block
    Block d;
    load(part, d, kf);
    use(part, d, kf);
  }

  // the waves' sums, in wave order; wave v finishes the tiles v, v + nw ..
  floatx4* red = (floatx4*)lds;                    // [nw][NT][MT][64]
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < MT; ++i) red[((w * NT + t) * MT + i) * 64 + lane] = acc[t][i];
  __syncthreads();
#pragma unroll 1
  for (int f = w; f < (SILU ? MT : NT * MT); f += nw) {
    floatx4 s = red[f * 64 + lane], u = SILU ? red[(MT + f) * 64 + lane] : s;
#pragma unroll 4
    for (int v = 1; v < nw; ++v) {
      s += red[(v * NT * MT + f) * 64 + lane];
      if (SILU) u += red[(v * NT * MT + MT + f) * 64 + lane];
    }
    // lane (c, g) holds columns 4 g .. + 3 of row c
    const int t = SILU ? 0 : f / MT, i = SILU ? f : f - t * MT;
    const int row = m0 + 16 * i + c, col = n0 + 16 * t + 4 * g, nv = (SILU ? a.half : a.n) - col;
    if (row >= a.m || nv <= 0) continue;
    const float r = a.rscale ? a.rscale[row] : 1.f;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = SILU ? silu_mul_f32(r * s[e], r * u[e]) : r * s[e];
    if (!SILU && a.res) {
      float x[4];
      load4<O>((const O*)a.res + (int64_t)row * a.rs + col, x, nv);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += x[e];
    }
    store4<O>((O*)a.out + (int64_t)row * a.os + col, v, nv);
  }
}

template <typename S, typename O, int NT, int MT, bool SILU>
static int launch_few_k(const Fp8GemmArgs& a, hipStream_t st) {
  // 8 waves: 4 and 16 were slower by 5 to 15 % over n 4096 to 22016, k 4096 to 11008
  const int nw = std::max(1, std::min(8, a.kb));
  const size_t lds = (size_t)nw * NT * MT * 1024;
  const int64_t tiles = ceil_div(SILU ? a.half : a.n, SILU ? 16 : 16 * NT);
  const dim3 grid((unsigned)(round_up(tiles, 8) * ceil_div(a.m, 16 * MT)));
  hipLaunchKernelGGL((fp8_few_kernel<S, O, NT, MT, SILU>), grid, dim3(64 * nw), lds, st, a);
  return (int)hipGetLastError();
}
template <typename S, typename O> static int launch_few_t(const Fp8GemmArgs& a, const Fp8Plan& p, bool silu, hipStream_t st) {
  if (silu) return p.bm == 16 ? launch_few_k<S, O, 2, 1, true>(a, st) : launch_few_k<S, O, 2, 2, true>(a, st);
  return p.bm == 16 ? launch_few_k<S, O, 1, 1, false>(a, st) : launch_few_k<S, O, 1, 2, false>(a, st);
}
template <typename S> static int launch_few_o(const Fp8GemmArgs& a, const Fp8Plan& p, int od, bool silu, hipStream_t st) {
  if (od == STARKV_F16) return launch_few_t<S, _Float16>(a, p, silu, st);
  if (od == STARKV_BF16) return launch_few_t<S, __bf16>(a, p, silu, st);
  return launch_few_t<S, float>(a, p, silu, st);
}

int launch_fp8_few(const Fp8GemmArgs& a, const Fp8Plan& p, int out_dtype, int scale_dtype, bool silu, hipStream_t st) {
  return scale_dtype == STARKV_E8M0 ? launch_few_o<ScaleE8>(a, p, out_dtype, silu, st)
                                    : launch_few_o<ScaleF32>(a, p, out_dtype, silu, st);
}

}  // namespace starkv
