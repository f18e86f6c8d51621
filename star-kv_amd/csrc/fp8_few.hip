// e4m3 projection of at most 16 rows (decode steps): out = x W^T with the
// weight read once.
//
//   y[i][j] = r_i sum_b sx[i][b] sw[j / 128][b] sum_{k in b} qx[i][k] qw[j][k]
//
// One matrix instruction (16 x 16 x 128) is one block of 128 columns of 16
// weight rows against the (at most 16) activation rows; its partial sums are
// scaled by sx sw in fp32.  A workgroup owns 16 weight rows (SiLU-multiply:
// 16 gate rows and their 16 up rows); its waves split the blocks of k and
// meet in LDS at the end.  Weight bytes go from memory to the matrix operand
// registers directly, FW blocks of 16 x 128 bytes in flight per wave.  16-bit
// activations are quantised on the way, in registers: a lane holds the 32
// values of its row that the operand wants of it, four lanes share a block,
// so the block's maximum takes two lane exchanges.
//
// Bound by the weight stream; see launch_fp8_few for the shape of a launch.
#include <algorithm>

#include "fp8.hpp"

namespace starkv {

namespace {
constexpr int FW = 4;                              // k blocks a wave loads at a time
constexpr int FEW_MAX_WAVES = 16;
struct E4m3In {};                                  // activations that are e4m3 with scales
}  // namespace

// X: _Float16 / __bf16 activations to quantise, or E4m3In; O: output type; NT: weight tiles (2: gate and up)
template <typename X, typename S, typename O, int NT>
__global__ __launch_bounds__(64 * FEW_MAX_WAVES) void fp8_few_kernel(const Fp8GemmArgs a) {
  constexpr bool Q = !__is_same(X, E4m3In);
  extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const int c = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int b0 = (int)((int64_t)a.kb * w / nw), b1 = (int)((int64_t)a.kb * (w + 1) / nw);
  const int last = (a.k - 1) >> 4;                 // the last 16-byte piece that holds a column
  const bool live = c < a.m;                       // this lane's activation row exists

  // lane (c, g): bytes 16 g .. and 16 (g + 4) .. of each block of row c
  const uint8_t* wrow[NT];
  const typename S::T* wsc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r0 = n0 + t * a.half;
    wrow[t] = a.w + (int64_t)min(r0 + c, a.n - 1) * a.ws;
    wsc[t] = (const typename S::T*)a.sw + (int64_t)(r0 >> 7) * a.swr;
  }
  const int xr = live ? c : 0;
  const uint8_t* xrow = (const uint8_t*)a.x + (int64_t)xr * a.xs * (Q ? 2 : 1);
  const typename S::T* xsc = (const typename S::T*)a.sx + (Q ? 0 : xr * a.sxr);

  floatx4 acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = floatx4{0.f, 0.f, 0.f, 0.f};
  float ss = 0.f;
  for (int b = b0; b < b1; b += FW) {
    uint4 wv[FW][NT][2];
#pragma unroll
    for (int u = 0; u < FW; ++u) {
      const int bb = min(b + u, b1 - 1);
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          wv[u][t][h] = *(const uint4*)(wrow[t] + (int64_t)min(bb * 8 + g + 4 * h, last) * 16);
    }
#pragma unroll
    for (int u = 0; u < FW; ++u) {
      const int bb = b + u;
      if (bb >= b1) break;
      uint4 xq[2];
      float sx;
      if constexpr (Q) {
        uint32_t xv[2][8] = {};
        if (live) {
#pragma unroll
          for (int h = 0; h < 2; ++h) load16<X>(xrow, bb * FP8_BLOCK + 16 * (g + 4 * h), a.k, a.vec_x != 0, xv[h]);
        }
        uint32_t m = max2_u16(amax16(xv[0]), amax16(xv[1]));
        m = max(m & 0xffffu, m >> 16);
        m = max(m, (uint32_t)__shfl_xor((int)m, 16, 64));
        m = max(m, (uint32_t)__shfl_xor((int)m, 32, 64));
        float inv;
        sx = scale_f32(block_scale<S>(mag_bits<X>(m), inv));
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          xq[h] = quant16<X>(xv[h], inv);
          if (a.rms) ss = sumsq16<X>(xv[h], ss);
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h) xq[h] = *(const uint4*)(xrow + (int64_t)min(bb * 8 + g + 4 * h, last) * 16);
        sx = scale_f32(xsc[(int64_t)bb * a.sxb]);
      }
      if ((bb + 1) * FP8_BLOCK > a.k) {            // bytes past column k: any value in either operand
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int nv = a.k - bb * FP8_BLOCK - 16 * (g + 4 * h);
          xq[h] = keep_bytes(xq[h], nv);
#pragma unroll
          for (int t = 0; t < NT; ++t) wv[u][t][h] = keep_bytes(wv[u][t][h], nv);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const intx8 wf = frag8(wv[u][t][0], wv[u][t][1]), xf = frag8(xq[0], xq[1]);
        const floatx4 p = __is_same(O, float) ? mfma8_exact(wf, xf)
                                              : mfma8(wf, xf, floatx4{0.f, 0.f, 0.f, 0.f}, E8_ONE, E8_ONE);
        const float sc = sx * scale_f32(wsc[t][(int64_t)bb * a.swb]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][e] = fmaf(p[e], sc, acc[t][e]);
      }
    }
  }

  // the waves' sums, in wave order
  floatx4* red = (floatx4*)lds;                    // [nw][NT][64]
  float* red_ss = (float*)(red + nw * NT * 64);    // [nw][16]
  if (a.rms) {
    ss += __shfl_xor(ss, 16, 64);
    ss += __shfl_xor(ss, 32, 64);
    if (g == 0) red_ss[w * 16 + c] = ss;
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) red[(w * NT + t) * 64 + lane] = acc[t];
  __syncthreads();
  if (w > 0) return;
  for (int v = 1; v < nw; ++v)
#pragma unroll
    for (int t = 0; t < NT; ++t) acc[t] += red[(v * NT + t) * 64 + lane];
  float r = 1.f;
  if (a.rms) {
    float tot = 0.f;
    for (int v = 0; v < nw; ++v) tot += red_ss[v * 16 + c];
    r = rsqrtf(tot / (float)a.k + a.rms_eps);
  }
  // lane (c, g) holds columns n0 + 4g .. + 3 of row c
  if (!live) return;
  const int col = n0 + 4 * g, nv = (NT == 2 ? a.half : a.n) - col;
  if (nv <= 0) return;
  O* o = (O*)a.out + c * a.os + col;
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = NT == 2 ? silu_mul_f32(r * acc[0][e], r * acc[NT - 1][e]) : r * acc[0][e];
  if (NT == 1 && a.res) {
    float t[4];
    load4<O>((const O*)a.res + c * a.rs + col, t, nv, a.vec_out != 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] += t[e];
  }
  store4<O>(o, v, nv, a.vec_out != 0);
}

template <typename X, typename S, typename O> static int launch_few_t(const Fp8GemmArgs& a, bool silu, hipStream_t st) {
  const int nt = silu ? 2 : 1;
  const int tiles = (int)ceil_div(silu ? a.half : a.n, 16);
  int nw = 8;
  nw = std::max(1, std::min(nw, a.kb));
  const size_t lds = (size_t)nw * (nt * 1024 + 64);
  if (silu) hipLaunchKernelGGL((fp8_few_kernel<X, S, O, 2>), dim3(tiles), dim3(64 * nw), lds, st, a);
  else hipLaunchKernelGGL((fp8_few_kernel<X, S, O, 1>), dim3(tiles), dim3(64 * nw), lds, st, a);
  return (int)hipGetLastError();
}
template <typename X, typename S> static int launch_few_o(const Fp8GemmArgs& a, int od, bool silu, hipStream_t st) {
  if (od == STARKV_F16) return launch_few_t<X, S, _Float16>(a, silu, st);
  if (od == STARKV_BF16) return launch_few_t<X, S, __bf16>(a, silu, st);
  return launch_few_t<X, S, float>(a, silu, st);
}
template <typename S> static int launch_few_s(const Fp8GemmArgs& a, int dt, int od, bool silu, hipStream_t st) {
  if (dt == STARKV_F16) return launch_few_o<_Float16, S>(a, od, silu, st);
  if (dt == STARKV_BF16) return launch_few_o<__bf16, S>(a, od, silu, st);
  return launch_few_o<E4m3In, S>(a, od, silu, st);
}

int launch_fp8_few(const Fp8GemmArgs& a, int dtype, int out_dtype, int scale_dtype, bool silu, hipStream_t st) {
  return scale_dtype == STARKV_E8M0 ? launch_few_s<ScaleE8>(a, dtype, out_dtype, silu, st)
                                    : launch_few_s<ScaleF32>(a, dtype, out_dtype, silu, st);
}

}  // namespace starkv
