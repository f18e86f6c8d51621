// Activations to e4m3 with a scale for each row's block of 128 columns.
//
//   a = max |x| of the block,  s = scale(a),  q = e4m3(x / s)
//
// Eight lanes hold a block, 16 values each (32 bytes read, 16 written per
// lane): the maximum is taken on packed 16-bit magnitudes, which order as
// integers, within the lane and then over three lane exchanges.  One pass,
// bound by HBM: 3 bytes move per value.  With power-of-two scales the
// quotient is exact, so each value is rounded once; fp32 scales take the
// product with the rounded reciprocal instead of a division per value.
//
// With `rscale` (the GEMM's RMS-normalised input) a workgroup takes one row
// (of more than 2^22 rows, every 2^22-th: a launch has less than 2^32 threads)
// and also sums its squares: rscale = rsqrt(mean x^2 + eps).
#include <algorithm>

#include "fp8.hpp"

namespace starkv {

namespace {
constexpr int QT = 256;                            // threads per workgroup
constexpr int QB = QT / 8;                         // blocks of 128 a workgroup holds at a time
constexpr int QROWS = 1 << 22;                     // workgroups of a launch that take rows
}  // namespace

// block `kb` of row `row`, this thread's 16 of its 128 values; returns them for the sum of squares
template <typename T, typename S>
__device__ inline void quant_block(const Fp8QuantArgs& a, int64_t row, int kb, int sub, uint32_t (&w)[8]) {
  const int c0 = kb * FP8_BLOCK + sub * 16;
  load16<T>((const uint8_t*)a.x + row * a.xs * 2, c0, a.k, a.vec != 0, w);
  uint32_t m = amax16(w);
  m = max(m & 0xffffu, m >> 16);
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  float inv;
  const typename S::T s = block_scale<S>(mag_bits<T>(m), inv);
  uint4 q = quant16<T, S>(w, inv, scale_f32(s));
  if (c0 + 16 > a.k) q = keep_bytes(q, a.k - c0);   // the row's padding is zero, also where the scale is NaN
  if (c0 < a.k) *(uint4*)(a.q + row * a.qs + c0) = q;
  if (sub == 0) ((typename S::T*)a.s)[row * a.ssr + kb * a.ssb] = s;
}

template <typename T, typename S>
__global__ __launch_bounds__(QT) void fp8_quant_kernel(const Fp8QuantArgs a) {
  // whole groups of eight lanes leave together
  const int64_t id = (int64_t)blockIdx.x * QB + (threadIdx.x >> 3);
  if (id >= (int64_t)a.rows * a.kb) return;
  const int64_t row = id / a.kb;
  uint32_t w[8];
  quant_block<T, S>(a, row, (int)(id - row * a.kb), threadIdx.x & 7, w);
}

template <typename T, typename S>
__global__ __launch_bounds__(QT) void fp8_quant_rms_kernel(const Fp8QuantArgs a) {
  __shared__ float parts[2][QT / 64];              // of this row and the next: one barrier a row
  int odd = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, odd ^= 1) {
    float* const part = parts[odd];
    float ss = 0.f;
    for (int kb = threadIdx.x >> 3; kb < a.kb; kb += QB) {
      uint32_t w[8];
      quant_block<T, S>(a, row, kb, threadIdx.x & 7, w);
      ss = sumsq16<T>(w, ss);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, 64);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = ss;
    __syncthreads();
    if (threadIdx.x == 0) {
      const float tot = (part[0] + part[1]) + (part[2] + part[3]);
      a.rscale[row] = rsqrtf(tot / (float)a.k + a.rms_eps);
    }
  }
}

template <typename T, typename S> static int launch_q(const Fp8QuantArgs& a, hipStream_t st) {
  if (a.rscale)
    hipLaunchKernelGGL((fp8_quant_rms_kernel<T, S>), dim3((unsigned)std::min(a.rows, QROWS)), dim3(QT), 0, st, a);
  else
    hipLaunchKernelGGL((fp8_quant_kernel<T, S>), dim3((unsigned)ceil_div((int64_t)a.rows * a.kb, QB)), dim3(QT), 0, st, a);
  return (int)hipGetLastError();
}

int launch_fp8_quant(const Fp8QuantArgs& a, int dtype, int scale_dtype, hipStream_t st) {
  if (a.rows == 0) return 0;
  if (dtype == STARKV_F16)
    return scale_dtype == STARKV_E8M0 ? launch_q<_Float16, ScaleE8>(a, st) : launch_q<_Float16, ScaleF32>(a, st);
  return scale_dtype == STARKV_E8M0 ? launch_q<__bf16, ScaleE8>(a, st) : launch_q<__bf16, ScaleF32>(a, st);
}

}  // namespace starkv
