// Decode attention of a batch whose sequences share a long prefix, on gfx950.
//
// The prefix's latents are the same for every sequence, so its keys are formed
// once and every query meets them, and P.V over it is one matrix product of all
// (sequence, head) rows with the shared value latent.  With q at a position
// behind the sequence's own first one and keys stored before rotation,
//     l[b, q, p] = c RoPE_P(q) . RoPE_p(X_k[p] B_k)      (p < P)
// is the logit of the distance that the two have (P positions lie between the
// prefix's first and the sequence's first).
//
// Layout (made once, prefix_pack): what a kernel reads with one instruction lies
// together.  K latents: [KV head][32 positions][chunk of 8 ranks][position][8];
// B_k^T: the MFMA operands of 32 x 16 dims x ranks as registers hold them; V
// latents: [8 positions][column][8], fp16.
//
// 1. prefix_logits_kernel: one wave takes 64 positions (a strip) of one KV head
//    at a time.  K^T = B_k^T X^T has a position in each lane and the RoPE pairs
//    (d, d + 64) in one lane, so it is rotated in registers and is, as fp16, the
//    A operand of K q^T as it stands.  There each lane holds 32 logits of one
//    query row: maximum and sum take one exchange of the wave's halves.  It
//    writes p = 2^(l - m) in fp16, l in units of log 2 and m the strip's maximum
//    rounded up to a whole number, and the strip's (m, sum).
// 2. prefix_pv_kernel: the product P V, split over strips.  A strip's rows are
//    brought to the row's maximum over the whole prefix by a factor
//    2^15 2^(m - the row's m) on the operand, a power of two, so exact: strips 2^-28
//    below the row's largest weight still keep all bits of fp16.  Each split's sums leave
//    divided by its weights' sum, in fp32: fp16 means of values that cancel, or that
//    are small beside the latent's largest, would be subnormal.
// 3. prefix_up_kernel adds the splits and, if the sequences have positions of
//    their own, the decode kernels' sums over those, in a fixed order, relative to
//    the larger of the two maxima, and multiplies them by U_v; prefix_finish_kernel
//    adds the products of its column slices.
//
// Range: queries are scaled by a power of two to [1, 2) per row, K latents by one
// that bounds every key by 2^15 (the prefix's by one for all, dense own ones by one
// for each position), bf16 value latents by one that brings the largest to [2^14,
// 2^15); each is undone in fp32.
//
// Roundings to fp16, as the decode kernels have them: the query after its turn, the
// key after its rotation, the rotation's table (2^-11 each, of the vectors' lengths: a
// logit's error, of which a matrix operand of 16 bits takes the first two in any case; two
// terms of each and a table of fp32 took the logits of 16 behind 32768 from 75 us to 93);
// weights (2^-11 of a term, once).  Statistics, sums and split means are
// fp32, and the up-projection takes its operand in terms that keep 22 bits or more (fp16:
// of what is above 2^-18 of a row's largest value, 2^-39 of it below).
#include <algorithm>
#include <type_traits>

#include "fp8.hpp"

namespace starkv {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float PX_LIFT = 15.f;                    // log2 of the largest factor of a strip

template <typename XT> __device__ inline floatx16 px_mfma(uint4 a, uint4 b, floatx16 c) {
  if constexpr (__is_same(XT, _Float16))
    return mfma_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c);
  else
    return mfma_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c);
}

__device__ inline float max_halves(float v) {
  auto x = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(x[0]), __int_as_float(x[1]));
}

// two fp32 values as fp16, nearest even (an instruction for both; left to itself the compiler joins each conversion to
// the sum before it, in a form that takes twice as long)
__device__ inline uint32_t px_pack(float a, float b) {
  uint32_t r;
  asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}

// position within a 32-position tile of MFMA row m: lane half hh of the result
// then holds positions 16 hh .. 16 hh + 15 in register order
__device__ inline int px_pos(int m) { return ((m >> 2) & 1) * 16 + (m >> 3) * 4 + (m & 3); }
// dim of row m of B_k^T tile w: pairs (d, d + 64) in one lane
__device__ inline int px_dim(int w, int m) {
  const int g = m >> 3;
  return (g >> 1) * 64 + 16 * w + 8 * (g & 1) + (m & 7);
}

// ---------------------------------------------------------------------------
// Packing
// ---------------------------------------------------------------------------
// largest magnitudes (as bits; a NaN is larger than infinity) of the K latents, B_k and the V latents
template <typename XT>
__global__ __launch_bounds__(256) void px_amax_kernel(const PrefixPackArgs a) {
  const int u = blockIdx.y;                        // K heads, B_k heads, V
  const bool is_v = u == 2 * a.Hkv, is_b = u >= a.Hkv && !is_v;
  const int h = is_v ? 0 : u % a.Hkv;
  const int64_t rows = is_b ? a.rank[h] : a.P;
  const int cols = is_v ? a.Rv : is_b ? HEAD_DIM : a.rank[h];
  const int64_t pitch = is_v ? a.v_ss : is_b ? a.bk_rs : a.kpitch[h];
  const XT* base = (const XT*)(is_v ? a.v : is_b ? a.bk : a.k) + (is_v ? 0 : is_b ? a.bkoff[h] : a.koff[h]);
  uint32_t m = 0;
  for (int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * 4)
    for (int c = 8 * (threadIdx.x & 63); c < cols; c += 512) {
      XT e[8];
      if (c + 8 <= cols) {
        __builtin_memcpy(e, base + r * pitch + c, 16);           // any alignment
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = base[r * pitch + min(c + j, cols - 1)];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(to_f32(e[j])) & 0x7fffffffu);
    }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  // one atomic a workgroup, and none where the maximum is there already: thousands on one word took 3 ms
  __shared__ uint32_t red[4];
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(red[0], red[1]), max(red[2], red[3]));
  uint32_t* to = (uint32_t*)a.head + 2 + (is_v ? 2 : is_b ? 1 : 0);
  if (threadIdx.x == 0 && m > __hip_atomic_load(to, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) atomicMax(to, m);
}

// 2^e, |e| <= 126
__device__ inline float pow2f(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

// exponent that brings a row's largest magnitude (its bits) to [2^14, 2^15)
__device__ inline int px_row_exp(uint32_t top) {
  const int e = (int)(top >> 23) - 141;
  return top == 0 || top >= 0x7f800000u ? 0 : max(e, -112);
}

// exponent by which K latents are scaled down: |K| <= bound = |X| |B_k| ranks sqrt 2 (the rotation) becomes at most 2^15
__device__ inline int px_k_exp(const PrefixPackArgs& a) {
  const float x = a.head[2], b = a.head[3];
  if (!(x < INFINITY) || !(b < INFINITY)) return 0;
  const double bound = (double)x * b * a.bound;
  int e = 0;
  if (bound > 32768.0) frexp(bound / 32768.0, &e);
  return min(e, 120);
}
// exponent by which bf16 V latents are scaled down
__device__ inline int px_v_exp(const PrefixPackArgs& a) {
  const float v = a.head[4];
  if (!(v < INFINITY) || v == 0.f || !a.scale_v) return 0;
  int e;
  frexpf(v, &e);                                   // v < 2^e
  return max(-120, min(e - 15, 120));
}

// 16-byte pieces of the packed K latents (unit = head), B_k operands (Hkv + head) and V latents (2 Hkv)
template <typename XT>
__global__ __launch_bounds__(256) void px_pack_kernel(const PrefixPackArgs a) {
  const int u = blockIdx.y;
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  if (u == 0 && i0 == 0) {
    a.head[0] = pow2f(px_k_exp(a));
    a.head[1] = pow2f(px_v_exp(a));
    a.head[5] = (float)((double)a.head[3] * a.bound);            // of |key| over |latent|
  }
  if (u < a.Hkv) {
    const int h = u, r = a.rank[h], nc = (r + 7) / 8;
    const float f = pow2f(-px_k_exp(a));
    const XT* x = (const XT*)a.k + a.koff[h];
    uint4* out = (uint4*)(a.xk + a.xkoff[h]);
    const int64_t n = (int64_t)a.strips * 2 * nc * 32;
    for (int64_t i = i0; i < n; i += step) {
      const int64_t tile = i / (nc * 32);
      const int c = (int)(i / 32 % nc), p = (int)(i & 31);
      const int64_t s = tile * 32 + p;
      XT e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = s < a.P && 8 * c + j < r ? (XT)(to_f32(x[s * a.kpitch[h] + 8 * c + j]) * f) : (XT)0.f;
      uint4 w;
      __builtin_memcpy(&w, e, 16);
      out[i] = w;
    }
  } else if (u < 2 * a.Hkv) {
    const int h = u - a.Hkv, r = a.rank[h], ks = (r + 15) / 16;
    const XT* b = (const XT*)a.bk + a.bkoff[h];
    uint4* out = (uint4*)(a.xb + a.xboff[h]);
    for (int64_t i = i0; i < ks * 4 * 64; i += step) {
      const int lane = (int)i & 63, w = (int)(i >> 6) & 3, k = (int)(i >> 8) * 16 + (lane >> 5) * 8;
      const int d = px_dim(w, lane & 31);
      XT e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = k + j < r ? b[(int64_t)(k + j) * a.bk_rs + d] : (XT)0.f;
      uint4 v;
      __builtin_memcpy(&v, e, 16);
      out[i] = v;
    }
  } else {
    const float f = pow2f(-px_v_exp(a));
    const XT* x = (const XT*)a.v;
    uint4* out = (uint4*)a.xv;
    const int64_t n = (int64_t)a.strips * 8 * a.Rvp;
    for (int64_t i = i0; i < n; i += step) {
      const int64_t s = i / a.Rvp * 8;
      const int c = (int)(i % a.Rvp);
      _Float16 e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // fp16 values as they are (f = 1: the product would change a NaN's bits only)
        e[j] = s + j < a.P && c < a.Rv ? (_Float16)(to_f32(x[(s + j) * a.v_ss + c]) * f) : (_Float16)0.f;
      }
      uint4 w;
      __builtin_memcpy(&w, e, 16);
      out[i] = w;
    }
  }
}

// ---------------------------------------------------------------------------
// Logits and weights
// ---------------------------------------------------------------------------
// A wave takes 32 positions at a time, and of them 32 dims: those keys are rotated
// and at once multiplied with the queries' same dims, so few registers are held and
// four waves a SIMD cover each other's waits.  KP: pairs of 16 ranks, so that the
// operand reads and products of a tile are one block of code (a test of the rank
// before each product left every one waiting for its own read).
//
// What bounds it is the vector unit: 32 heads x 32768 positions of 16 rows are
// 26 GFLOP of products, and 256 multiply-adds of the rotation (16 us of the 49), 64
// conversions and 32 exponentials a lane and strip; reads taken out as a trial it
// still took 44.  Two waves a SIMD with two tiles each took 61,
// the next keys formed under this rotation at three waves a SIMD 64.
//
// NG: groups of 32 query rows.  acc[g][r] += the logits of query row n of group g
// and positions px_pos, in register order, of the tile whose latents are in xf.
// STRAIGHT: the four tiles of dims as straight code (strips that follow one another;
// with own positions 64 us, rolled 70); rolled otherwise: a wave that runs through the code once or twice
// waited for its instructions (4 x 1024 own positions of 8 heads: 33 us straight, 13
// rolled).  `between` runs when xf has been used for the last time.
template <typename XT, int NG, int KP, bool STRAIGHT, typename F>
__device__ __forceinline__ void px_tile(const uint4* bl, const uint4* ql, const uint4* rope, const uint4 (&xf)[2 * KP],
                                        floatx16 (&acc)[NG], F between) {
  const int lane = threadIdx.x & 63;
  auto keys = [&](int w) {
    floatx16 kx = px_mfma<XT>(bl[w * 64 + lane], xf[0], floatx16{});
#pragma unroll
    for (int k = 1; k < 2 * KP; ++k) kx = px_mfma<XT>(bl[(k * 4 + w) * 64 + lane], xf[k], kx);
    return kx;
  };
  auto turn = [&](int w, const floatx16& kx, const uint4 (&rt)[2]) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const half8 t = __builtin_bit_cast(half8, rt[g]);
#pragma unroll
      for (int j = 0; j < 4; j += 2) {
        float l[2], u[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float k0 = kx[4 * g + j + i], k1 = kx[8 + 4 * g + j + i];
          const float c = (float)t[2 * (j + i)], sp = (float)t[2 * (j + i) + 1];
          // (k sin + 0 takes the table's fp16 as it is; a plain product would convert it first)
          l[i] = fmaf(c, k0, -fmaf(sp, k1, 0.f));
          u[i] = fmaf(c, k1, fmaf(sp, k0, 0.f));
        }
        lo[2 * g + j / 2] = px_pack(l[0], l[1]);
        hi[2 * g + j / 2] = px_pack(u[0], u[1]);
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      acc[g] = px_mfma<_Float16>(make_uint4(lo[0], lo[1], lo[2], lo[3]), ql[(g * 8 + 2 * w) * 64 + lane], acc[g]);
      acc[g] = px_mfma<_Float16>(make_uint4(hi[0], hi[1], hi[2], hi[3]), ql[(g * 8 + 2 * w + 1) * 64 + lane], acc[g]);
    }
  };
  if constexpr (STRAIGHT) {
    uint4 rt[2][2] = {{rope[0], rope[64]}, {}};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < 3) {
        rt[(w + 1) & 1][0] = rope[128 * (w + 1)];
        rt[(w + 1) & 1][1] = rope[128 * (w + 1) + 64];
      }
      const floatx16 kx = keys(w);
      if (w == 3) between();
      turn(w, kx, rt[w & 1]);
      __builtin_amdgcn_sched_barrier(0);           // loads hoisted across the dims' tiles cost registers
    }
  } else {
    uint4 next[2] = {rope[0], rope[64]};
#pragma unroll 1
    for (int w = 0; w < 4; ++w) {
      const uint4 rt[2] = {next[0], next[1]};
      const int more = w < 3 ? 128 * (w + 1) : 0;  // (the last reads the first again)
      next[0] = rope[more];
      next[1] = rope[more + 64];
      turn(w, keys(w), rt);
    }
    between();
  }
}

// B_k's operands of one head and the query rows r0 .. of it into LDS: the rows of (sequence, head of the group) from
// sequence b0 on, turned by (cos, sin), scaled to [1, 2) by a power of two each, in the operand's order
template <typename XT, int NG, int KP, int NW>
__device__ __forceinline__ void px_stage(const PrefixLogitsArgs& a, int h, int b0, int r0, int nr, float cs, float sn, float kmul, uint4* bl,
                                         uint4* ql, float* mul) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, ks_n = ((a.rank[h] + 7) / 8 + 1) / 2;
  const uint4* src = (const uint4*)(a.xb + a.xboff[h]);
  constexpr int RW = 32 * NG / NW;
  XT q0[RW], q1[RW];
#pragma unroll
  for (int i = 0; i < RW; ++i) {                   // (rows past the last repeat it)
    const int r = min(r0 + wave + NW * i, nr - 1);
    const XT* q = (const XT*)a.q + (b0 + r / a.gs) * a.q_sb + (h * a.gs + r % a.gs) * a.q_sh;
    q0[i] = q[lane];
    q1[i] = q[lane + 64];
  }
#pragma unroll
  for (int i = 0; i < 8 * KP / NW; ++i)
    bl[tid + 64 * NW * i] = tid + 64 * NW * i < ks_n * 256 ? src[tid + 64 * NW * i] : make_uint4(0, 0, 0, 0);
#pragma unroll
  for (int i = 0; i < RW; ++i) {
    const int r = wave + NW * i;
    const float x0 = to_f32(q0[i]), x1 = to_f32(q1[i]), y0 = x0 * cs - x1 * sn, y1 = x1 * cs + x0 * sn;
    const float m = wave_max(fmaxf(fabsf(y0), fabsf(y1)));
    const int e = m < INFINITY && m > 0.f ? min(max((int)(__float_as_uint(m) >> 23), 1), 253) - 127 : 0;
    const float f = pow2f(-e);
    _Float16* dst = (_Float16*)(ql + ((r >> 5) * 8 + 2 * (lane >> 4)) * 64 + ((lane >> 2) & 1) * 32 + (r & 31)) +
                    4 * ((lane >> 3) & 1) + (lane & 3);
    dst[0] = (_Float16)(y0 * f);
    dst[64 * 8] = (_Float16)(y1 * f);
    if (lane == 0) mul[r] = kmul * pow2f(e);
  }
}

// the largest over the workgroup's waves of each row's maximum, in wm[row]
template <int NG, int NW> __device__ __forceinline__ void px_row_max(const float (&top)[NG], float* wm) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
#pragma unroll
  for (int g = 0; g < NG; ++g)
    if (lane < 32) wm[wave * NG * 32 + g * 32 + lane] = top[g];
  __syncthreads();
  if (tid >= NG * 32) return;
  float m = wm[tid];
#pragma unroll
  for (int w = 1; w < NW; ++w) m = fmaxf(m, wm[w * NG * 32 + tid]);
  wm[tid] = m;
}

// Workgroup of eight waves = (chunk of strips, KV head, NG groups of rows), a wave a strip at a time.
template <typename XT, int NG, int KP>
__device__ __forceinline__ void px_prefix_logits(const PrefixLogitsArgs& a, uint8_t* lds, int chunk, int h) {
  constexpr int KS = 2 * KP;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, n = lane & 31;
  const int nr = a.B * a.gs, r0 = blockIdx.y * NG * 32, nc = (a.rank[h] + 7) / 8;
  uint4* bl = (uint4*)lds;                         // [k step][tile w][lane]
  uint4* ql = bl + KS * 256;                       // [group][4 tiles x 2 halves][lane]
  float* mul = (float*)(ql + NG * 512);            // [group * 32 + row]
  float* wm = mul + NG * 32;                       // [wave][group * 32 + row]
  const int at_lane = 32 * hh + px_pos(n), s_end = min(a.strips, (chunk + 1) * a.ch_len);
  int s = chunk * a.ch_len + wave;
  uint4 xf[KS];
  // (of an odd number of chunks the last one's upper lanes, and of an odd number of k steps the last, read what lies
  // behind: the packed B_k at most, and replaced by zeros)
  auto fetch = [&](int tile) {
    const uint4* x = (const uint4*)(a.xk + a.xkoff[h]) + (int64_t)tile * nc * 32;
#pragma unroll
    for (int k = 0; k < KS; ++k) xf[k] = x[at_lane + 64 * min(k, (nc - 1) / 2)];
  };
  auto clear = [&]() {
#pragma unroll
    for (int k = KS - 2; k < KS; ++k)
      if (2 * k + hh >= nc) xf[k] = make_uint4(0, 0, 0, 0);
  };
  if (s < s_end) fetch(2 * s);
  px_stage<XT, NG, KP, 8>(a, h, 0, r0, nr, a.cos_p[lane], a.sin_p[lane], a.scale * LOG2E * a.head[0], bl, ql, mul);
  __syncthreads();
  float top[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) top[g] = -INFINITY;
  for (; s < s_end; s += 8) {
    floatx16 acc[2][NG] = {};
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) {
      clear();
      px_tile<XT, NG, KP, true>(bl, ql, a.rope + (int64_t)(2 * s + pt) * 512 + at_lane, xf, acc[pt],
                                [&]() { fetch(pt == 0 ? 2 * s + 1 : 2 * min(s + 8, s_end - 1)); });
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float f = mul[g * 32 + n];
      const int rl = r0 + g * 32 + n, row = h * nr + rl;
      float m = -INFINITY;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[pt][g][r] *= f;
      if (64 * (s + 1) > a.P) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (64 * s + 32 * pt + 16 * hh + r >= a.P) acc[pt][g][r] = -INFINITY;
      }
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[pt][g][r]);
      // a whole power of two at or above the largest, so that a weight is rounded once: its strip's factor and their product
      // are exact.  A strip of -inf alone: weights 0
      m = __builtin_ceilf(fmaxf(max_halves(m), -3.0e38f));
      top[g] = fmaxf(top[g], m);
      float l = 0.f;
      uint8_t* o = (uint8_t*)(a.p + (int64_t)8 * s * a.Mp);
      uint32_t at = (uint32_t)(2 * hh * a.Mp + row) * 16;
      const uint32_t step = (uint32_t)a.Mp * 16;
      asm("" : "+v"(at));                          // formed here: kept across the loop its sums were spilled, and a reload waits for the fetch
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        half8 v[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float e = __builtin_amdgcn_exp2f(acc[pt][g][r] - m);
          l += e;
          v[r >> 3][r & 7] = (_Float16)e;
        }
        if (rl < nr) {
          *(uint4*)(o + (at + 4 * pt * step)) = __builtin_bit_cast(uint4, v[0]);
          *(uint4*)(o + (at + (4 * pt + 1) * step)) = __builtin_bit_cast(uint4, v[1]);
        }
      }
      l = add_halves(l);
      if (rl < nr && hh == 0) *(float2*)((uint8_t*)(a.stat + (int64_t)s * a.Mp) + (uint32_t)row * 8) = make_float2(m, l);
    }
  }
  px_row_max<NG, 8>(top, wm);
  if (tid < NG * 32 && r0 + tid < nr) a.cmax[(int64_t)chunk * a.Mp + (int64_t)h * nr + r0 + tid] = wm[tid];
}

// a logit under its mask; one of no finite number in a place that the mask takes out (at or below a type's lowest value) is
// not looked at
constexpr float PX_MASKED = -65504.f;
__device__ inline float px_mask(float l, float m) { return !(fabsf(l) < INFINITY) && m <= PX_MASKED ? -INFINITY : l + m; }

// The exponent by which a position's key may pass 2^15 (0: it does not): |key| <= |latent| per_latent, the latent's chunks in
// the lanes of both halves.  By the 2-norm in fp16 (one instruction for two ranks; the largest magnitude takes two), by
// the largest magnitude in bf16, whose squares pass fp32's range.  None for infinities and NaN.
template <typename XT, int KS> __device__ __forceinline__ int px_own_exp(const uint4 (&xf)[KS], float per_latent) {
  float size;
  if constexpr (__is_same(XT, _Float16)) {
    float s[2] = {};
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const kh2 x = __builtin_bit_cast(kh2, j == 0 ? xf[k].x : j == 1 ? xf[k].y : j == 2 ? xf[k].z : xf[k].w);
        s[j & 1] = __builtin_amdgcn_fdot2(x, x, s[j & 1], false);
      }
    size = __builtin_amdgcn_sqrtf(add_halves(s[0] + s[1]));
  } else {
    uint32_t big = 0;
#pragma unroll
    for (int k = 0; k < KS; ++k)
      big = max2_u16(max2_u16(max2_u16(big, xf[k].x & 0x7fff7fffu), xf[k].y & 0x7fff7fffu),
                     max2_u16(xf[k].z & 0x7fff7fffu, xf[k].w & 0x7fff7fffu));
    size = max_halves(fmaxf(__uint_as_float(big << 16), __uint_as_float(big & 0xffff0000u)));
  }
  const float bound = size * per_latent;
  return bound > 32768.f && bound < INFINITY ? min((int)(__float_as_uint(bound) >> 23) - 141, 100) : 0;
}
// The latents times 2^-e: exact in bf16.  fp16 ones may round at 2^-25, which beside the scaled latent (2^-12 or more: B_k
// below 2^16, 128 ranks) is less than the key's own rounding; twice half the way, as 2^-e itself may be too small a number.
template <typename XT, int KS> __device__ __forceinline__ void px_scale_down(uint4 (&xf)[KS], int e) {
  const float f = pow2f(-e), f1 = pow2f(-(e >> 1)), f2 = pow2f(-(e - (e >> 1)));
#pragma unroll
  for (int k = 0; k < KS; ++k) {
    uint32_t w[4] = {xf[k].x, xf[k].y, xf[k].z, xf[k].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (__is_same(XT, _Float16)) {
        const kh2 d1 = {(_Float16)f1, (_Float16)f1}, d2 = {(_Float16)f2, (_Float16)f2};
        w[j] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, w[j]) * d1 * d2);
      } else {                                     // (every product is a bf16 number: its low bits are zeros)
        w[j] = __float_as_uint(__uint_as_float(w[j] << 16) * f) >> 16 | (__float_as_uint(__uint_as_float(w[j] & 0xffff0000u) * f) & 0xffff0000u);
      }
    }
    xf[k] = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// A sequence's own positions: dense latents where they lie (rows at any alignment),
// the queries of one KV head and sequence, and the logits go out in fp32 as the
// decode's P.V kernels read them.  Workgroup = (sequence, KV head, chunk of tiles
// of 32 positions), a wave a tile at a time.
template <typename XT, int NG, int KP>
__device__ __forceinline__ void px_own_logits(const PrefixLogitsArgs& a, uint8_t* lds, int chunk, int h, int b) {
  constexpr int KS = 2 * KP;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, n = lane & 31;
  const int rank = a.rank[h], nc = (rank + 7) / 8, tail = rank & 7, pn = px_pos(n);
  uint4* bl = (uint4*)lds;
  uint4* ql = bl + KS * 256;
  float* mul = (float*)(ql + NG * 512);
  float* wm = mul + NG * 32;
  const int t_end = min((a.S + 31) / 32, (chunk + 1) * a.oc_len);
  int t = chunk * a.oc_len + wave;
  uint4 xf[KS];
  const XT* x = (const XT*)a.ox + b * a.ox_sb + a.oxoff[h];
  auto fetch = [&](int tile) {
    const XT* row = x + min(32 * tile + pn, a.S - 1) * a.oxpitch[h];
    if (KP == 1 && rank < 8) {
      XT e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = row[min(j, rank - 1)];
      __builtin_memcpy(&xf[0], e, 16);
      return;
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) __builtin_memcpy(&xf[k], row + min(8 * (2 * k + hh), rank - 8), 16);   // the last ends with the row
  };
  if (t < t_end) fetch(t);
  px_stage<XT, NG, KP, 8>(a, h, b, 0, a.gs, 1.f, 0.f, a.scale, bl, ql, mul);
  __syncthreads();
  const int last_pos = a.last_pos ? *a.last_pos : INT32_MAX;
  // a last chunk of fewer than 8 ranks: to its front (of a row of fewer in all the last was repeated), zeros behind
  const int sh = rank >= 8 && tail ? 16 * (8 - tail) : 0;
  const uint64_t ml = tail == 0 || tail >= 4 ? ~0ull : (1ull << (16 * tail)) - 1;
  const uint64_t mh = tail == 0 ? ~0ull : tail <= 4 ? 0 : (1ull << (16 * (tail - 4))) - 1;
  float top[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) top[g] = -INFINITY;
#pragma unroll 1
  for (; t < t_end; t += 8) {
#pragma unroll
    for (int k = KS - 2; k < KS; ++k) {
      uint64_t lo = xf[k].x | ((uint64_t)xf[k].y << 32), hi = xf[k].z | ((uint64_t)xf[k].w << 32);
      if (2 * k + hh == nc - 1) {
        if (sh >= 64) {
          lo = hi >> (sh - 64);
          hi = 0;
        } else if (sh) {
          lo = (lo >> sh) | (hi << (64 - sh));
          hi >>= sh;
        }
        lo &= ml;
        hi &= mh;
      }
      if (2 * k + hh >= nc) lo = hi = 0;
      xf[k] = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
    }
    // keys can pass fp16's range: each position's latent is scaled by what bounds its key (the prefix's were when it was
    // packed; by position, not by tile: what lies in masked places has no say in the others' bits)
    int e = px_own_exp<XT, KS>(xf, a.head[5]);
    const bool scaled = __any(e != 0);
    if (scaled) px_scale_down<XT, KS>(xf, e);
    floatx16 acc[NG] = {};
    px_tile<XT, NG, KP, false>(bl, ql, a.rope + (int64_t)t * 512 + 32 * hh + pn, xf, acc,
                               [&]() { if (t + 8 < t_end) fetch(t + 8); });
    const int p0 = 32 * t + 16 * hh;
    if (scaled) {                                  // undone: position 16 hh + r of the tile lies in lane (r / 4) * 8 + 4 hh + r % 4
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float up = pow2f(__shfl(e, (r >> 2) * 8 + 4 * hh + (r & 3), 64));
#pragma unroll
        for (int g = 0; g < NG; ++g) acc[g][r] *= up;
      }
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float f = mul[g * 32 + n];
      const int rl = g * 32 + n;
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[g][r] *= f;
      if (a.mask != nullptr && rl < a.gs) {
        const int64_t at = b * a.m_sb + (h * a.gs + rl) * a.m_sh;
        if (a.mask_dtype == STARKV_F32) {
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[g][r] = px_mask(acc[g][r], ((const float*)a.mask)[at + min(p0 + r, a.S - 1)]);
        } else {
          const uint16_t* mk = (const uint16_t*)a.mask + at;
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const uint16_t v = mk[min(p0 + r, a.S - 1)];
            acc[g][r] = px_mask(acc[g][r], a.mask_dtype == STARKV_F16 ? (float)__builtin_bit_cast(_Float16, v) : bf16_bits_to_float(v));
          }
        }
      }
      float m = -INFINITY;
      bool bad = false;                            // not a number: a maximum of +inf, by which the join makes the row NaN
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if (p0 + r > last_pos) acc[g][r] = -1e30f;
        if (p0 + r >= a.S) acc[g][r] = -INFINITY;
        m = fmaxf(m, acc[g][r]);
        bad |= !(acc[g][r] == acc[g][r]);
      }
      if (bad) m = INFINITY;
      top[g] = fmaxf(top[g], max_halves(m));
      if (rl < a.gs) {
        uint32_t at = (uint32_t)((h * a.gs + rl) * 32 + 16 * hh) * 4;
        asm("" : "+v"(at));                        // formed here, as above
        float4* o = (float4*)((uint8_t*)(a.ol + b * a.ol_sb + t * a.ol_st) + at);
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = make_float4(acc[g][4 * r], acc[g][4 * r + 1], acc[g][4 * r + 2], acc[g][4 * r + 3]);
      }
    }
  }
  px_row_max<NG, 8>(top, wm);
  if (tid < a.gs) a.own_max[((int64_t)b * a.Hq + h * a.gs + tid) * a.n_c1 + chunk] = wm[tid];
}

// f(a constant of the pairs of 16 ranks)
template <typename F> __device__ __forceinline__ void px_pairs(int rank, F f) {
  const int kp = (rank + 31) / 32;
  if (kp == 1) f(std::integral_constant<int, 1>());
  else if (kp == 2) f(std::integral_constant<int, 2>());
  else if (kp == 3) f(std::integral_constant<int, 3>());
  else f(std::integral_constant<int, 4>());
}

// The prefix's workgroups, then the sequences' own (NG and NO groups of rows), in one launch: neither fills the chip where
// prompts are short (8 behind 4099 positions: 11.8 + 11 us one after the other, 13; 4 behind 16384: 27, 20).  One group takes
// 128 registers, four waves a SIMD; two groups in one workgroup, which form the keys once for 64 rows, two.
template <typename XT, int NG, int NO>
__global__ __launch_bounds__(512, NG == 1 ? 4 : 2) void prefix_logits_kernel(const PrefixLogitsArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t px_lds[];
  const int bx = blockIdx.x, n_prefix = (a.n_ch + 7) / 8 * 8 * a.Hkv;
  if (bx < n_prefix) {
    // workgroups of one chunk of strips on one XCD: its L2 serves the rotation table to all heads
    const int chunk = (bx & 7) + 8 * ((bx >> 3) / a.Hkv), h = (bx >> 3) % a.Hkv;
    if (chunk < a.n_ch) px_pairs(a.rank[h], [&](auto kp) { px_prefix_logits<XT, NG, decltype(kp)::value>(a, px_lds, chunk, h); });
  } else if (blockIdx.y == 0) {
    const int at = bx - n_prefix, chunk = at % a.n_c1, h = at / a.n_c1 % a.Hkv, b = at / a.n_c1 / a.Hkv;
    px_pairs(a.rank[h], [&](auto kp) { px_own_logits<XT, NO, decltype(kp)::value>(a, px_lds, chunk, h, b); });
  }
}

// ---------------------------------------------------------------------------
// P V
// ---------------------------------------------------------------------------
// One 1 KB global -> LDS copy, 16 bytes per lane from base + off to LDS address
// `lds` + 16 lane (as inline assembly: the compiler then adds no waits of its own
// before reads of other stages; m0 needs a wait state before the copy).
__device__ inline void px_dma(const void* base, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "s"(lds) : "memory", "m0");
}
// all but the last N copies of this wave have landed, its LDS reads are done; then the workgroup's
template <int N> __device__ inline void px_stage_ready() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// Workgroup of 8 waves = (split of the strips, BM rows, 256 columns), wave (wm, wn)
// of WM x WN: RM x RN MFMA tiles, two waves a SIMD.  Steps of 32 positions go
// through a ring of four LDS stages, two of them in flight behind the one that is
// read ahead; the strips' factors are formed 56 strips at a time.  Weights are
// fp16 (2^-11 of each position's term, of either sign), factors powers of two, sums fp32.
// 512 rows x 32768 positions x 1640 columns: 71 us, 846 TFLOP/s of the tiles' products
// (1792 columns; 69 with means of 16 bits, 66 of those with every load from the caches):
// matrix unit and LDS reads, nearly level (operands read when they are needed, not a step
// ahead: 5 us more).
template <int RM, int RN, int WM, int WN>
__global__ __launch_bounds__(512, 2) void prefix_pv_kernel(const PrefixArgs a) {
  constexpr int BM = 32 * RM * WM, BN = 32 * RN * WN, RING = 4;
  constexpr int AI = (BM * 4 / 64 + 7) / 8, BI = BN * 4 / 64 / 8, NI = AI + BI;     // copies per wave and stage
  constexpr int STAGE = 4 * (BM + BN);             // 16-byte pieces
  constexpr int FS = 56;                           // strips whose factors lie in LDS (what the ring of BM 256 leaves)
  static_assert(2 * FS % RING == 0, "whole rounds of the ring");
  static_assert(WM * WN == 8 && BN == PX_BN, "eight waves");
  __shared__ uint4 ring[RING * STAGE];
  __shared__ _Float16 fac[FS * BM];                // [strip][row]
  __shared__ float row_f[BM];                      // 1 / sum
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hh = lane >> 5, n = lane & 31;
  const int wm = wave / WN, wn = wave % WN;
  // consecutive (split, tile) pairs on one XCD: a split's tiles share its weights and latents in that L2
  const int tiles = a.tiles_m * a.tiles_n, total = a.n_split * tiles, per = (total + 7) / 8;
  const int at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || at >= total) return;
  const int split = at / tiles, m0 = (at % tiles) / a.tiles_n * BM, n0 = (at % tiles) % a.tiles_n * BN;
  const int s0 = split * a.sp_len, s1 = min(a.strips, s0 + a.sp_len);

  // this wave's copies: instruction i brings 64 rows (columns) of one group of 8 positions
  uint32_t off[NI], dst[NI];
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint4*)ring;
#pragma unroll
  for (int i = 0; i < AI; ++i) {
    const int j = (wave * AI + i) % (BM / 16), k8 = j / (BM / 64), r = j % (BM / 64) * 64;   // fewer than 8: some twice
    off[i] = (uint32_t)(k8 * a.Mp + r + lane) * 16;
    dst[i] = lds0 + (k8 * BM + r) * 16;
  }
#pragma unroll
  for (int i = 0; i < BI; ++i) {
    const int j = wave * BI + i, k8 = j / (BN / 64), c = j % (BN / 64) * 64;
    off[AI + i] = (uint32_t)(k8 * a.Rvp + min(n0 + c + lane, a.Rvp - 1)) * 16;
    dst[AI + i] = lds0 + (4 * BM + k8 * BN + c) * 16;
  }
  const uint4* pa = a.p + (int64_t)8 * s0 * a.Mp + m0;
  const uint4* pb = a.xv + (int64_t)8 * s0 * a.Rvp;
  const int steps = 2 * (s1 - s0);
  int issued = 0;
  auto issue = [&](int slot) {                     // past the end the last step again (never read): the counts stay
#pragma unroll
    for (int i = 0; i < NI; ++i) px_dma(i < AI ? pa : pb, off[i], dst[i] + slot * STAGE * 16);
    if (++issued < steps) { pa += 4 * (int64_t)a.Mp; pb += 4 * (int64_t)a.Rvp; }
  };
  // the row's maximum; its strips' factors and sum, FS strips at a time, a row per thread
  float row_max = -INFINITY, lsum = 0.f;
  if (tid < BM) {
    const float* cm = a.cmax + m0 + tid;
#pragma unroll 8
    for (int c = 0; c < a.n_ch; ++c) row_max = fmaxf(row_max, cm[(int64_t)c * a.Mp]);
    if (split == 0 && n0 == 0) a.rmax[m0 + tid] = row_max;
  }
  auto factors = [&](int from) {
    if (tid >= BM) return;
    const float2* st = a.stat + (int64_t)(s0 + from) * a.Mp + m0 + tid;
#pragma unroll 8
    for (int s = 0; s < min(FS, s1 - s0 - from); ++s) {
      const float2 v = st[(int64_t)s * a.Mp];
      const _Float16 f = (_Float16)__builtin_amdgcn_exp2f((v.x - row_max) + PX_LIFT);
      fac[s * BM + tid] = f;
      lsum = fmaf(v.y, (float)f, lsum);
    }
  };
  factors(0);
  floatx16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[i][j] = floatx16{};
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // only copies are counted from here on
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) issue(i);
  // operands of 16 positions, read under the products of the 16 before them
  uint4 fa[2][RM], fb[2][RN];
  auto read = [&](int slot, int kk) {
    const uint4* sa = ring + slot * STAGE + (2 * kk + hh) * BM + (wm * RM) * 32 + n;
    const uint4* sb = ring + slot * STAGE + 4 * BM + (2 * kk + hh) * BN + (wn * RN) * 32 + n;
#pragma unroll
    for (int i = 0; i < RM; ++i) fa[kk][i] = sa[32 * i];
#pragma unroll
    for (int j = 0; j < RN; ++j) fb[kk][j] = sb[32 * j];
    __builtin_amdgcn_sched_barrier(0);
  };
  kh2 fc[RM];
  auto strip_factors = [&](int t) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const _Float16 f = fac[(t / 2 % FS) * BM + (wm * RM + i) * 32 + n];
      fc[i] = kh2{f, f};
    }
  };
  auto products = [&](int kk) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      uint4 v = fa[kk][i];
      v.x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.x) * fc[i]);
      v.y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.y) * fc[i]);
      v.z = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.z) * fc[i]);
      v.w = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.w) * fc[i]);
#pragma unroll
      for (int j = 0; j < RN; ++j) acc[i][j] = px_mfma<_Float16>(v, fb[kk][j], acc[i][j]);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  px_stage_ready<(RING - 2) * NI>();
  read(0, 0);
  strip_factors(0);
  for (int t0 = 0; t0 < steps; t0 += RING) {
    if (t0 && t0 % (2 * FS) == 0) {
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");        // the last ones have been used
      factors(t0 / 2);
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      strip_factors(t0);
    }
#pragma unroll
    for (int u = 0; u < RING; ++u) {
      if (t0 + u >= steps) break;
      px_stage_ready<(RING - 3) * NI>();           // the next step's copies; all reads of the one before have ended
      issue((u + RING - 1) % RING);
      read(u, 1);
      products(0);
      read((u + 1) % RING, 0);
      products(1);
      if (u % 2) strip_factors(t0 + u + 1);        // (stale where they are formed anew, and read again there)
    }
  }
  if (tid < BM) {
    row_f[tid] = lsum == 0.f ? 0.f : 1.f / lsum;
    if (n0 == 0) a.lsum[(int64_t)split * a.Mp + m0 + tid] = lsum;
  }
  px_stage_ready<0>();                             // the sums, and the last copies before the LDS is another's
  float* out = a.part + ((int64_t)split * a.M + m0) * a.Rvp + n0;
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int row = (wm * RM + i) * 32 + 8 * (r >> 2) + 4 * hh + (r & 3);
      const float inv = row_f[row];
      if (m0 + row >= a.M) continue;
#pragma unroll
      for (int j = 0; j < RN; ++j) {
        const int col = (wn * RN + j) * 32 + n;
        if (n0 + col < a.Rvp) out[(int64_t)row * a.Rvp + col] = acc[i][j][r] * inv;
      }
    }
}

// ---------------------------------------------------------------------------
// Join and up-projection
// ---------------------------------------------------------------------------
// 32 bits of fp32 in a type of 16: fp16 as a sum of two (of a row scaled to its
// largest value: 22 bits), bf16 as a sum of three (24 bits)
template <typename WT> struct PxTerms;
template <> struct PxTerms<_Float16> { static constexpr int N = 2; };
template <> struct PxTerms<__bf16> { static constexpr int N = 3; };

// threads: with few workgroups more of them to ask for the partials (4 behind 16384 positions: 11.3 us, 256 threads 15.0),
// with many fewer (batch 16 behind 32768: 25 of 256, 36 of 512)
template <int SC> constexpr int PX_UP_T = SC == 128 ? 256 : 512;

// Workgroup = (SC columns of the V rank, KV head, 32 of its rows (sequence, head of
// the group)).  It adds the rows' sums over the prefix's splits and over their own
// positions' chunks, in a fixed order, relative to the larger of the two maxima and
// divided by the weights' sum, and multiplies them by its columns of U_v: a term of
// the output, [column slice][row][128], that prefix_finish_kernel adds up.  Batch 16
// behind 32768: 18 splits of 512 rows, 61 MB, and own partials in 24 us; where workgroups
// are few (11 to 13 us) two to four batches of loads, one after another.
template <typename WT, int SC>
__global__ __launch_bounds__(PX_UP_T<SC>) void prefix_up_kernel(const PrefixArgs a) {
  constexpr int NT = PxTerms<WT>::N, PIECES = 32 * SC / 8, T = PX_UP_T<SC>, RL = T / 32;
  constexpr int PP = PIECES > T ? PIECES / T : 1, GR = PIECES > T ? 1 : T / PIECES;
  __shared__ uint4 op[NT][SC / 8][32];             // the rows' terms, [8 columns][row]
  __shared__ float wsplit[32][PX_MAX_SPLITS + 1], wown[32];
  __shared__ uint32_t row_top[32];
  __shared__ float red[GR > 1 ? (GR - 1) * PIECES : 1][8];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hh = lane >> 5, n = lane & 31;
  const int j0 = blockIdx.x * SC, h = blockIdx.y, nr = a.B * a.gs, r0 = blockIdx.z * 32, rows = min(32, nr - r0);
  // 32 dims of U_v of each of the first four waves: lane n one, 8 columns a piece
  uint4 uf[SC / 16];
  const WT* u = (const WT*)a.uv + (int64_t)(h * HEAD_DIM + 32 * (wave & 3) + n) * a.uv_rs;
#pragma unroll
  for (int k = 0; k < SC / 16; ++k) {
    const int c = j0 + 16 * k + 8 * hh;
    if (c + 8 <= a.Rv) {
      __builtin_memcpy(&uf[k], u + c, 16);
    } else {
      WT e[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = c + i < a.Rv ? u[c + i] : (WT)0.f;
      __builtin_memcpy(&uf[k], e, 16);
    }
  }
  // the rows' weights, RL lanes a row
  {
    const int r = min(tid / RL, rows - 1), i0 = tid % RL, row = h * nr + r0 + r, b = (r0 + r) / a.gs, q = h * a.gs + (r0 + r) % a.gs;
    const int64_t bq = (int64_t)b * a.n_hg + (q >> 5);
    const float mp = a.rmax[row];
    float ms = -INFINITY;                          // in units of log 2, as the prefix's
    for (int c = i0; c < a.n_c1; c += RL) ms = fmaxf(ms, a.own_max[((int64_t)b * a.Hq + q) * a.n_c1 + c] * LOG2E);
    float lp = 0.f, lo = 0.f;
    for (int s = i0; s < a.n_split; s += RL) {
      const float l = a.lsum[(int64_t)s * a.Mp + row];
      wsplit[tid / RL][s] = l;
      lp += l;
    }
    const float* psum = a.own_sum + bq * a.n_c2 * 32 + (q & 31);
    for (int c = i0; c < a.n_c2; c += RL) lo += psum[(int64_t)c * 32];
#pragma unroll
    for (int o = RL / 2; o >= 1; o >>= 1) {
      ms = fmaxf(ms, __shfl_xor(ms, o, RL));
      lp += __shfl_xor(lp, o, RL);
      lo += __shfl_xor(lo, o, RL);
    }
    const float m = fmaxf(mp, ms);
    const float wp = __builtin_amdgcn_exp2f((mp - m) - PX_LIFT);
    // own positions without weight are not looked at (their sums may be NaN)
    const float wo = ms > -INFINITY ? __builtin_amdgcn_exp2f(ms - m) : 0.f;
    const float l = wo == 0.f ? lp * wp : lp * wp + lo * wo, inv = 1.f / l;
    for (int s = i0; s < a.n_split; s += RL) wsplit[tid / RL][s] *= a.head[1] * wp * inv;
    if (i0 == 0) {
      wown[tid / RL] = wo == 0.f ? 0.f : wo * inv;
      row_top[tid / RL] = 0;
      if (a.jmax && blockIdx.x == 0 && (tid / RL) < rows) {
        a.jmax[(int64_t)b * a.Hq + q] = m * (1.f / LOG2E);
        a.jsum[bq * 32 + (q & 31)] = l;
      }
    }
  }
  __syncthreads();
  // piece i of this thread: 8 columns (from 8 ec) of row er + i * T / (SC / 8), the splits grp, grp + GR, ...
  float v[PP][8] = {};
  const int e = tid % PIECES, grp = GR == 1 ? 0 : tid / PIECES, er = e / (SC / 8), ec = e % (SC / 8);
  constexpr int RS = T / (SC / 8);
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    const int r = er + i * RS, c = j0 + 8 * ec;
    if (r >= rows || c >= a.Rvp) continue;
    const int b = (r0 + r) / a.gs, q = h * a.gs + (r0 + r) % a.gs;
    const float* p = a.part + (int64_t)(h * nr + r0 + r) * a.Rvp + c;
    const int64_t step = (int64_t)a.M * a.Rvp;
    for (int s0 = grp; s0 < a.n_split; s0 += 8 * GR) {
      floatx4 x[8][2] = {};
#pragma unroll
      for (int g = 0; g < 8; ++g)
        if (s0 + GR * g < a.n_split) {
          const floatx4* from = (const floatx4*)(p + (s0 + GR * g) * step);
          x[g][0] = from[0];
          x[g][1] = from[1];
        }
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        if (s0 + GR * g >= a.n_split) break;
        const float f = wsplit[r][s0 + GR * g];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = fmaf(x[g][k >> 2][k & 3], f, v[i][k]);
      }
    }
    const float wo = wown[r];
    const int64_t bq = (int64_t)b * a.n_hg + (q >> 5);
    const float* psum = a.own_sum + bq * a.n_c2 * 32 + (q & 31);
#pragma unroll 4
    for (int s = grp; s < (wo == 0.f ? 0 : a.n_c2); s += GR) {
      const int64_t at = ((bq * a.n_c2 + s) * 32 + (q & 31)) * a.own_Rvp + c;
      if (a.own_part16) {
        const half8 x = *(const half8*)((const _Float16*)a.own_part + at);
        const float f = wo * psum[(int64_t)s * 32];
#pragma unroll
        for (int k = 0; k < 8; ++k) v[i][k] = fmaf((float)x[k], f, v[i][k]);
      } else {
        const floatx4* x = (const floatx4*)((const float*)a.own_part + at);
        const floatx4 lo = x[0], hi = x[1];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          v[i][k] = fmaf(lo[k], wo, v[i][k]);
          v[i][4 + k] = fmaf(hi[k], wo, v[i][4 + k]);
        }
      }
    }
  }
  if constexpr (GR > 1) {
    if (grp) {
#pragma unroll
      for (int k = 0; k < 8; ++k) red[(grp - 1) * PIECES + e][k] = v[0][k];
    }
    __syncthreads();
    if (!grp) {
      for (int g = 0; g < GR - 1; ++g)
#pragma unroll
        for (int k = 0; k < 8; ++k) v[0][k] += red[g * PIECES + e][k];
    }
  }
  // columns past the rank hold what their tiles left (the packed zeros' sums, or none at all of own positions)
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    uint32_t most = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (j0 + 8 * ec + k >= a.Rv) v[i][k] = 0.f;
      most = max(most, __float_as_uint(v[i][k]) & 0x7fffffffu);
    }
    if (__is_same(WT, _Float16) && grp == 0) atomicMax(&row_top[er + i * RS], most);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    if (grp) continue;
    const int r = er + i * RS;
    float f = 1.f;
    if constexpr (__is_same(WT, _Float16)) f = pow2f(-px_row_exp(row_top[r]));
    WT w[NT][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      float x = v[i][k] * f;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        w[t][k] = (WT)x;
        x -= (float)w[t][k];
      }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t) __builtin_memcpy(&op[t][ec][r], w[t], 16);
  }
  __syncthreads();
  if (wave >= 4) return;
  floatx16 acc = {};
#pragma unroll
  for (int k = 0; k < SC / 16; ++k)
#pragma unroll
    for (int t = NT - 1; t >= 0; --t) acc = px_mfma<WT>(op[t][2 * k + hh][n], uf[k], acc);
  float* out = a.ypart + (((int64_t)blockIdx.x * a.Hkv + h) * nr + r0) * HEAD_DIM + 32 * wave + n;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int row = 8 * (r >> 2) + 4 * hh + (r & 3);
    float f = 1.f;
    if constexpr (__is_same(WT, _Float16)) f = pow2f(px_row_exp(row_top[row]));
    if (row < rows) out[row * HEAD_DIM] = acc[r] * f;
  }
}

// whether element `at` of the mask leaves nothing of a position (as low as the lowest value of a type, or -inf)
__device__ inline bool px_masked(const PrefixArgs& a, int64_t at) {
  if (a.mask == nullptr) return false;
  if (a.mask_dtype == STARKV_F32) return ((const float*)a.mask)[at] <= PX_MASKED;
  const uint16_t v = ((const uint16_t*)a.mask)[at];
  return (a.mask_dtype == STARKV_F16 ? (float)__builtin_bit_cast(_Float16, v) : bf16_bits_to_float(v)) <= PX_MASKED;
}

// The output: the terms of the column slices added in order.  Of quantised own latents the logits' maxima pass over what is
// no number, and the join over the sums of own positions without weight: such a row (all its maxima -inf, or as far below the
// prefix as a finite mask or last_pos_device puts them) is looked through here, and NaN unless its mask takes them all out.
template <typename OT>
__global__ __launch_bounds__(256) void prefix_finish_kernel(const PrefixArgs a) {
  __shared__ int live[2], bad[2];
  const int half = threadIdx.x >> 7, row = min(blockIdx.x * 2 + half, a.M - 1), d = threadIdx.x & 127, nr = a.B * a.gs;
  const int h = row / nr, b = row % nr / a.gs, q = h * a.gs + row % a.gs;
  const float* p = a.ypart + (int64_t)row * HEAD_DIM + d;
  const int64_t step = (int64_t)a.M * HEAD_DIM;
  float s = 0.f;
#pragma unroll 8
  for (int i = 0; i < a.n_sl; ++i) s += p[i * step];
  if (a.n_c1 && a.oc_len == 0) {
    if (d == 0) live[half] = bad[half] = 0;
    __syncthreads();
    const float mp = a.rmax[row];
    for (int c = d; c < a.n_c1; c += 128) {        // (a weight that the join takes for 0 is 0 here)
      const float ms = a.own_max[((int64_t)b * a.Hq + q) * a.n_c1 + c] * LOG2E;
      if (ms > -INFINITY && __builtin_amdgcn_exp2f(ms - fmaxf(mp, ms)) != 0.f) live[half] = 1;
    }
    __syncthreads();
    if (!live[half]) {
#pragma unroll 8
      for (int t = d; t < a.S; t += 128) {
        const float l = a.ol[b * a.ol_sb + (t >> 5) * a.ol_st + q * 32 + (t & 31)];
        if (!(l == l) && !px_masked(a, (int64_t)b * a.m_sb + (int64_t)q * a.m_sh + t)) bad[half] = 1;
      }
    }
    __syncthreads();
    if (bad[half]) {
      s = NAN;
      if (a.jmax && d == 0) a.jsum[((int64_t)b * a.n_hg + (q >> 5)) * 32 + (q & 31)] = NAN;   // and every weight of the row
    }
  }
  if ((int)(blockIdx.x * 2 + half) < a.M) ((OT*)a.out)[b * a.o_sb + q * a.o_sh + d] = (OT)s;
}

}  // namespace

int launch_prefix_pack(const PrefixPackArgs& a, int dtype, hipStream_t st) {
  int e = launch_fill_i32((int*)a.head, 8, 0, st);
  if (e) return e;
  const dim3 rows((unsigned)std::min<int64_t>(ceil_div(std::max(a.P, 128), 32), 512), 2 * a.Hkv + 1);
  const dim3 pieces((unsigned)std::min<int64_t>((int64_t)a.strips * 4, 2048), 2 * a.Hkv + 1);
  if (dtype == STARKV_F16) {
    hipLaunchKernelGGL(px_amax_kernel<_Float16>, rows, dim3(256), 0, st, a);
    hipLaunchKernelGGL(px_pack_kernel<_Float16>, pieces, dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL(px_amax_kernel<__bf16>, rows, dim3(256), 0, st, a);
    hipLaunchKernelGGL(px_pack_kernel<__bf16>, pieces, dim3(256), 0, st, a);
  }
  return (int)hipGetLastError();
}

static size_t px_logits_lds(const PrefixLogitsArgs& a, int ng) { return (size_t)round_up(a.ks_max, 2) * 4096 + ng * (8192 + 32 * 4 * 9); }

template <typename XT> static void launch_logits(const PrefixLogitsArgs& a, bool own, hipStream_t st) {
  const int groups = (int)ceil_div((int64_t)a.B * a.gs, 32);
  const dim3 grid((unsigned)(round_up(a.n_ch, 8) * a.Hkv + (own ? a.B * a.Hkv * a.n_c1 : 0)), (unsigned)ceil_div(groups, groups == 1 ? 1 : PX_GROUPS));
  const size_t lds = px_logits_lds(a, groups == 1 ? 1 : PX_GROUPS);
  if (groups == 1) hipLaunchKernelGGL((prefix_logits_kernel<XT, 1, 1>), grid, dim3(512), lds, st, a);
  else if (a.gs <= 32) hipLaunchKernelGGL((prefix_logits_kernel<XT, PX_GROUPS, 1>), grid, dim3(512), lds, st, a);
  else hipLaunchKernelGGL((prefix_logits_kernel<XT, PX_GROUPS, 2>), grid, dim3(512), lds, st, a);
}
int launch_prefix_logits(const PrefixLogitsArgs& a, int dtype, bool own, hipStream_t st) {
  if (dtype == STARKV_F16) launch_logits<_Float16>(a, own, st);
  else launch_logits<__bf16>(a, own, st);
  return (int)hipGetLastError();
}

int launch_prefix_pv(const PrefixArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(8 * ceil_div((int64_t)a.n_split * a.tiles_m * a.tiles_n, 8)));
  if (a.bm == 256) hipLaunchKernelGGL((prefix_pv_kernel<2, 4, 4, 2>), grid, dim3(512), 0, st, a);
  else if (a.bm == 128) hipLaunchKernelGGL((prefix_pv_kernel<2, 2, 2, 4>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((prefix_pv_kernel<2, 1, 1, 8>), grid, dim3(512), 0, st, a);
  return (int)hipGetLastError();
}

template <typename WT> static void launch_up(const PrefixArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)a.n_sl, (unsigned)a.Hkv, (unsigned)ceil_div((int64_t)a.B * a.gs, 32));
  if (a.sc == 128) hipLaunchKernelGGL((prefix_up_kernel<WT, 128>), grid, dim3(PX_UP_T<128>), 0, st, a);
  else if (a.sc == 64) hipLaunchKernelGGL((prefix_up_kernel<WT, 64>), grid, dim3(PX_UP_T<64>), 0, st, a);
  else hipLaunchKernelGGL((prefix_up_kernel<WT, 32>), grid, dim3(PX_UP_T<32>), 0, st, a);
}
int launch_prefix_up(const PrefixArgs& a, int dtype, bool out_f32, hipStream_t st) {
  if (dtype == STARKV_F16) launch_up<_Float16>(a, st);
  else launch_up<__bf16>(a, st);
  const dim3 grid((unsigned)ceil_div(a.M, 2));
  if (out_f32) hipLaunchKernelGGL(prefix_finish_kernel<float>, grid, dim3(256), 0, st, a);
  else if (dtype == STARKV_F16) hipLaunchKernelGGL(prefix_finish_kernel<_Float16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(prefix_finish_kernel<__bf16>, grid, dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace starkv
