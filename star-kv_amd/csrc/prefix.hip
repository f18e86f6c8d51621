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
//    writes p = exp(l - strip maximum) in fp16, and the strip's (maximum, sum).
// 2. prefix_pv_kernel: the product P V, split over strips.  A strip's rows are
//    brought to the row's maximum over the whole prefix by a factor
//    2^15 exp(strip maximum - row maximum) on the operand: strips 2^-29 below the
//    row's largest weight still keep all bits of fp16.  Each split's sums leave
//    divided by its weights' sum, in fp16 (half of them: a mean of values up to
//    65504 that is rounded up stays finite).
// 3. prefix_join_kernel adds the splits and, if the sequences have positions of
//    their own, the decode kernels' sums over those, in a fixed order, relative to
//    the larger of the two maxima; the decode's up-projection ends the call.
//
// Range: queries are scaled by a power of two to [1, 2) per row, K latents by one
// that bounds every key by 2^15, bf16 value latents by one that brings the largest
// to [2^14, 2^15); each is undone in fp32.
#include <algorithm>

#include "common.hpp"

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

__device__ inline float px_wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
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
    for (int c = threadIdx.x & 63; c < cols; c += 64) m = max(m, __float_as_uint(to_f32(base[r * pitch + c])) & 0x7fffffffu);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, o, 64));
  if ((threadIdx.x & 63) == 0 && m) atomicMax((uint32_t*)a.head + 2 + (is_v ? 2 : is_b ? 1 : 0), m);
}

// 2^e, |e| <= 126
__device__ inline float pow2f(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }

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
template <typename XT>
__global__ __launch_bounds__(256, 2) void prefix_logits_kernel(const PrefixArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t px_lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hh = lane >> 5, n = lane & 31;
  // workgroups of one chunk of strips on one XCD: its L2 serves the rotation table to all heads
  const int bx = blockIdx.x, chunk = (bx & 7) + 8 * ((bx >> 3) / a.Hkv), h = (bx >> 3) % a.Hkv;
  if (chunk >= a.n_ch) return;
  const int nr = a.B * a.gs, r0 = blockIdx.y * PX_GROUPS * 32, ng = min(PX_GROUPS, (nr - r0 + 31) / 32);
  const int nc = a.nc[h], ks_n = (nc + 1) / 2;
  uint4* bl = (uint4*)px_lds;                      // [k step][tile w][lane]
  uint4* ql = bl + a.ks_max * 256;                 // [group][4 tiles x 2 halves][lane]
  float* mul = (float*)(ql + PX_GROUPS * 512);     // [group * 32 + row]
  float* wm = mul + PX_GROUPS * 32;                // [wave][group * 32 + row]
  {
    const uint4* src = (const uint4*)(a.xb + a.xboff[h]);
    for (int i = tid; i < ks_n * 256; i += 256) bl[i] = src[i];
  }
  // queries turned by P positions, scaled to [1, 2) by row, in the operand's order
  const float cs = a.cos_p[lane], sn = a.sin_p[lane], kmul = a.head[0];
  for (int r = wave; r < ng * 32; r += 4) {
    float y0 = 0.f, y1 = 0.f;
    if (r0 + r < nr) {
      const XT* q = (const XT*)a.q + (r0 + r) / a.gs * a.q_sb + (h * a.gs + (r0 + r) % a.gs) * a.q_sh;
      const float x0 = to_f32(q[lane]), x1 = to_f32(q[lane + 64]);
      y0 = x0 * cs - x1 * sn;
      y1 = x1 * cs + x0 * sn;
    }
    const float m = px_wave_max(fmaxf(fabsf(y0), fabsf(y1)));
    const int e = m < INFINITY && m > 0.f ? min(max((int)(__float_as_uint(m) >> 23), 1), 253) - 127 : 0;
    const float f = pow2f(-e);
    _Float16* dst = (_Float16*)(ql + ((r >> 5) * 8 + 2 * (lane >> 4)) * 64 + ((lane >> 2) & 1) * 32 + (r & 31)) +
                    4 * ((lane >> 3) & 1) + (lane & 3);
    dst[0] = (_Float16)(y0 * f);
    dst[64 * 8] = (_Float16)(y1 * f);
    if (lane == 0) mul[r] = a.scale_log2 * kmul * pow2f(e);
  }
  __syncthreads();

  float top[PX_GROUPS];
#pragma unroll
  for (int g = 0; g < PX_GROUPS; ++g) top[g] = -INFINITY;
  const int pn = px_pos(n);
  const int s_end = min(a.strips, (chunk + 1) * a.ch_len);
  for (int s = chunk * a.ch_len + wave; s < s_end; s += 4) {
    uint4 xf[2][8], kf[2][4][2];
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) {
      const uint4* x = (const uint4*)(a.xk + a.xkoff[h]) + (int64_t)(2 * s + pt) * nc * 32 + pn;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k < ks_n) {
          const int c = 2 * k + hh;
          xf[pt][k] = x[min(c, nc - 1) * 32];
          if (c >= nc) xf[pt][k] = make_uint4(0, 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      floatx16 acc[2] = {};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k < ks_n) {
          const uint4 b = bl[(k * 4 + w) * 64 + lane];
          acc[0] = px_mfma<XT>(b, xf[0][k], acc[0]);
          acc[1] = px_mfma<XT>(b, xf[1][k], acc[1]);
        }
      }
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        half8 lo, hi;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const half8 t = __builtin_bit_cast(half8, a.rope[((int64_t)(2 * s + pt) * 8 + 2 * w + g) * 64 + hh * 32 + pn]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float k0 = acc[pt][4 * g + j], k1 = acc[pt][8 + 4 * g + j], c = (float)t[2 * j], sp = (float)t[2 * j + 1];
            lo[4 * g + j] = (_Float16)(k0 * c - k1 * sp);
            hi[4 * g + j] = (_Float16)(k1 * c + k0 * sp);
          }
        }
        kf[pt][w][0] = __builtin_bit_cast(uint4, lo);
        kf[pt][w][1] = __builtin_bit_cast(uint4, hi);
      }
    }
#pragma unroll
    for (int g = 0; g < PX_GROUPS; ++g) {
      if (g >= ng) break;
      floatx16 acc[2] = {};
#pragma unroll
      for (int f = 0; f < 8; ++f) {
        const uint4 q = ql[(g * 8 + f) * 64 + lane];
        acc[0] = px_mfma<_Float16>(kf[0][f >> 1][f & 1], q, acc[0]);
        acc[1] = px_mfma<_Float16>(kf[1][f >> 1][f & 1], q, acc[1]);
      }
      const float f = mul[g * 32 + n];
      float m = -INFINITY;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[pt][r] *= f;
      if (64 * (s + 1) > a.P) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (64 * s + 32 * pt + 16 * hh + r >= a.P) acc[pt][r] = -INFINITY;
      }
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[pt][r]);
      m = fmaxf(max_halves(m), -3.0e38f);          // a strip of -inf alone: weights 0
      top[g] = fmaxf(top[g], m);
      float l = 0.f;
      uint4 p[4];
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        half8 v[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r >> 3][r & 7] = (_Float16)__builtin_amdgcn_exp2f(acc[pt][r] - m);
#pragma unroll
        for (int r = 0; r < 16; ++r) l += (float)v[r >> 3][r & 7];
        p[2 * pt] = __builtin_bit_cast(uint4, v[0]);
        p[2 * pt + 1] = __builtin_bit_cast(uint4, v[1]);
      }
      l = add_halves(l);
      const int rl = r0 + g * 32 + n;
      if (rl < nr) {
        const int64_t row = (int64_t)h * nr + rl;
        uint4* o = a.p + (int64_t)(8 * s + 2 * hh) * a.Mp + row;
        o[0] = p[0];
        o[a.Mp] = p[1];
        o[4 * (int64_t)a.Mp] = p[2];
        o[5 * (int64_t)a.Mp] = p[3];
        if (hh == 0) a.stat[(int64_t)s * a.Mp + row] = make_float2(m, l);
      }
    }
  }
  // the chunk's maximum of each row
#pragma unroll
  for (int g = 0; g < PX_GROUPS; ++g)
    if (g < ng && hh == 0) wm[wave * PX_GROUPS * 32 + g * 32 + n] = top[g];
  __syncthreads();
  for (int r = tid; r < ng * 32; r += 256) {
    if (r0 + r >= nr) continue;
    float m = wm[r];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, wm[w * PX_GROUPS * 32 + r]);
    a.cmax[(int64_t)chunk * a.Mp + (int64_t)h * nr + r0 + r] = m;
  }
}

// ---------------------------------------------------------------------------
// P V
// ---------------------------------------------------------------------------
// Workgroup = (split of the strips, 32 WM RM rows, 32 WN RN columns); wave (wm, wn)
// of WM x WN owns RM x RN MFMA tiles.
template <int RM, int RN, int WM, int WN>
__global__ __launch_bounds__(256, RM * RN >= 16 ? 1 : 2) void prefix_pv_kernel(const PrefixArgs a) {
  constexpr int BM = 32 * RM * WM, BN = 32 * RN * WN, AU = BM * 8 / 256, BU = BN * 8 / 256;
  static_assert(WM * WN == 4 && BN == PX_BN, "four waves");
  __shared__ uint4 sa[2][8 * BM], sb[2][8 * BN];
  __shared__ float row_f[BM];                      // row maximum, then 1 / (2 sum)
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hh = lane >> 5, n = lane & 31;
  const int wm = wave / WN, wn = wave % WN;
  // consecutive (split, tile) pairs on one XCD: a split's tiles share its weights and latents in that L2
  const int tiles = a.tiles_m * a.tiles_n, total = a.n_split * tiles, per = (total + 7) / 8;
  const int at = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if ((int)(blockIdx.x >> 3) >= per || at >= total) return;
  const int split = at / tiles, m0 = (at % tiles) / a.tiles_n * BM, n0 = (at % tiles) % a.tiles_n * BN;
  const int s0 = split * a.sp_len, s1 = min(a.strips, s0 + a.sp_len);

  const uint4* asrc[AU];
  const uint4* bsrc[BU];
#pragma unroll
  for (int u = 0; u < AU; ++u) asrc[u] = a.p + (int64_t)(8 * s0 + (tid + 256 * u) / BM) * a.Mp + m0 + (tid + 256 * u) % BM;
#pragma unroll
  for (int u = 0; u < BU; ++u)
    bsrc[u] = a.xv + (int64_t)(8 * s0 + (tid + 256 * u) / BN) * a.Rvp + min(n0 + (tid + 256 * u) % BN, a.Rvp - 1);
  uint4 ra[AU], rb[BU];
  auto fetch = [&]() {
#pragma unroll
    for (int u = 0; u < AU; ++u) { ra[u] = *asrc[u]; asrc[u] += 8 * (int64_t)a.Mp; }
#pragma unroll
    for (int u = 0; u < BU; ++u) { rb[u] = *bsrc[u]; bsrc[u] += 8 * (int64_t)a.Rvp; }
  };
  auto place = [&](int st) {
#pragma unroll
    for (int u = 0; u < AU; ++u) sa[st][tid + 256 * u] = ra[u];
#pragma unroll
    for (int u = 0; u < BU; ++u) sb[st][tid + 256 * u] = rb[u];
  };
  fetch();
  if (tid < BM) {
    float m = -INFINITY;
    for (int c = 0; c < a.n_ch; ++c) m = fmaxf(m, a.cmax[(int64_t)c * a.Mp + m0 + tid]);
    row_f[tid] = m;
    if (split == 0 && n0 == 0) a.rmax[m0 + tid] = m;
  }
  __syncthreads();
  float rmx[RM], lsum[RM];
  const float2* st_src[RM];
  float2 st[RM];
#pragma unroll
  for (int i = 0; i < RM; ++i) {
    const int r = (wm * RM + i) * 32 + n;
    rmx[i] = row_f[r];
    lsum[i] = 0.f;
    st_src[i] = a.stat + (int64_t)s0 * a.Mp + m0 + r;
    st[i] = *st_src[i];
  }
  floatx16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[i][j] = floatx16{};
  place(0);
  __syncthreads();
  for (int s = s0; s < s1; ++s) {
    const int cur = (s - s0) & 1;
    kh2 fac[RM];
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const _Float16 f = (_Float16)__builtin_amdgcn_exp2f((st[i].x - rmx[i]) + PX_LIFT);
      fac[i] = kh2{f, f};
      lsum[i] = fmaf(st[i].y, (float)f, lsum[i]);
    }
    const bool more = s + 1 < s1;
    if (more) {
      fetch();
#pragma unroll
      for (int i = 0; i < RM; ++i) { st_src[i] += a.Mp; st[i] = *st_src[i]; }
    }
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      uint4 fa[RM], fb[RN];
#pragma unroll
      for (int i = 0; i < RM; ++i) {
        const uint4 v = sa[cur][(2 * kk + hh) * BM + (wm * RM + i) * 32 + n];
        fa[i].x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.x) * fac[i]);
        fa[i].y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.y) * fac[i]);
        fa[i].z = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.z) * fac[i]);
        fa[i].w = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.w) * fac[i]);
      }
#pragma unroll
      for (int j = 0; j < RN; ++j) fb[j] = sb[cur][(2 * kk + hh) * BN + (wn * RN + j) * 32 + n];
#pragma unroll
      for (int i = 0; i < RM; ++i)
#pragma unroll
        for (int j = 0; j < RN; ++j) acc[i][j] = px_mfma<_Float16>(fa[i], fb[j], acc[i][j]);
    }
    if (more) {
      place(cur ^ 1);
      __syncthreads();
    }
  }
  __syncthreads();
  if (wn == 0 && hh == 0) {
#pragma unroll
    for (int i = 0; i < RM; ++i) {
      const int r = (wm * RM + i) * 32 + n;
      row_f[r] = lsum[i] == 0.f ? 0.f : 0.5f / lsum[i];
      if (n0 == 0) a.lsum[(int64_t)split * a.Mp + m0 + r] = lsum[i];
    }
  }
  __syncthreads();
  _Float16* out = a.part + ((int64_t)split * a.M + m0) * a.Rvp + n0;
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
        if (n0 + col < a.Rvp) out[(int64_t)row * a.Rvp + col] = (_Float16)(acc[i][j][r] * inv);
      }
    }
}

// ---------------------------------------------------------------------------
// Join: row (b, q)'s sums over the prefix's splits and over its own positions' chunks
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(256) void prefix_join_kernel(const PrefixArgs a) {
  const int row = blockIdx.x, nr = a.B * a.gs, h = row / nr, b = row % nr / a.gs, q = h * a.gs + row % a.gs;
  const int64_t bq = (int64_t)b * a.n_hg + (q >> 5);
  const float mp = a.rmax[row];
  float ms = -INFINITY;                            // in units of log 2, as the prefix's
  for (int c = 0; c < a.n_c1; ++c) ms = fmaxf(ms, a.own_max[((int64_t)b * a.Hq + q) * a.n_c1 + c] * LOG2E);
  const float m = fmaxf(mp, ms);
  const float wp = __builtin_amdgcn_exp2f(mp - m - PX_LIFT);
  const float wo = ms > -INFINITY ? __builtin_amdgcn_exp2f(ms - m) : 0.f;
  const float vmul = 2.f * a.head[1];
  const float* psum = a.own_sum + (bq * a.n_c2) * 32 + (q & 31);
  const int n_own = wo > 0.f ? a.n_c2 : 0;         // own positions without weight are not looked at (their sums may be NaN)
  if (threadIdx.x == 0) {
    float l = 0.f, o = 0.f;
    for (int s = 0; s < a.n_split; ++s) l += a.lsum[(int64_t)s * a.Mp + row];
    for (int c = 0; c < n_own; ++c) o += psum[(int64_t)c * 32];
    a.jsum[bq * 32 + (q & 31)] = n_own ? l * wp + o * wo : l * wp;
    if (a.jmax) a.jmax[(int64_t)b * a.Hq + q] = m * (1.f / LOG2E);
  }
  for (int c0 = 4 * threadIdx.x; c0 < a.Rvp; c0 += 1024) {
    float v[4] = {};
    const _Float16* p = a.part + (int64_t)row * a.Rvp + c0;
#pragma unroll 8
    for (int s = 0; s < a.n_split; ++s) {
      const half4 e = *(const half4*)(p + (int64_t)s * a.M * a.Rvp);
      const float f = a.lsum[(int64_t)s * a.Mp + row];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = fmaf((float)e[i], f, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= wp * vmul;
    for (int c = 0; c < n_own; ++c) {
      const int64_t at = ((bq * a.n_c2 + c) * 32 + (q & 31)) * a.own_Rvp + c0;
      float f = wo;
      if (a.own_part16) f *= psum[(int64_t)c * 32];
#pragma unroll
      for (int i = 0; i < 4; ++i)
        v[i] = fmaf(a.own_part16 ? (float)((const _Float16*)a.own_part)[at + i] : ((const float*)a.own_part)[at + i], f, v[i]);
    }
    *(float4*)(a.jpart + (bq * 32 + (q & 31)) * a.Rvp + c0) = make_float4(v[0], v[1], v[2], v[3]);
  }
}

}  // namespace

int launch_prefix_pack(const PrefixPackArgs& a, int dtype, hipStream_t st) {
  int e = launch_fill_i32((int*)a.head, 8, 0, st);
  if (e) return e;
  const dim3 rows((unsigned)std::min<int64_t>(ceil_div(std::max(a.P, 128), 4), 512), 2 * a.Hkv + 1);
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

int launch_prefix(const PrefixArgs& a, int dtype, hipStream_t st) {
  const int groups = (int)ceil_div((int64_t)a.B * a.gs, 32);
  const size_t lds = (size_t)a.ks_max * 4096 + PX_GROUPS * 8192 + PX_GROUPS * 32 * 4 * 5;
  const dim3 g1((unsigned)(round_up(a.n_ch, 8) * a.Hkv), (unsigned)ceil_div(groups, PX_GROUPS));
  if (dtype == STARKV_F16) hipLaunchKernelGGL(prefix_logits_kernel<_Float16>, g1, dim3(256), lds, st, a);
  else hipLaunchKernelGGL(prefix_logits_kernel<__bf16>, g1, dim3(256), lds, st, a);
  const dim3 g2((unsigned)(8 * ceil_div((int64_t)a.n_split * a.tiles_m * a.tiles_n, 8)));
  if (a.bm == 256) hipLaunchKernelGGL((prefix_pv_kernel<4, 4, 2, 2>), g2, dim3(256), 0, st, a);
  else if (a.bm == 128) hipLaunchKernelGGL((prefix_pv_kernel<2, 4, 2, 2>), g2, dim3(256), 0, st, a);
  else if (a.bm == 64) hipLaunchKernelGGL((prefix_pv_kernel<2, 2, 1, 4>), g2, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((prefix_pv_kernel<1, 2, 1, 4>), g2, dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

int launch_prefix_join(const PrefixArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(prefix_join_kernel, dim3((unsigned)a.M), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace starkv
