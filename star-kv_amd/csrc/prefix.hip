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
// NG: groups of 32 query rows per workgroup.  A tile of B_k^T (32 dims) at a
// time: its keys are rotated and at once multiplied with the queries' same dims,
// so no more than a tile's keys are held; the next tile's rotation and the next
// strip's latents are asked for ahead.
// OWN: a sequence's own positions instead: dense latents where they lie (rows at
// any alignment), the queries of one KV head and sequence, and the logits go out
// in fp32 as the decode's P.V kernels read them.
template <typename XT, int NG, bool OWN>
__device__ __forceinline__ void px_logits(const PrefixArgs& a, uint8_t* px_lds, int bx) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, hh = lane >> 5, n = lane & 31;
  int chunk, h, b = 0;
  if constexpr (OWN) {
    chunk = bx % a.n_c1;
    h = bx / a.n_c1 % a.Hkv;
    b = bx / a.n_c1 / a.Hkv;
  } else {
    // workgroups of one chunk of strips on one XCD: its L2 serves the rotation table to all heads
    chunk = (bx & 7) + 8 * ((bx >> 3) / a.Hkv);
    h = (bx >> 3) % a.Hkv;
    if (chunk >= a.n_ch) return;
  }
  const int nr = OWN ? a.gs : a.B * a.gs, r0 = OWN ? 0 : blockIdx.y * NG * 32;
  const int rank = a.rank[h], nc = (rank + 7) / 8, ks_n = (nc + 1) / 2;
  const int len = OWN ? a.S : a.P, strips = OWN ? (a.S + PX_STRIP - 1) / PX_STRIP : a.strips;
  const int per = OWN ? a.oc_len : a.ch_len;
  uint4* bl = (uint4*)px_lds;                      // [k step][tile w][lane]
  uint4* ql = bl + a.ks_max * 256;                 // [group][4 tiles x 2 halves][lane]
  float* mul = (float*)(ql + NG * 512);            // [group * 32 + row]
  float* wm = mul + NG * 32;                       // [wave][group * 32 + row]
  const int pn = px_pos(n), s_end = min(strips, (chunk + 1) * per);
  int s = chunk * per + wave;
  uint4 xf[2][8];
  const uint4* xk = (const uint4*)(a.xk + a.xkoff[h]) + pn;
  const XT* xo = OWN ? (const XT*)a.ox + b * a.ox_sb + a.oxoff[h] : nullptr;
  const int64_t xpitch = OWN ? a.oxpitch[h] : 0;
  auto fetch = [&](int at) {
#pragma unroll
    for (int pt = 0; pt < 2; ++pt) {
      const XT* row = OWN ? xo + min(64 * at + 32 * pt + pn, len - 1) * xpitch : nullptr;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k < ks_n) {
          const int c = min(2 * k + hh, nc - 1);
          if constexpr (!OWN) {
            xf[pt][k] = xk[((int64_t)(2 * at + pt) * nc + c) * 32];
          } else if (rank >= 8) {                  // a last chunk of fewer ranks ends with the row
            __builtin_memcpy(&xf[pt][k], row + min(8 * c, rank - 8), 16);
          } else {
            XT e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = row[min(j, rank - 1)];
            __builtin_memcpy(&xf[pt][k], e, 16);
          }
        }
      }
    }
  };
  if (s < s_end) fetch(s);
  {
    const uint4* src = (const uint4*)(a.xb + a.xboff[h]);
    for (int i = tid; i < ks_n * 256; i += 256) bl[i] = src[i];
  }
  // queries (the prefix's: turned by P positions), scaled to [1, 2) by row, in the operand's order
  const float cs = OWN ? 1.f : a.cos_p[lane], sn = OWN ? 0.f : a.sin_p[lane];
  const float kmul = OWN ? a.scale : a.scale * LOG2E * a.head[0];
  for (int r = wave; r < NG * 32; r += 4) {
    float y0 = 0.f, y1 = 0.f;
    if (r0 + r < nr) {
      const int qb = OWN ? b : (r0 + r) / a.gs, qg = OWN ? r : (r0 + r) % a.gs;
      const XT* q = (const XT*)a.q + qb * a.q_sb + (h * a.gs + qg) * a.q_sh;
      const float x0 = to_f32(q[lane]), x1 = to_f32(q[lane + 64]);
      y0 = OWN ? x0 : x0 * cs - x1 * sn;
      y1 = OWN ? x1 : x1 * cs + x0 * sn;
    }
    const float m = px_wave_max(fmaxf(fabsf(y0), fabsf(y1)));
    const int e = m < INFINITY && m > 0.f ? min(max((int)(__float_as_uint(m) >> 23), 1), 253) - 127 : 0;
    const float f = pow2f(-e);
    _Float16* dst = (_Float16*)(ql + ((r >> 5) * 8 + 2 * (lane >> 4)) * 64 + ((lane >> 2) & 1) * 32 + (r & 31)) +
                    4 * ((lane >> 3) & 1) + (lane & 3);
    dst[0] = (_Float16)(y0 * f);
    dst[64 * 8] = (_Float16)(y1 * f);
    if (lane == 0) mul[r] = kmul * pow2f(e);
  }
  __syncthreads();

  float top[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) top[g] = -INFINITY;
  const int last_pos = OWN && a.last_pos ? *a.last_pos : INT32_MAX;
  const int tail = OWN ? rank & 7 : 0;             // ranks of a last chunk that is not whole
  for (; s < s_end; s += 4) {
    floatx16 acc[NG][2] = {};
    // the last k step: a partial chunk's ranks to its front, zeros behind the rank
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k != ks_n - 1) continue;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        if (OWN && tail) {
          const uint4 v = xf[pt][k];
          uint64_t lo = v.x | ((uint64_t)v.y << 32), hi = v.z | ((uint64_t)v.w << 32);
          if (rank >= 8) {
            const int sh = 16 * (8 - tail);
            lo = sh >= 64 ? hi >> (sh - 64) : (lo >> sh) | (hi << (64 - sh));
            hi = sh >= 64 ? 0 : hi >> sh;
          }
          // (of a row of fewer than 8 ranks the last was repeated)
          const uint64_t ml = tail >= 4 ? ~0ull : (1ull << (16 * tail)) - 1, mh = tail <= 4 ? 0 : (1ull << (16 * (tail - 4))) - 1;
          lo &= ml;
          hi &= mh;
          if (min(2 * k + hh, nc - 1) == nc - 1)
            xf[pt][k] = make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
        }
        if (2 * k + hh >= nc) xf[pt][k] = make_uint4(0, 0, 0, 0);
      }
    }
    // bf16 keys of own positions can pass fp16's range: scaled by what bounds them (the prefix's were when it was packed)
    int ke = 0;
    if constexpr (OWN && __is_same(XT, __bf16)) {
      uint32_t big = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k >= ks_n) continue;
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
          big = max2_u16(max2_u16(max2_u16(big, xf[pt][k].x & 0x7fff7fffu), xf[pt][k].y & 0x7fff7fffu),
                         max2_u16(xf[pt][k].z & 0x7fff7fffu, xf[pt][k].w & 0x7fff7fffu));
      }
      const float bound = px_wave_max(fmaxf(__uint_as_float(big << 16), __uint_as_float(big & 0xffff0000u))) * a.head[5];
      if (bound > 32768.f && bound < INFINITY) ke = min((int)(__float_as_uint(bound) >> 23) - 141, 100);
      ke = __builtin_amdgcn_readfirstlane(ke);
    }
    const float kdown = pow2f(-ke);
    uint4 rt[2][2][2];
    auto turn = [&](int w) {
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int g = 0; g < 2; ++g)
          rt[w & 1][pt][g] = a.rope[((int64_t)min(2 * s + pt, (len - 1) >> 5) * 8 + 2 * w + g) * 64 + hh * 32 + pn];
    };
    turn(0);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      if (w < 3) turn(w + 1);
      floatx16 kx[2] = {};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (k < ks_n) {
          const uint4 bf = bl[(k * 4 + w) * 64 + lane];
          kx[0] = px_mfma<XT>(bf, xf[0][k], kx[0]);
          kx[1] = px_mfma<XT>(bf, xf[1][k], kx[1]);
        }
      }
      if (OWN && ke) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int r = 0; r < 16; ++r) kx[pt][r] *= kdown;
      }
      uint4 kf[2][2];
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        half8 lo, hi;
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const half8 t = __builtin_bit_cast(half8, rt[w & 1][pt][g]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float k0 = kx[pt][4 * g + j], k1 = kx[pt][8 + 4 * g + j], c = (float)t[2 * j], sp = (float)t[2 * j + 1];
            lo[4 * g + j] = (_Float16)(k0 * c - k1 * sp);
            hi[4 * g + j] = (_Float16)(k1 * c + k0 * sp);
          }
        }
        kf[pt][0] = __builtin_bit_cast(uint4, lo);
        kf[pt][1] = __builtin_bit_cast(uint4, hi);
      }
#pragma unroll
      for (int g = 0; g < NG; ++g)
#pragma unroll
        for (int f = 0; f < 2; ++f) {
          const uint4 q = ql[(g * 8 + 2 * w + f) * 64 + lane];
          acc[g][0] = px_mfma<_Float16>(kf[0][f], q, acc[g][0]);
          acc[g][1] = px_mfma<_Float16>(kf[1][f], q, acc[g][1]);
        }
      __builtin_amdgcn_sched_barrier(0);           // loads hoisted across tiles cost a hundred spills
    }
    const int cur = s;
    if (s + 4 < s_end) fetch(s + 4);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float f = OWN ? mul[g * 32 + n] * pow2f(ke) : mul[g * 32 + n];
      const int rl = r0 + g * 32 + n, p0 = 64 * cur + 16 * hh;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[g][pt][r] *= f;
      if (OWN && a.mask != nullptr && rl < nr) {
        const int64_t at = b * a.m_sb + (h * a.gs + rl) * a.m_sh;
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[g][pt][r] += load_elem_f32(a.mask, a.mask_dtype, at + min(p0 + 32 * pt + r, len - 1));
      }
      if (64 * (cur + 1) > min(len, last_pos + (last_pos < INT32_MAX ? 1 : 0))) {
#pragma unroll
        for (int pt = 0; pt < 2; ++pt)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (p0 + 32 * pt + r > last_pos) acc[g][pt][r] = -1e30f;
            if (p0 + 32 * pt + r >= len) acc[g][pt][r] = -INFINITY;
          }
      }
      float m = -INFINITY;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[g][pt][r]);
      m = max_halves(m);
      if constexpr (OWN) {
        top[g] = fmaxf(top[g], m);
        if (rl < nr) {
#pragma unroll
          for (int pt = 0; pt < 2; ++pt) {
            float4* o = (float4*)(a.ol + b * a.ol_sb + (2 * cur + pt) * a.ol_st + (h * a.gs + rl) * 32 + 16 * hh);
#pragma unroll
            for (int r = 0; r < 4; ++r) o[r] = make_float4(acc[g][pt][4 * r], acc[g][pt][4 * r + 1], acc[g][pt][4 * r + 2], acc[g][pt][4 * r + 3]);
          }
        }
        continue;
      }
      m = fmaxf(m, -3.0e38f);                      // a strip of -inf alone: weights 0
      top[g] = fmaxf(top[g], m);
      float l = 0.f;
      const int64_t row = (int64_t)h * nr + rl;
      uint4* o = a.p + (int64_t)(8 * cur + 2 * hh) * a.Mp + row;
#pragma unroll
      for (int pt = 0; pt < 2; ++pt) {
        half8 v[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r >> 3][r & 7] = (_Float16)__builtin_amdgcn_exp2f(acc[g][pt][r] - m);
#pragma unroll
        for (int r = 0; r < 16; ++r) l += (float)v[r >> 3][r & 7];
        if (rl < nr) {
          o[4 * pt * (int64_t)a.Mp] = __builtin_bit_cast(uint4, v[0]);
          o[(4 * pt + 1) * (int64_t)a.Mp] = __builtin_bit_cast(uint4, v[1]);
        }
      }
      l = add_halves(l);
      if (rl < nr && hh == 0) a.stat[(int64_t)cur * a.Mp + row] = make_float2(m, l);
    }
  }
  // the chunk's maximum of each row
#pragma unroll
  for (int g = 0; g < NG; ++g)
    if (hh == 0) wm[wave * NG * 32 + g * 32 + n] = top[g];
  __syncthreads();
  for (int r = tid; r < NG * 32; r += 256) {
    if (r0 + r >= nr) continue;
    float m = wm[r];
#pragma unroll
    for (int w = 1; w < 4; ++w) m = fmaxf(m, wm[w * NG * 32 + r]);
    if constexpr (OWN) a.own_max[((int64_t)b * a.Hq + h * a.gs + r) * a.n_c1 + chunk] = m;
    else a.cmax[(int64_t)chunk * a.Mp + (int64_t)h * nr + r0 + r] = m;
  }
}

// The first own_wg workgroups: own positions (while they wait for their few latents the prefix's compute).
template <typename XT, int NG>
__global__ __launch_bounds__(256, 2) void prefix_logits_kernel(const PrefixArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint8_t px_lds[];
  const int bx = blockIdx.x;
  if (bx >= a.own_wg) px_logits<XT, NG, false>(a, px_lds, bx - a.own_wg);
  else if (blockIdx.y == 0) px_logits<XT, NG, true>(a, px_lds, bx);
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
// through a ring of four LDS stages, three of them in flight.  The factors of the
// split's strips are formed once, before the loop.
template <int RM, int RN, int WM, int WN>
__global__ __launch_bounds__(512, 2) void prefix_pv_kernel(const PrefixArgs a) {
  constexpr int BM = 32 * RM * WM, BN = 32 * RN * WN, RING = 4;
  constexpr int AI = (BM * 4 / 64 + 7) / 8, BI = BN * 4 / 64 / 8, NI = AI + BI;     // copies per wave and stage
  constexpr int STAGE = 4 * (BM + BN);             // 16-byte pieces
  static_assert(WM * WN == 8 && BN == PX_BN, "eight waves");
  __shared__ uint4 ring[RING * STAGE];
  __shared__ _Float16 fac[PX_SPLIT_STRIPS * BM];   // [strip][row]
  __shared__ float row_f[BM];                      // 1 / (2 sum)
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
  // strips' factors and sums, a row per thread
  float lsum = 0.f;
  if (tid < BM) {
    float m = -INFINITY;
    const float* cm = a.cmax + m0 + tid;
#pragma unroll 8
    for (int c = 0; c < a.n_ch; ++c) m = fmaxf(m, cm[(int64_t)c * a.Mp]);
    if (split == 0 && n0 == 0) a.rmax[m0 + tid] = m;
    const float2* st = a.stat + (int64_t)s0 * a.Mp + m0 + tid;
#pragma unroll 8
    for (int s = 0; s < s1 - s0; ++s) {
      const float2 v = st[(int64_t)s * a.Mp];
      const _Float16 f = (_Float16)__builtin_amdgcn_exp2f((v.x - m) + PX_LIFT);
      fac[s * BM + tid] = f;
      lsum = fmaf(v.y, (float)f, lsum);
    }
    row_f[tid] = lsum == 0.f ? 0.f : 0.5f / lsum;
    if (n0 == 0) a.lsum[(int64_t)split * a.Mp + m0 + tid] = lsum;
  }
  floatx16 acc[RM][RN];
#pragma unroll
  for (int i = 0; i < RM; ++i)
#pragma unroll
    for (int j = 0; j < RN; ++j) acc[i][j] = floatx16{};
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // only copies are counted from here on
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) issue(i);
  kh2 fc[RM];
  for (int t0 = 0; t0 < steps; t0 += RING) {
#pragma unroll
    for (int u = 0; u < RING; ++u) {
      if (t0 + u >= steps) break;
      px_stage_ready<(RING - 2) * NI>();
      issue((u + RING - 1) % RING);
      if (u % 2 == 0) {
#pragma unroll
        for (int i = 0; i < RM; ++i) {
          const _Float16 f = fac[((t0 + u) >> 1) * BM + (wm * RM + i) * 32 + n];
          fc[i] = kh2{f, f};
        }
      }
      const uint4* sa = ring + u * STAGE + (wm * RM) * 32 + n;
      const uint4* sb = ring + u * STAGE + 4 * BM + (wn * RN) * 32 + n;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        uint4 fa[RM], fb[RN];
#pragma unroll
        for (int j = 0; j < RN; ++j) fb[j] = sb[(2 * kk + hh) * BN + 32 * j];
#pragma unroll
        for (int i = 0; i < RM; ++i) {
          const uint4 v = sa[(2 * kk + hh) * BM + 32 * i];
          fa[i].x = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.x) * fc[i]);
          fa[i].y = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.y) * fc[i]);
          fa[i].z = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.z) * fc[i]);
          fa[i].w = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, v.w) * fc[i]);
        }
#pragma unroll
        for (int i = 0; i < RM; ++i)
#pragma unroll
          for (int j = 0; j < RN; ++j) acc[i][j] = px_mfma<_Float16>(fa[i], fb[j], acc[i][j]);
      }
    }
  }
  px_stage_ready<0>();                             // the last copies, before the workgroup's LDS is another's
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
// Workgroup = (row, 512 columns), a lane 8 columns, wave w splits and chunks w, w + 4, ...
__global__ __launch_bounds__(256) void prefix_join_kernel(const PrefixArgs a) {
  __shared__ float red[3][64][9];
  const int row = blockIdx.x, nr = a.B * a.gs, h = row / nr, b = row % nr / a.gs, q = h * a.gs + row % a.gs;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t bq = (int64_t)b * a.n_hg + (q >> 5);
  const float mp = a.rmax[row];
  float ms = -INFINITY;                            // in units of log 2, as the prefix's
  for (int c = 0; c < a.n_c1; ++c) ms = fmaxf(ms, a.own_max[((int64_t)b * a.Hq + q) * a.n_c1 + c] * LOG2E);
  const float m = fmaxf(mp, ms);
  const float wp = __builtin_amdgcn_exp2f((mp - m) - PX_LIFT);
  const float wo = ms > -INFINITY ? __builtin_amdgcn_exp2f(ms - m) : 0.f;
  const float vmul = 2.f * a.head[1];
  const float* psum = a.own_sum + (bq * a.n_c2) * 32 + (q & 31);
  const int n_own = wo > 0.f ? a.n_c2 : 0;         // own positions without weight are not looked at (their sums may be NaN)
  if (threadIdx.x == 0 && blockIdx.y == 0) {
    float l = 0.f, o = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.n_split; ++s) l += a.lsum[(int64_t)s * a.Mp + row];
#pragma unroll 8
    for (int c = 0; c < n_own; ++c) o += psum[(int64_t)c * 32];
    a.jsum[bq * 32 + (q & 31)] = n_own ? l * wp + o * wo : l * wp;
    if (a.jmax) a.jmax[(int64_t)b * a.Hq + q] = m * (1.f / LOG2E);
  }
  const int c0 = blockIdx.y * 512 + 8 * lane;
  float v[8] = {};
  if (c0 < a.Rvp) {
    const _Float16* p = a.part + (int64_t)row * a.Rvp + c0;
#pragma unroll 8
    for (int s = wave; s < a.n_split; s += 4) {
      const half8 e = *(const half8*)(p + (int64_t)s * a.M * a.Rvp);
      const float f = a.lsum[(int64_t)s * a.Mp + row];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf((float)e[i], f, v[i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= wp * vmul;
#pragma unroll 2
    for (int c = wave; c < n_own; c += 4) {
      const int64_t at = ((bq * a.n_c2 + c) * 32 + (q & 31)) * a.own_Rvp + c0;
      if (a.own_part16) {
        const half8 e = *(const half8*)((const _Float16*)a.own_part + at);
        const float f = wo * psum[(int64_t)c * 32];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = fmaf((float)e[i], f, v[i]);
      } else {
        const float4* e = (const float4*)((const float*)a.own_part + at);
        const float4 x = e[0], y = e[1];
        v[0] = fmaf(x.x, wo, v[0]); v[1] = fmaf(x.y, wo, v[1]); v[2] = fmaf(x.z, wo, v[2]); v[3] = fmaf(x.w, wo, v[3]);
        v[4] = fmaf(y.x, wo, v[4]); v[5] = fmaf(y.y, wo, v[5]); v[6] = fmaf(y.z, wo, v[6]); v[7] = fmaf(y.w, wo, v[7]);
      }
    }
  }
  if (wave) {
#pragma unroll
    for (int i = 0; i < 8; ++i) red[wave - 1][lane][i] = v[i];
  }
  __syncthreads();
  if (wave || c0 >= a.Rvp) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] += (red[0][lane][i] + red[1][lane][i]) + red[2][lane][i];
  float4* o = (float4*)(a.jpart + (bq * 32 + (q & 31)) * a.Rvp + c0);
  o[0] = make_float4(v[0], v[1], v[2], v[3]);
  o[1] = make_float4(v[4], v[5], v[6], v[7]);
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

template <typename XT, int NG> static void launch_logits(const PrefixArgs& a, int groups, hipStream_t st) {
  const size_t lds = (size_t)a.ks_max * 4096 + NG * 8192 + NG * 32 * 4 * 5;
  const dim3 grid((unsigned)(round_up(a.n_ch, 8) * a.Hkv + a.own_wg), (unsigned)ceil_div(groups, NG));
  hipLaunchKernelGGL((prefix_logits_kernel<XT, NG>), grid, dim3(256), lds, st, a);
}

int launch_prefix_logits(const PrefixArgs& a, int dtype, hipStream_t st) {
  const int groups = (int)ceil_div((int64_t)a.B * a.gs, 32);
  if (groups == 1) {
    if (dtype == STARKV_F16) launch_logits<_Float16, 1>(a, groups, st);
    else launch_logits<__bf16, 1>(a, groups, st);
  } else {
    if (dtype == STARKV_F16) launch_logits<_Float16, PX_GROUPS>(a, groups, st);
    else launch_logits<__bf16, PX_GROUPS>(a, groups, st);
  }
  return (int)hipGetLastError();
}

int launch_prefix_pv(const PrefixArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(8 * ceil_div((int64_t)a.n_split * a.tiles_m * a.tiles_n, 8)));
  if (a.bm == 256) hipLaunchKernelGGL((prefix_pv_kernel<2, 4, 4, 2>), grid, dim3(512), 0, st, a);
  else if (a.bm == 128) hipLaunchKernelGGL((prefix_pv_kernel<2, 2, 2, 4>), grid, dim3(512), 0, st, a);
  else hipLaunchKernelGGL((prefix_pv_kernel<2, 1, 1, 8>), grid, dim3(512), 0, st, a);
  return (int)hipGetLastError();
}

int launch_prefix_join(const PrefixArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(prefix_join_kernel, dim3((unsigned)a.M, (unsigned)ceil_div(a.Rvp, 512)), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace starkv
