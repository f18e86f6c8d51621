// A bounded latent cache: attention weights summed by position, the positions
// worth keeping, and the cache's rows moved together in place.
//
// 1. Scores.  s[b, p] (+)= sum_h softmax_p(l[b, h, :])[p].  A softmax row's
//    maximum and sum have to be known before its first weight, and the sum over
//    heads runs across the rows, so the logits are read twice: score_stat_kernel
//    forms each row's (maximum, sum) by pieces of 4096 logits, score_kernel joins
//    the pieces and adds the heads' weights of 256 positions, each of its four
//    waves a quarter of the heads, joined in a fixed order (no atomics: the sums
//    are the same on every run).  Behind a decode call both are there already
//    (the chunk maxima of the K-logit kernel and the chunk sums of the P.V one)
//    and only the second kernel runs.  Statistics and sums are fp32.
// 2. Selection.  select_kernel finds the key (the score's bits, ordered) of the
//    last position kept by radix selection, 11 + 11 + 10 bits from the top, one
//    workgroup a row, and writes the kept positions in ascending order with a
//    running prefix sum: positions above the key, and the first few at it.
// 3. Moving rows.  Row positions[i] >= i goes to row i.  A workgroup owns a slice
//    of a row's bytes and takes the rows in order, a chunk at a time: every row
//    that a chunk writes lies before every row that a later chunk reads, and the
//    chunk's own rows are in registers before its first write.  So the move is in
//    place without a copy of the cache, and slices run side by side.
#include <algorithm>

#include "common.hpp"

namespace starkv {

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int SCORE_PIECE = 4096;                  // logits per workgroup of the statistics
constexpr int SCORE_COLS = 256;                    // positions per workgroup of the sums

// four logits at any alignment of their type, in fp32
__device__ inline void load4(const float* p, float (&v)[4]) { __builtin_memcpy(v, p, 16); }
template <typename T> __device__ inline void load4(const T* p, float (&v)[4]) {
  T e[4];
  __builtin_memcpy(e, p, 8);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = to_f32(e[i]);
}
__device__ inline float one(const float* p) { return *p; }
template <typename T> __device__ inline float one(const T* p) { return to_f32(*p); }

// logits s .. s + 3 of a row (s a multiple of 4: they share a 32-position tile); -inf from S on
template <typename T>
__device__ inline void row4(const ScoreArgs& a, const T* row, int s, float (&v)[4]) {
  const T* p = row + (int64_t)(s >> 5) * a.x_st + (s & 31);
  if (s + 4 <= a.S) {
    load4(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = s + i < a.S ? one(p + i) : -INFINITY;
  }
}

__device__ inline float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ inline float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// (maximum, sum of exp(l - maximum)) of one piece of one row.  A piece of -inf
// alone has (-inf, 0); a NaN makes the sum NaN (the maximum passes it over).
template <typename T>
__global__ __launch_bounds__(256) void score_stat_kernel(const ScoreArgs a) {
  __shared__ float red[4];
  const int tid = threadIdx.x, piece = blockIdx.x % a.n_max;
  const int64_t r = blockIdx.x / a.n_max;
  const T* row = (const T*)a.x + (r / a.H) * a.x_sb + (r % a.H) * a.x_sh;
  const int s0 = piece * SCORE_PIECE;
  float v[4][4];
  float m = -INFINITY;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int s = s0 + 4 * (tid + 256 * k);
    if (s < a.S) row4(a, row, s, v[k]);
    else v[k][0] = v[k][1] = v[k][2] = v[k][3] = -INFINITY;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) m = fmaxf(m, v[k][i]);
  m = wave_max(m);
  if ((tid & 63) == 0) red[tid >> 6] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float m0 = m > -INFINITY ? m : 0.f;
  float l = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < 4; ++i) l += __builtin_amdgcn_exp2f((v[k][i] - m0) * LOG2E);
  l = wave_sum(l);
  __syncthreads();
  if ((tid & 63) == 0) red[tid >> 6] = l;
  __syncthreads();
  if (tid == 0) a.stat[blockIdx.x] = make_float2(m, (red[0] + red[1]) + (red[2] + red[3]));
}

// FUSED: statistics of a decode call (rmax, rsum), else of score_stat_kernel
template <typename T, bool FUSED>
__global__ __launch_bounds__(256) void score_kernel(const ScoreArgs a) {
  __shared__ float2 row_stat[SCORE_MAX_H];         // (maximum, 1 / sum); an empty row has (0, 0)
  __shared__ float part[4][SCORE_COLS];
  const int tid = threadIdx.x, b = blockIdx.y;
  for (int h = tid; h < a.H; h += 256) {
    const int64_t at = ((int64_t)b * a.H + h) * a.n_max;
    float m = -INFINITY, l = 0.f;
    for (int c = 0; c < a.n_max; ++c) m = fmaxf(m, FUSED ? a.rmax[at + c] : a.stat[at + c].x);
    const float m0 = m > -INFINITY ? m : 0.f;
    if constexpr (FUSED) {
      const float* p = a.rsum + (int64_t)(b * a.n_hg + (h >> 5)) * a.n_sum * 32 + (h & 31);
      if (m > -INFINITY)                           // the decode's sums of an empty row are NaN
        for (int c = 0; c < a.n_sum; ++c) l += p[(int64_t)c * 32];
    } else {
      for (int c = 0; c < a.n_max; ++c) l += a.stat[at + c].y * __builtin_amdgcn_exp2f((a.stat[at + c].x - m0) * LOG2E);
    }
    row_stat[h] = make_float2(m0, l == 0.f ? 0.f : 1.f / l);
  }
  __syncthreads();
  const int wave = tid >> 6, lane = tid & 63, s = blockIdx.x * SCORE_COLS + 4 * lane;
  float w[4] = {};
  if (s < a.S) {
    const T* x = (const T*)a.x + b * a.x_sb;
    const int h0 = wave * a.H / 4, h1 = (wave + 1) * a.H / 4;
#pragma unroll 8
    for (int h = h0; h < h1; ++h) {
      float v[4];
      row4(a, x + h * a.x_sh, s, v);
      const float2 st = row_stat[h];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += __builtin_amdgcn_exp2f((v[i] - st.x) * LOG2E) * st.y;
    }
  }
  *(float4*)&part[wave][4 * lane] = make_float4(w[0], w[1], w[2], w[3]);
  __syncthreads();
  const int p = blockIdx.x * SCORE_COLS + tid;
  if (p < a.S) {
    float* o = a.out + b * a.o_sb + p;
    const float t = (part[0][tid] + part[1][tid]) + (part[2][tid] + part[3][tid]);
    *o = a.add ? *o + t : t;
  }
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------
constexpr int SEL_T = 1024, SEL_TILE = 4 * SEL_T;

// a score's bits in ascending order of value: NaN counts as -infinity, -0 as 0
__device__ inline uint32_t score_key(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

// inclusive sum over the wave's lanes
__device__ inline int wave_scan(int v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int t = __shfl_up(v, o, 64);
    if (lane >= o) v += t;
  }
  return v;
}

// NT: tiles of 4096 candidates held in registers (0: read again in each pass)
template <int NT>
__global__ __launch_bounds__(SEL_T) void select_kernel(const SelectArgs a) {
  // four copies of each bin, a lane's by its number: equal scores (positions that
  // never got any weight) otherwise queue 64 deep
  __shared__ uint32_t hist[2048 * 4];
  __shared__ int tot[2][16];
  __shared__ int found[2];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* x = a.scores + blockIdx.x * a.s_sb + a.sinks;
  int* out = a.out + blockIdx.x * a.o_sb;
  const int n = a.length - a.sinks - a.recent, need0 = a.keep - a.sinks - a.recent;
  for (int i = tid; i < a.sinks; i += SEL_T) out[i] = i;
  for (int i = tid; i < a.recent; i += SEL_T) out[a.keep - a.recent + i] = a.length - a.recent + i;
  if (need0 == 0) return;
  const int tiles = (n + SEL_TILE - 1) / SEL_TILE;
  uint32_t held[NT ? NT : 1][4];
  auto fetch = [&](int t, uint32_t (&k)[4]) {
    const int p = t * SEL_TILE + 4 * tid;
    float v[4] = {};
    if (p + 4 <= n) {
      load4(x + p, v);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (p + i < n) v[i] = x[p + i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) k[i] = score_key(v[i]);
  };
  if constexpr (NT > 0) {
#pragma unroll
    for (int t = 0; t < NT; ++t) fetch(t, held[t]);
  }
  // f(tile, keys) for every tile
  auto each = [&](auto f) {
    if constexpr (NT > 0) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if (t < tiles) f(t, held[t]);
    } else {
      for (int t = 0; t < tiles; ++t) {
        uint32_t k[4];
        fetch(t, k);
        f(t, k);
      }
    }
  };
  uint32_t key = 0;
  int need = need0;                                // of the keys that share the digits found so far
  if (need0 < n) {
#pragma unroll
    for (int pass = 0; pass < 3; ++pass) {
      const int low = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
      for (int i = tid; i < 2048 * 4; i += SEL_T) hist[i] = 0;
      __syncthreads();
      each([&](int t, const uint32_t (&k)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = t * SEL_TILE + 4 * tid + i < n && (pass == 0 || (k[i] >> (low + bits)) == key);
          if (in) atomicAdd(&hist[((k[i] >> low) & ((1u << bits) - 1)) * 4 + (lane & 3)], 1u);
        }
      });
      __syncthreads();
      // thread j has bins 2047 - 2j and 2046 - 2j: sums from the largest key down
      const uint4 hi = *(const uint4*)&hist[(2047 - 2 * tid) * 4], lo = *(const uint4*)&hist[(2046 - 2 * tid) * 4];
      const int ch = (int)(hi.x + hi.y + hi.z + hi.w), cl = (int)(lo.x + lo.y + lo.z + lo.w);
      int incl = wave_scan(ch + cl);
      if (lane == 63) tot[0][wave] = incl;
      __syncthreads();
      for (int w = 0; w < wave; ++w) incl += tot[0][w];
      const int before = incl - ch - cl;           // keys of larger digits
      if (before < need && need <= incl) {
        const bool first = need <= before + ch;
        found[0] = first ? 2047 - 2 * tid : 2046 - 2 * tid;
        found[1] = first ? before : before + ch;
      }
      __syncthreads();
      key = (key << bits) | (uint32_t)found[0];
      need -= found[1];
    }
  }
  // positions above the key are all kept, of those at it the first `need`
  int above = 0, at = 0;                           // of the tiles before
  each([&](int t, const uint32_t (&k)[4]) {
    int c = 0;
    const int p = t * SEL_TILE + 4 * tid;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i < n) c += k[i] > key ? 1 : k[i] == key ? 0x10000 : 0;
    int incl = wave_scan(c);
    if (lane == 63) tot[t & 1][wave] = incl;
    __syncthreads();
    int all = 0, mine = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {
      if (w == wave) mine = all;
      all += tot[t & 1][w];
    }
    incl += mine - c;                              // before this thread, in this tile
    int g = above + (incl & 0xffff), e = at + (incl >> 16);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (p + i >= n) continue;
      if (k[i] > key) {
        out[a.sinks + g + min(e, need)] = a.sinks + p + i;
        ++g;
      } else if (k[i] == key) {
        if (e < need) out[a.sinks + g + e] = a.sinks + p + i;
        ++e;
      }
    }
    above += all & 0xffff;
    at += all >> 16;
  });
}

// ---------------------------------------------------------------------------
// Moving rows
// ---------------------------------------------------------------------------
constexpr int MOVE_U = 8;                          // pieces in flight per thread
typedef uint32_t piece16 __attribute__((ext_vector_type(4)));
typedef uint32_t piece8 __attribute__((ext_vector_type(2)));

// this wave's loads have returned (a barrier alone does not say that they have)
__device__ inline void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Bytes [0, w) of rows pos[i] to row i, i < keep, in pieces of P at any
// alignment; a row's last piece ends with it (and overlaps the one before).
template <typename P>
__device__ inline void move_rows(const MoveArgs& a, const int* pos, uint8_t* base, int64_t pitch, int w) {
  typedef P Q __attribute__((aligned(1)));
  const int tid = threadIdx.x, np = (w + (int)sizeof(P) - 1) / (int)sizeof(P);
  const int sh = np <= 1 ? 0 : 32 - __builtin_clz(np - 1);          // lanes of a row: np rounded up to 2^sh
  const int c = tid & ((1 << sh) - 1), r = tid >> sh, rp = 256 >> sh;
  const int off = min(c * (int)sizeof(P), w - (int)sizeof(P));
  for (int i0 = 0; i0 < a.keep; i0 += MOVE_U * rp) {
    P v[MOVE_U];
    bool ok[MOVE_U];
#pragma unroll
    for (int u = 0; u < MOVE_U; ++u) {
      const int i = i0 + u * rp + r;
      const int p = i < a.keep ? pos[i] : i;
      const bool in = p >= i && p < a.length;
      if (i < a.keep && !in && a.err != nullptr) *a.err = 1;
      ok[u] = c < np && in && p != i && i < a.keep;
      if (ok[u]) v[u] = *(const Q*)(base + (int64_t)p * pitch + off);
    }
    loads_done();                                  // of the whole workgroup: the writes begin
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MOVE_U; ++u)
      if (ok[u]) *(Q*)(base + (int64_t)(i0 + u * rp + r) * pitch + off) = v[u];
  }
}

__global__ __launch_bounds__(256) void move_kernel(const MoveArgs a) {
  const int b = blockIdx.y;
  const int* pos = a.pos + b * a.p_sb;
  int unit = blockIdx.x, kind = 0;
  while (unit >= a.units[kind]) unit -= a.units[kind++];
  uint8_t* base;
  int64_t pitch;
  int nb, slice = 0;
  if (kind == MOVE_SCORES) {
    float* s = a.scores + b * a.scores_sb;
    move_rows<uint32_t>(a, pos, (uint8_t*)s, 4, 4);
    loads_done();
    __syncthreads();
    for (int i = a.keep + threadIdx.x; i < a.length; i += 256) s[i] = 0.f;
    return;
  }
  if (kind < MOVE_V) {
    const int h = unit;
    const bool second = kind == MOVE_K2 || kind == MOVE_KS2;
    if (kind == MOVE_K1 || kind == MOVE_K2) {
      base = (second ? a.k2 + b * a.k2_sb + a.off2[h] : a.k1 + b * a.k1_sb + a.off1[h]);
      pitch = second ? a.pitch2[h] : a.pitch1[h];
      nb = second ? a.nb2[h] : a.nb1[h];
      if (nb == 0) return;
    } else {
      base = second ? a.ks2 + b * a.ks2_sb + h * a.ks2_sh : a.ks1 + b * a.ks1_sb + h * a.ks1_sh;
      pitch = 2;
      nb = 2;
    }
  } else {
    const MoveRows& v = a.v[kind - MOVE_V];
    base = v.base + b * v.sb;
    pitch = v.pitch;
    nb = v.nb;
    slice = unit * MOVE_SLICE;
  }
  base += slice;
  const int w = min(nb - slice, MOVE_SLICE);
  if (w >= 16) move_rows<piece16>(a, pos, base, pitch, w);
  else if (w >= 8) move_rows<piece8>(a, pos, base, pitch, w);
  else if (w >= 4) move_rows<uint32_t>(a, pos, base, pitch, w);
  else if (w >= 2) move_rows<uint16_t>(a, pos, base, pitch, w);
  else move_rows<uint8_t>(a, pos, base, pitch, w);
}

}  // namespace

int score_pieces(int S) { return (int)ceil_div(S, SCORE_PIECE); }

template <typename T> static void launch_score_t(const ScoreArgs& a, bool fused, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.S, SCORE_COLS), (unsigned)a.B);
  if (fused) {
    hipLaunchKernelGGL((score_kernel<T, true>), grid, dim3(256), 0, st, a);
    return;
  }
  hipLaunchKernelGGL(score_stat_kernel<T>, dim3((unsigned)((int64_t)a.B * a.H * a.n_max)), dim3(256), 0, st, a);
  hipLaunchKernelGGL((score_kernel<T, false>), grid, dim3(256), 0, st, a);
}

int launch_scores(const ScoreArgs& a, int dtype, bool fused, hipStream_t st) {
  if (dtype == STARKV_F32) launch_score_t<float>(a, fused, st);
  else if (dtype == STARKV_F16) launch_score_t<_Float16>(a, fused, st);
  else launch_score_t<__bf16>(a, fused, st);
  return (int)hipGetLastError();
}

int launch_select(const SelectArgs& a, int B, hipStream_t st) {
  const int tiles = (int)ceil_div(a.length - a.sinks - a.recent, SEL_TILE);
  const dim3 grid((unsigned)B), block(SEL_T);
  if (tiles <= 1) hipLaunchKernelGGL(select_kernel<1>, grid, block, 0, st, a);
  else if (tiles <= 4) hipLaunchKernelGGL(select_kernel<4>, grid, block, 0, st, a);
  else if (tiles <= 8) hipLaunchKernelGGL(select_kernel<8>, grid, block, 0, st, a);
  else hipLaunchKernelGGL(select_kernel<0>, grid, block, 0, st, a);
  return (int)hipGetLastError();
}

int launch_move(const MoveArgs& a, int B, hipStream_t st) {
  int n = 0;
  for (int k = 0; k < MOVE_KINDS; ++k) n += a.units[k];
  if (n == 0) return 0;
  hipLaunchKernelGGL(move_kernel, dim3((unsigned)n, (unsigned)B), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace starkv
