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
//    workgroup a row (long rows: many), and writes the kept positions in ascending
//    order by prefix sums: positions above the key, and the first few at it.
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
  const int wave = tid >> 6, lane = tid & 63, s = blockIdx.x * SCORE_COLS + 4 * lane;
  const int h0 = wave * a.H / 4, h1 = (wave + 1) * a.H / 4;
  const T* x = (const T*)a.x + b * a.x_sb;
  // eight heads' logits at a time, the first asked for before the statistics (16 x 32 rows of
  // 32768: 15.5 us, 17 without; 67 MB, read again from the caches)
  float v[8][4];
  auto fetch = [&](int h) {
    if (s < a.S)
#pragma unroll
      for (int i = 0; i < 8; ++i) row4(a, x + min(h + i, a.H - 1) * a.x_sh, s, v[i]);
  };
  fetch(h0);
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
  float w[4] = {};
  for (int h = h0; h < h1; h += 8) {
    if (h > h0) fetch(h);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (h + i >= h1 || s >= a.S) break;
      const float2 st = row_stat[h + i];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] += __builtin_amdgcn_exp2f((v[i][j] - st.x) * LOG2E) * st.y;
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
constexpr int SEL_TILES = 7;                       // whose keys fit LDS beside the histogram

// a score's bits in ascending order of value: NaN counts as -infinity, -0 as 0
__device__ inline uint32_t score_key(float x) {
  x = x == x ? x + 0.f : -INFINITY;
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}

constexpr uint32_t ZERO_KEY = 0x80000000u;

// inclusive sum over the wave's lanes, in six adds that take another lane's value (by exchanges through LDS four scans cost
// 2 us of a row's 13)
template <int CTRL, int ROWS> __device__ inline int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xf, false);
}
__device__ inline int wave_scan(int v) {
  v = dpp_add<0x111, 0xf>(v);                      // 1, 2, 4 and 8 lanes on within rows of 16
  v = dpp_add<0x112, 0xf>(v);
  v = dpp_add<0x114, 0xf>(v);
  v = dpp_add<0x118, 0xf>(v);
  v = dpp_add<0x142, 0xa>(v);                      // a row's sum to the odd rows, that of 32 lanes to the upper 32
  return dpp_add<0x143, 0xc>(v);
}

// the keys of candidates t * 4096 + 4 tid .. + 3 of n, 0 behind the last
__device__ inline void sel_fetch(const float* x, int n, int t, uint32_t (&k)[4]) {
  const int p = t * SEL_TILE + 4 * threadIdx.x;
  float v[4] = {};
  if (p + 4 <= n) {
    load4(x + p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (p + i < n) v[i] = x[p + i];
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) k[i] = p + i < n ? score_key(v[i]) : 0;
}

constexpr int SEL_LOW[3] = {21, 10, 0}, SEL_BITS[3] = {11, 11, 10};
struct SelShared {
  // four copies of each bin, a lane's by its number: equal digits otherwise queue 64 deep
  uint32_t hist[2048 * 4];
  int tot[2][16];
  int found[2];
};

// counts the digits [low, low + bits) of four keys a thread whose digits above are `key`.  (Keys of no candidate, behind the
// last, are 0: below every score's, so the largest ones are found before they are reached.)
__device__ inline void sel_count(SelShared& sh, int low, int bits, const uint32_t (&k)[4], uint32_t key) {
  const int lane = threadIdx.x & 63, top = low + bits;
  const uint32_t digits = (1u << bits) - 1;
  uint32_t* mine = &sh.hist[lane & 3];
  auto all = [&](auto one) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if ((top == 32 || (k[i] >> (top & 31)) == key) && one(k[i])) atomicAdd(mine + ((k[i] >> low) & digits) * 4, 1u);
  };
  const bool zero = k[0] == ZERO_KEY || k[1] == ZERO_KEY || k[2] == ZERO_KEY || k[3] == ZERO_KEY;
  if ((top == 32 || key == ZERO_KEY >> (top & 31)) && __any(zero)) {
    // positions that never got any weight are many, and alike: counted by the wave
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += k[i] == ZERO_KEY;
    n = wave_scan(n);
    if (lane == 63) atomicAdd(&sh.hist[((ZERO_KEY >> low) & digits) * 4], (uint32_t)n);
    all([](uint32_t v) { return v != ZERO_KEY; });
  } else {
    all([](uint32_t) { return true; });
  }
}

// The digit at which the keys counted from the largest down reach `need`, and how many lie above it: thread j brings the
// counts of digits 2047 - 2j and 2046 - 2j
__device__ inline void sel_find(SelShared& sh, int hi, int lo, int need) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int incl = wave_scan(hi + lo);
  if (lane == 63) sh.tot[0][wave] = incl;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 15; ++w) incl += w < wave ? sh.tot[0][w] : 0;
  const int before = incl - hi - lo;
  if (before < need && need <= incl) {
    const bool first = need <= before + hi;
    sh.found[0] = first ? 2047 - 2 * tid : 2046 - 2 * tid;
    sh.found[1] = first ? before : before + hi;
  }
  __syncthreads();
}

// how many of four keys a thread lie above `key` (low half), and at it
__device__ inline int sel_compare(const uint32_t (&k)[4], uint32_t key) {
  int c = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) c += k[i] > key ? 1 : k[i] == key ? 0x10000 : 0;
  return c;
}

// Writes the kept ones of a thread's four candidates, number p of the row on: those above the key, and of those at
// it the first `need`; g above and e at it lie before them
__device__ inline void sel_put(const SelectArgs& a, int* out, int p, const uint32_t (&k)[4], uint32_t key, int need, int g, int e) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (k[i] > key) {
      out[a.sinks + g + min(e, need)] = a.sinks + p + i;
      ++g;
    } else if (k[i] == key) {
      if (e < need) out[a.sinks + g + e] = a.sinks + p + i;
      ++e;
    }
  }
}

__device__ inline void sel_fixed(const SelectArgs& a, int* out) {
  for (int i = threadIdx.x; i < a.sinks; i += SEL_T) out[i] = i;
  for (int i = threadIdx.x; i < a.recent; i += SEL_T) out[a.keep - a.recent + i] = a.length - a.recent + i;
}

// all candidates or none
__global__ __launch_bounds__(SEL_T) void select_all_kernel(const SelectArgs a) {
  int* out = a.out + blockIdx.x * a.o_sb;
  sel_fixed(a, out);
  for (int i = a.sinks + threadIdx.x; i < a.keep - a.recent; i += SEL_T) out[i] = i;
}

// One workgroup a row, its keys in LDS.  About 7 us of it are the sixteen barriers, three histograms and the first load
// (100 positions: 9.5 us with the launch), then 1.5 us a tile of 4096 (8 rows of 8449: 11.6 us, of 16384 14.4): the tile's
// instructions on its one CU.  A row in pieces takes four launches, 28 us at 100000 positions, so it starts where the keys
// no longer fit LDS (28672: 19 us here, 27 in pieces).
__global__ __launch_bounds__(SEL_T) void select_kernel(const SelectArgs a) {
  extern __shared__ __attribute__((aligned(16))) uint32_t sel_keys[];
  __shared__ SelShared sh;
  __shared__ int place[SEL_TILES * 16];            // [tile][wave]: above (low half) and at the key, then those before
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const float* x = a.scores + blockIdx.x * a.s_sb + a.sinks;
  int* out = a.out + blockIdx.x * a.o_sb;
  const int n = a.length - a.sinks - a.recent, tiles = (n + SEL_TILE - 1) / SEL_TILE;
#pragma unroll 1
  for (int j0 = 0; j0 < 4 * tiles; j0 += 16) {
    float v[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = x[min((j0 + j) * SEL_T + tid, n - 1)];
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (j0 + j < 4 * tiles) sel_keys[(j0 + j) * SEL_T + tid] = (j0 + j) * SEL_T + tid < n ? score_key(v[j]) : 0;
  }
  auto four = [&](int t, uint32_t (&k)[4]) { __builtin_memcpy(k, __builtin_assume_aligned(&sel_keys[t * SEL_TILE + 4 * tid], 16), 16); };
  uint32_t key = 0;
  int need = a.keep - a.sinks - a.recent;          // of the keys that share the digits found so far
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int low = pass == 0 ? SEL_LOW[0] : pass == 1 ? SEL_LOW[1] : SEL_LOW[2], bits = pass == 2 ? SEL_BITS[2] : SEL_BITS[0];
    uint4* clear = (uint4*)sh.hist + tid;
    clear[0] = clear[SEL_T] = make_uint4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll 1
    for (int t = 0; t < tiles; ++t) {
      uint32_t k[4];
      four(t, k);
      sel_count(sh, low, bits, k, key);
    }
    __syncthreads();
    const uint4 hi = *(const uint4*)&sh.hist[(2047 - 2 * tid) * 4], lo = *(const uint4*)&sh.hist[(2046 - 2 * tid) * 4];
    sel_find(sh, (int)(hi.x + hi.y + hi.z + hi.w), (int)(lo.x + lo.y + lo.z + lo.w), need);
    key = (key << bits) | (uint32_t)sh.found[0];
    need -= sh.found[1];
  }
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    uint32_t k[4];
    four(t, k);
    const int sum = wave_scan(sel_compare(k, key));
    if (lane == 63) place[t * 16 + wave] = sum;
  }
  sel_fixed(a, out);
  __syncthreads();
  if (wave == 0) {                                 // (halves of 16 bits: fewer than 65536 candidates)
    static_assert(SEL_TILES * 16 <= 128 && SEL_TILES * SEL_TILE < 65536, "two a lane");
    const int i = 2 * lane, x0 = i < 16 * tiles ? place[i] : 0, x1 = i < 16 * tiles ? place[i + 1] : 0;
    const int before = wave_scan(x0 + x1) - x0 - x1;
    if (i < 16 * tiles) { place[i] = before; place[i + 1] = before + x0; }
  }
  __syncthreads();
#pragma unroll 1
  for (int t = 0; t < tiles; ++t) {
    uint32_t k[4];
    four(t, k);
    const int c = sel_compare(k, key), at = place[t * 16 + wave] + wave_scan(c) - c;
    sel_put(a, out, t * SEL_TILE + 4 * tid, k, key, need, at & 0xffff, at >> 16);
  }
}

// Long rows: a workgroup counts the digits of a piece (its own histogram in memory, no atomics between workgroups); the
// next launch adds the pieces up, finds the digit and counts the next; the last finds its place from the histograms of
// the pieces before it, and writes.  state[row][pass]: (key so far, keys still needed at it).
template <int PASS>
__device__ inline void sel_join(SelShared& sh, const SelectArgs& a, int need0, uint32_t& key, int& need) {
  const int tid = threadIdx.x, row = blockIdx.y;
  key = 0;
  need = need0;
  if constexpr (PASS > 1) { const int2 s = a.state[row * 3 + PASS - 2]; key = (uint32_t)s.x; need = s.y; }
  const uint2* h = (const uint2*)(a.hist + ((int64_t)(PASS - 1) * a.B + row) * a.pieces * 2048) + (1023 - tid);
  int hi = 0, lo = 0;
  for (int i0 = 0; i0 < a.pieces; i0 += 16) {
    uint2 v[16];                                   // digits 2046 - 2 tid, 2047 - 2 tid
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = h[(int64_t)min(i0 + i, a.pieces - 1) * 1024];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      lo += i0 + i < a.pieces ? (int)v[i].x : 0;
      hi += i0 + i < a.pieces ? (int)v[i].y : 0;
    }
  }
  if (PASS == 3 && tid < 512) hi = lo = 0;         // digits past 1023: none (the last word holds another count)
  sel_find(sh, hi, lo, need);
  key = (key << SEL_BITS[PASS - 1]) | (uint32_t)sh.found[0];
  need -= sh.found[1];
  if (blockIdx.x == 0 && tid == 0) a.state[row * 3 + PASS - 1] = make_int2((int)key, need);
}

// f(tile, keys of it and the next) for the tiles of a piece, two at a time, asked for under the work of the two before
template <typename F> __device__ inline void sel_each(const float* x, int n, F f) {
  const int tiles = (n + SEL_TILE - 1) / SEL_TILE;
  uint32_t k[2][4], cur[2][4];
  sel_fetch(x, n, 0, k[0]);
  sel_fetch(x, n, 1, k[1]);
  for (int t = 0; t < tiles; t += 2) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) cur[i][j] = k[i][j];
      sel_fetch(x, n, t + 2 + i, k[i]);
    }
    f(t, cur);
  }
}

template <int PASS>
__global__ __launch_bounds__(SEL_T) void select_count_kernel(const SelectArgs a) {
  __shared__ SelShared sh;
  const int tid = threadIdx.x, row = blockIdx.y, n = a.length - a.sinks - a.recent, p0 = blockIdx.x * a.piece_len;
  uint32_t key = 0;
  int need, above = 0;
  if constexpr (PASS > 0) sel_join<PASS>(sh, a, a.keep - a.sinks - a.recent, key, need);
  for (int i = tid; i < 2048 * 4; i += SEL_T) sh.hist[i] = 0;
  __syncthreads();
  const int m = min(a.piece_len, n - p0);
  sel_each(a.scores + row * a.s_sb + a.sinks + p0, m, [&](int, const uint32_t (&k)[2][4]) {
    sel_count(sh, SEL_LOW[PASS], SEL_BITS[PASS], k[0], key);
    sel_count(sh, SEL_LOW[PASS], SEL_BITS[PASS], k[1], key);
    if constexpr (PASS == 2) {
#pragma unroll
      for (int i = 0; i < 8; ++i) above += k[i >> 2][i & 3] >> SEL_BITS[2] > key;
    }
  });
  if constexpr (PASS == 2) {                       // bins that the last pass leaves free: what lies above the key's other digits
    above = wave_scan(above);
    if ((tid & 63) == 63) atomicAdd(&sh.hist[2047 * 4], (uint32_t)above);
  }
  __syncthreads();
  uint2* out = (uint2*)(a.hist + (((int64_t)PASS * a.B + row) * a.pieces + blockIdx.x) * 2048) + tid;
  const uint4 lo = *(const uint4*)&sh.hist[tid * 8], hi = *(const uint4*)&sh.hist[tid * 8 + 4];
  *out = make_uint2(lo.x + lo.y + lo.z + lo.w, hi.x + hi.y + hi.z + hi.w);
}

__global__ __launch_bounds__(SEL_T) void select_write_kernel(const SelectArgs a) {
  __shared__ SelShared sh;
  const int tid = threadIdx.x, row = blockIdx.y, n = a.length - a.sinks - a.recent, p0 = blockIdx.x * a.piece_len;
  int* out = a.out + row * a.o_sb;
  if (blockIdx.x == 0) sel_fixed(a, out);
  uint32_t key;
  int need;
  sel_join<3>(sh, a, a.keep - a.sinks - a.recent, key, need);
  // keys above the threshold, and at it, in the pieces before
  int above = 0, at = 0;
  {
    const int before = blockIdx.x, digit = (int)(key & 1023);
    const uint2* h = (const uint2*)(a.hist + ((int64_t)2 * a.B + row) * a.pieces * 2048) + tid;
    if (tid < 512 || tid == 1023)
      for (int i0 = 0; i0 < before; i0 += 16) {
        uint2 v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = h[(int64_t)min(i0 + i, before - 1) * 1024];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (i0 + i >= before) continue;
          above += (2 * tid > digit && tid != 1023 ? (int)v[i].x : 0) + (2 * tid + 1 > digit ? (int)v[i].y : 0);
          if (2 * tid <= digit) at += 2 * tid == digit ? (int)v[i].x : 2 * tid + 1 == digit ? (int)v[i].y : 0;
        }
      }
  }
  __syncthreads();
  sh.hist[tid] = (uint32_t)above;
  sh.hist[SEL_T + tid] = (uint32_t)at;
  __syncthreads();
  for (int w = SEL_T / 2; w >= 1; w >>= 1) {
    if (tid < w) {
      sh.hist[tid] += sh.hist[tid + w];
      sh.hist[SEL_T + tid] += sh.hist[SEL_T + tid + w];
    }
    __syncthreads();
  }
  above = (int)sh.hist[0];
  at = (int)sh.hist[SEL_T];
  const int m = min(a.piece_len, n - p0);
  sel_each(a.scores + row * a.s_sb + a.sinks + p0, m,
           [&](int t, const uint32_t (&k)[2][4]) {
    int c[2], sum[2];
    __syncthreads();                               // the totals before have been read
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = sel_compare(k[i], key);
      sum[i] = wave_scan(c[i]);
      if ((tid & 63) == 63) sh.tot[i][tid >> 6] = sum[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      int all = 0, mine = 0;
#pragma unroll
      for (int w = 0; w < 16; ++w) {
        if (w == tid >> 6) mine = all;
        all += sh.tot[i][w];
      }
      const int before = sum[i] + mine - c[i];     // of this thread, in this tile
      sel_put(a, out, p0 + (t + i) * SEL_TILE + 4 * tid, k[i], key, need, above + (before & 0xffff), at + (before >> 16));
      above += all & 0xffff;
      at += all >> 16;
    }
  });
}

// ---------------------------------------------------------------------------
// Moving rows
// ---------------------------------------------------------------------------
constexpr int MOVE_U = 8, MOVE_T = 1024;           // pieces in flight per thread, threads
typedef uint32_t piece16 __attribute__((ext_vector_type(4)));
typedef uint32_t piece8 __attribute__((ext_vector_type(2)));

// this wave's loads have returned (a barrier alone does not say that they have)
__device__ inline void loads_done() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// Bytes [0, w) of rows pos[i] to row i, i < keep, in pieces of P at any
// alignment; a row's last piece ends with it (and overlaps the one before).
//
// Bound by the memory system: rows lie anywhere, their ends share lines.  A slice of
// 128 bytes a workgroup: 8 x 2048 rows of int8 / int4 latents 31 us (81 MB moved), 4 x
// 8192 fp16 rows of 6.5 KB 188 (409 MB, 2.2 TB/s); 256 bytes 35 and 180; with 512
// threads 30 to 32 and 199 to 217.
template <typename P>
__device__ inline void move_rows(const MoveArgs& a, const int* pos, uint8_t* base, int64_t pitch, int w) {
  typedef P Q __attribute__((aligned(1)));
  const int tid = threadIdx.x, np = (w + (int)sizeof(P) - 1) / (int)sizeof(P);
  const int sh = np <= 1 ? 0 : 32 - __builtin_clz(np - 1);          // lanes of a row: np rounded up to 2^sh
  const int c = tid & ((1 << sh) - 1), r = tid >> sh, rp = MOVE_T >> sh;
  const int off = min(c * (int)sizeof(P), w - (int)sizeof(P));
  const int n = MOVE_U * rp;                       // rows of a chunk
  P v[2][MOVE_U];
  int pos_of[2][MOVE_U];                           // where row i comes from; i itself: it stays
  auto places = [&](int i0, int (&p)[MOVE_U]) {
#pragma unroll
    for (int u = 0; u < MOVE_U; ++u) {
      const int i = i0 + u * rp + r;
      p[u] = i < a.keep ? pos[i] : i;
    }
  };
  auto load = [&](int i0, int (&p)[MOVE_U], P (&to)[MOVE_U]) {
#pragma unroll
    for (int u = 0; u < MOVE_U; ++u) {
      const int i = i0 + u * rp + r;
      if (i < a.keep && (p[u] < i || p[u] >= a.length)) {
        if (a.err != nullptr) *a.err = 1;
        p[u] = i;
      }
      if (c >= np) p[u] = i;
      if (p[u] != i) to[u] = *(const Q*)(base + (int64_t)p[u] * pitch + off);
    }
  };
  // a chunk's rows are asked for a chunk ahead, its positions two
  places(0, pos_of[0]);
  load(0, pos_of[0], v[0]);
  places(n, pos_of[1]);
  for (int i0 = 0; i0 < a.keep; i0 += 2 * n) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const int at = i0 + s * n;
      if (at >= a.keep) break;
      loads_done();                                // of the whole workgroup: the chunk's writes begin
      __syncthreads();
      load(at + n, pos_of[s ^ 1], v[s ^ 1]);
      bool moved[MOVE_U];
#pragma unroll
      for (int u = 0; u < MOVE_U; ++u) moved[u] = pos_of[s][u] != at + u * rp + r;
      places(at + 2 * n, pos_of[s]);
#pragma unroll
      for (int u = 0; u < MOVE_U; ++u)
        if (moved[u]) *(Q*)(base + (int64_t)(at + u * rp + r) * pitch + off) = v[s][u];
    }
  }
}

__global__ __launch_bounds__(MOVE_T) void move_kernel(const MoveArgs a) {
  // a row's slices on one XCD: the lines that two of them share are read, and written back, once
  int unit = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3), kind = 0;
  const int b = unit / a.per_row;
  if (b >= a.B) return;
  unit %= a.per_row;
  const int* pos = a.pos + b * a.p_sb;
  while (unit >= a.units[kind]) unit -= a.units[kind++];
  uint8_t* base;
  int64_t pitch;
  int nb, slice = 0;
  if (kind == MOVE_SCORES) {
    float* s = a.scores + b * a.scores_sb;
    move_rows<uint32_t>(a, pos, (uint8_t*)s, 4, 4);
    loads_done();
    __syncthreads();
    for (int i = a.keep + threadIdx.x; i < a.length; i += MOVE_T) s[i] = 0.f;
    return;
  }
  if (kind == MOVE_K1 || kind == MOVE_K2) {
    const int h = unit % a.Hk;
    const bool second = kind == MOVE_K2;
    base = second ? a.k2 + b * a.k2_sb + a.off2[h] : a.k1 + b * a.k1_sb + a.off1[h];
    pitch = second ? a.pitch2[h] : a.pitch1[h];
    nb = second ? a.nb2[h] : a.nb1[h];
    slice = unit / a.Hk * MOVE_SLICE;
    if (slice >= nb) return;
  } else if (kind < MOVE_V) {
    base = kind == MOVE_KS2 ? a.ks2 + b * a.ks2_sb + unit * a.ks2_sh : a.ks1 + b * a.ks1_sb + unit * a.ks1_sh;
    pitch = 2;
    nb = 2;
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

template <typename T> static void launch_score_t(const ScoreArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)ceil_div(a.S, SCORE_COLS), (unsigned)a.B);
  hipLaunchKernelGGL(score_stat_kernel<T>, dim3((unsigned)((int64_t)a.B * a.H * a.n_max)), dim3(256), 0, st, a);
  hipLaunchKernelGGL((score_kernel<T, false>), grid, dim3(256), 0, st, a);
}

int launch_scores(const ScoreArgs& a, int dtype, hipStream_t st) {
  if (dtype == STARKV_F32) launch_score_t<float>(a, st);
  else if (dtype == STARKV_F16) launch_score_t<_Float16>(a, st);
  else launch_score_t<__bf16>(a, st);
  return (int)hipGetLastError();
}

int launch_decode_scores(const ScoreArgs& a, hipStream_t st) {
  hipLaunchKernelGGL((score_kernel<float, true>), dim3((unsigned)ceil_div(a.S, SCORE_COLS), (unsigned)a.B), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

// Candidates per workgroup of a long row: at least 8192, at most 64 pieces; 0: one workgroup takes the row
int select_piece(int n, int keep_of_them) {
  if (n <= SEL_TILES * SEL_TILE || keep_of_them == 0 || keep_of_them == n) return 0;
  return (int)round_up(std::max<int64_t>(8192, ceil_div(n, 64)), SEL_TILE);
}

int launch_select(const SelectArgs& a, hipStream_t st) {
  const int n = a.length - a.sinks - a.recent, need = a.keep - a.sinks - a.recent, tiles = (int)ceil_div(n, SEL_TILE);
  const dim3 grid((unsigned)a.B), block(SEL_T);
  if (a.piece_len) {
    const dim3 pieces((unsigned)a.pieces, (unsigned)a.B);
    hipLaunchKernelGGL(select_count_kernel<0>, pieces, block, 0, st, a);
    hipLaunchKernelGGL(select_count_kernel<1>, pieces, block, 0, st, a);
    hipLaunchKernelGGL(select_count_kernel<2>, pieces, block, 0, st, a);
    hipLaunchKernelGGL(select_write_kernel, pieces, block, 0, st, a);
  } else if (need == 0 || need == n) {
    hipLaunchKernelGGL(select_all_kernel, grid, block, 0, st, a);
  } else {
    const size_t lds = (size_t)tiles * SEL_TILE * 4;
    if (lds > 16384) {                             // past 64 KB with the histogram: allowed by attribute
      const int e = (int)hipFuncSetAttribute((const void*)select_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, SEL_TILES * SEL_TILE * 4);
      if (e) return e;
    }
    hipLaunchKernelGGL(select_kernel, grid, block, lds, st, a);
  }
  return (int)hipGetLastError();
}

int launch_move(const MoveArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(move_kernel, dim3((unsigned)round_up((int64_t)a.per_row * a.B, 8)), dim3(MOVE_T), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace starkv
