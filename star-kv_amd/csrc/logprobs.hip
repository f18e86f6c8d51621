// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, one pass over each row:
//
//   m = max x,  Z = sum e^(x - m),  S = sum e^(x - m) (x - m)
//   logprob(t) = x_t - m - ln Z,   entropy = ln Z - S / Z
//
// (both terms of the entropy are >= 0: nothing cancels).  Every thread keeps
// its own m, Z and S over 16-byte pieces of the row; a larger maximum rescales
// them, which soon gets rare.  exp2 underflows to 0 at -inf, where S takes a
// clamped difference instead of 0 * inf.
//
// Top alternatives: keys are (logit, lowest index first) as one 64-bit number
// in a total order.  Each thread knows its greatest key from the pass.  With
// NW waves, the ceil(top / NW)-th greatest thread key of every wave is taken,
// and the least of those is a bound that at least `top` elements reach; only
// threads at or above it read their pieces again and gather the elements
// there, a few dozen as a rule.  The gathered keys are then ranked.  Where
// more elements than the buffer holds reach the bound (rows built so), the
// row is searched `top` times instead.
//
// Bound by HBM on many rows (16-bit logits: nearly as much by the exponential
// of every element).
#include <algorithm>

#include "common.hpp"

namespace starkv {

namespace {

constexpr float LOWEST = -3.402823466e38f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float FAR = -1000.f;                     // e^FAR is 0 in fp32

// logits ordered as unsigned integers: -0 = +0, a NaN above everything
__device__ inline uint32_t order32(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);    // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ inline float unorder32(uint32_t k) {
  if (k == 0xffffffffu) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ inline uint64_t make_key(float f, uint32_t idx) { return ((uint64_t)order32(f) << 32) | (uint32_t)~idx; }

struct Stat { float m, z, s; };
__device__ inline float exp_diff(float d) { return __builtin_amdgcn_exp2f(d * LOG2E); }
// both over the larger maximum (empty sides: m = LOWEST, z = s = 0)
__device__ inline Stat merge(const Stat& a, const Stat& b) {
  const float m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - m, FAR), db = fmaxf(b.m - m, FAR);
  const float fa = exp_diff(da), fb = exp_diff(db);
  return {m, a.z * fa + b.z * fb, fa * (a.s + a.z * da) + fb * (b.s + b.z * db)};
}
__device__ inline uint64_t shfl_xor64(uint64_t v, int o) {
  const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, o, 64), hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), o, 64);
  return ((uint64_t)hi << 32) | lo;
}
__device__ inline uint64_t wave_max64(uint64_t v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const uint64_t t = shfl_xor64(v, o);
    v = t > v ? t : v;
  }
  return v;
}

template <typename T> struct Piece;                // 16 bytes of logits
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ void get(uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <> struct Piece<_Float16> {
  static constexpr int N = 8;
  static __device__ void get(uint4 v, float (&f)[8]) {
    const half8 h = __builtin_bit_cast(half8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)h[e];
  }
};
template <> struct Piece<__bf16> {
  static constexpr int N = 8;
  static __device__ void get(uint4 v, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[2 * e] = __uint_as_float(w[e] << 16);
      f[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
    }
  }
};

}  // namespace

// NT threads per workgroup; TOP: alternatives are asked for
template <typename T, int NT, bool TOP>
__global__ __launch_bounds__(NT) void logprobs_kernel(const LogprobArgs a) {
  constexpr int N = Piece<T>::N, NW = NT / 64;
  constexpr int CAP = TOP ? NT * N + 64 : 1;       // one piece of every thread fits
  __shared__ uint64_t buf[CAP];
  __shared__ uint64_t wkey[NW];
  __shared__ Stat wstat[NW];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.pieces;
  const int piece = blockIdx.x - (int)row * a.pieces;
  const T* x = (const T*)a.x + row * a.xs;
  const int lo = piece * a.piece_len, hi = min(a.vocab, lo + a.piece_len);

  // [lo, hi): a head up to the first 16-byte boundary, whole pieces, a tail;
  // the head and the tail are single elements of threads 0 .. N - 2
  const int mis = (int)(((uintptr_t)(x + lo) & 15) / sizeof(T));
  const int head = min(hi - lo, mis ? N - mis : 0);
  const int body = (hi - lo - head) / N, tail0 = lo + head + body * N;
  const T* xb = x + lo + head;
  auto each_head = [&](auto f) {
    if (tid < head) f((float)x[lo + tid], lo + tid);
  };
  auto each_tail = [&](auto f) {
    if (tid < N && tail0 + tid < hi) f((float)x[tail0 + tid], tail0 + tid);
  };

  Stat st = {LOWEST, 0.f, 0.f};
  uint64_t best = 0;                               // this thread's greatest key
  auto raise = [&](float cm) {
    const float d = fmaxf(st.m - cm, FAR), f = exp_diff(d);
    st.s = f * (st.s + st.z * d);
    st.z *= f;
    st.m = cm;
  };
  auto add = [&](float v) {
    const float d = v - st.m, e = exp_diff(d);
    st.z += e;
    st.s = fmaf(e, fmaxf(d, FAR), st.s);
  };
  auto single = [&](float v, int i) {
    if (v > st.m) raise(v);
    add(v);
    if constexpr (TOP) {
      const uint64_t k = make_key(v, i);
      best = k > best ? k : best;
    }
  };
  // in the order of their indices: of equal logits the first one met is the greatest key
  each_head(single);
  for (int p = tid; p < body; p += NT) {
    float f[N];
    Piece<T>::get(*(const uint4*)(xb + (int64_t)p * N), f);
    float cm = f[0];
#pragma unroll
    for (int e = 1; e < N; ++e) cm = fmaxf(cm, f[e]);
    if (cm > st.m) raise(cm);
    if constexpr (TOP) {
      // fmaxf passes over a NaN; the sum below does not
      bool nan = false;
#pragma unroll
      for (int e = 0; e < N; ++e) nan |= f[e] != f[e];
      if (nan || order32(cm) > (uint32_t)(best >> 32)) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
          const uint64_t k = make_key(f[e], lo + head + p * N + e);
          best = k > best ? k : best;
        }
      }
    }
#pragma unroll
    for (int e = 0; e < N; ++e) add(f[e]);
  }
  each_tail(single);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const Stat t = {__shfl_xor(st.m, o, 64), __shfl_xor(st.z, o, 64), __shfl_xor(st.s, o, 64)};
    // the lower lane's side first, so that both lanes form the same sum
    st = (lane & o) ? merge(t, st) : merge(st, t);
  }
  if (lane == 0) wstat[wave] = st;
  if constexpr (TOP) {
    // the r-th greatest thread key of this wave (0: fewer threads hold elements)
    const int r = (a.top + NW - 1) / NW;
    uint64_t mine = best, top = 0;
    for (int i = 0; i < r; ++i) {
      top = wave_max64(mine);
      if (mine == top) mine = 0;                   // keys differ, but for the empty key 0
    }
    if (lane == 0) wkey[wave] = top;
    if (tid == 0) count = 0;
  }
  __syncthreads();
  st = wstat[0];
  for (int v = 1; v < NW; ++v) st = merge(st, wstat[v]);
  const float lnz = logf(st.z);
  if (a.pieces > 1) {
    if (tid == 0) {
      float* o = a.pstat + (row * a.pieces + piece) * 4;
      o[0] = st.m; o[1] = st.z; o[2] = st.s;
    }
  } else if (tid == 0) {
    if (a.tok) {
      const int64_t t = a.tok[row];
      a.lp[row] = t >= 0 && t < a.vocab ? ((float)x[t] - st.m) - lnz : __uint_as_float(0x7fc00000u);
    }
    if (a.ent) a.ent[row] = lnz - st.s / st.z;
  }
  if constexpr (TOP) {
    uint64_t bound = wkey[0];
    for (int v = 1; v < NW; ++v) bound = wkey[v] < bound ? wkey[v] : bound;
    if (best >= bound && best != 0) {
      auto gather = [&](float v, int i) {
        const uint64_t k = make_key(v, i);
        if (k >= bound) {
          const int at = atomicAdd(&count, 1);     // the order of the keys in the buffer does not matter
          if (at < CAP) buf[at] = k;
        }
      };
      each_head(gather);
      each_tail(gather);
      for (int p = tid; p < body; p += NT) {
        float f[N];
        Piece<T>::get(*(const uint4*)(xb + (int64_t)p * N), f);
#pragma unroll
        for (int e = 0; e < N; ++e) gather(f[e], lo + head + p * N + e);
      }
    }
    __syncthreads();
    const int n = count;
    auto emit = [&](int i, uint64_t k) {
      if (a.pieces > 1) {
        a.ptop[(row * a.pieces + piece) * a.top + i] = k;
      } else {
        a.tlp[row * a.top + i] = (unorder32((uint32_t)(k >> 32)) - st.m) - lnz;
        a.tid[row * a.top + i] = (uint32_t)~(uint32_t)k;
      }
    };
    const int have = min(a.top, hi - lo);          // a short last piece may hold fewer
    if (n <= 4 * NT && n <= CAP) {
      for (int i = tid; i < n; i += NT) {
        const uint64_t k = buf[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += buf[j] > k;
        if (rank < a.top) emit(rank, k);
      }
    } else {
      // `top` rounds of the greatest key below the last one, over the buffer or the row
      uint64_t prev = ~(uint64_t)0;
      for (int i = 0; i < have; ++i) {
        uint64_t b = 0;
        auto look = [&](uint64_t k) {
          if (k < prev && k > b) b = k;
        };
        if (n <= CAP) {
          for (int j = tid; j < n; j += NT) look(buf[j]);
        } else {
          auto look1 = [&](float v, int j) { look(make_key(v, j)); };
          each_head(look1);
          each_tail(look1);
          for (int p = tid; p < body; p += NT) {
            float f[N];
            Piece<T>::get(*(const uint4*)(xb + (int64_t)p * N), f);
#pragma unroll
            for (int e = 0; e < N; ++e) look(make_key(f[e], lo + head + p * N + e));
          }
        }
        b = wave_max64(b);
        __syncthreads();                           // the last round's wkey has been read
        if (lane == 0) wkey[wave] = b;
        __syncthreads();
        b = wkey[0];
        for (int v = 1; v < NW; ++v) b = wkey[v] > b ? wkey[v] : b;
        if (tid == 0) emit(i, b);
        prev = b;
      }
    }
    if (a.pieces > 1)
      for (int i = have + tid; i < a.top; i += NT) emit(i, 0);
  }
}

// joins the pieces of a row: statistics in piece order, the greatest of their keys
template <typename T> __global__ __launch_bounds__(256) void logprobs_join_kernel(const LogprobArgs a) {
  const int64_t row = blockIdx.x;
  const float* ps = a.pstat + row * a.pieces * 4;
  Stat st = {ps[0], ps[1], ps[2]};
  for (int p = 1; p < a.pieces; ++p) st = merge(st, Stat{ps[4 * p], ps[4 * p + 1], ps[4 * p + 2]});
  const float lnz = logf(st.z);
  if (threadIdx.x == 0) {
    const T* x = (const T*)a.x + row * a.xs;
    if (a.tok) {
      const int64_t t = a.tok[row];
      a.lp[row] = t >= 0 && t < a.vocab ? ((float)x[t] - st.m) - lnz : __uint_as_float(0x7fc00000u);
    }
    if (a.ent) a.ent[row] = lnz - st.s / st.z;
  }
  // each piece's keys are in descending order: a key's rank is its place in
  // its own piece and the number of greater keys in the others
  const uint64_t* pt = a.ptop + row * a.pieces * a.top;
  const int n = a.pieces * a.top;
  for (int i = threadIdx.x; i < n; i += 256) {
    const uint64_t k = pt[i];
    if (k == 0) continue;
    int rank = 0;
    for (int j = 0; j < n && rank < a.top; ++j) rank += pt[j] > k;
    if (rank < a.top) {
      a.tlp[row * a.top + rank] = (unorder32((uint32_t)(k >> 32)) - st.m) - lnz;
      a.tid[row * a.top + rank] = (uint32_t)~(uint32_t)k;
    }
  }
}

int plan_logprobs(int rows, int vocab, int esize, int cus) { return 1; }

template <typename T, int NT> static int launch_lp(const LogprobArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.rows * a.pieces));
  if (a.top) hipLaunchKernelGGL((logprobs_kernel<T, NT, true>), grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((logprobs_kernel<T, NT, false>), grid, dim3(NT), 0, st, a);
  if (a.pieces > 1) hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3((unsigned)a.rows), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

int launch_logprobs(const LogprobArgs& a, int dtype, hipStream_t st) {
  if (a.rows == 0) return 0;
  if (dtype == STARKV_F16) return launch_lp<_Float16, 512>(a, st);
  if (dtype == STARKV_BF16) return launch_lp<__bf16, 512>(a, st);
  return launch_lp<float, 512>(a, st);
}

}  // namespace starkv
