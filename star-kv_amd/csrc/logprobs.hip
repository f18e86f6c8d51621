// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, one pass over each row:
//
//   m = max x,  Z = sum e^(x - m),  S = sum e^(x - m) (x - m)
//   logprob(t) = x_t - m - ln Z,   entropy = ln Z - S / Z
//
// (both terms of the entropy are >= 0: nothing cancels).  Every thread keeps
// its own m, Z and S over 16-byte pieces of the row, in units of log 2: with
// c = log2 e and M = fl(m c), y = fma(x, c, -M) and 2^y replace x - m and
// e^(x - m), S sums 2^y y.  The rounding of M, e = m c - M, is the same for all
// terms and is taken back at the end (Z 2^-e; S - e Z likewise).  y stops at
// -150, where 2^y is 0, so that -inf adds 0 and not 0 * inf.  A larger maximum
// rescales the sums, which soon gets rare.  That leaves nine and a half issue
// slots an element, four of them the exponential: 16-bit logits are bound by
// those nearly as much as by HBM.
//
// This holds while 2^e is near 1: |e| is up to half a unit of M's last place,
// 0.07 for |m| = 2^20, but 64 for 1e9 and 440 for 1e10, where 2^e is infinite.
// So a thread's maximum starts at -2^20 (logits far below it, finite masks
// among them, add 0 as -inf does), and rows, or pieces of rows, whose maximum
// is outside +-2^20 are summed again with x - m formed first.  fp16 logits are
// all inside.
//
// Top alternatives: keys are (logit, lowest index first) as one 64-bit number
// in a total order.  Each thread knows its greatest logit and the first piece
// that holds it from the pass, (logit, lowest piece first) its coarse key.
// With NW waves, the ceil(top / NW)-th greatest coarse key of every wave is
// taken, and the least of those is a bound that at least `top` elements reach;
// only threads at or above it read pieces again and gather the elements there,
// a few dozen as a rule.  The gathered keys are then ranked.  Where more elements than the buffer holds reach the bound (rows
// built so), the row is searched `top` times instead.
//
// Few rows are split over workgroups, and a second launch joins the pieces.
#include <algorithm>

#include "common.hpp"

namespace starkv {

namespace {

constexpr int LP_NT = 256;                         // threads per workgroup: many rows, pieces of few, short rows
constexpr int LP_WIDE = 1024;                      // rows of 16 KB and more while there are few: one launch, a batch or two
constexpr int LP_MAX_PIECES = 64;                  // of a row (a lane each in the join)
constexpr int LP_BATCH = 4;                        // 16-byte pieces a thread asks for at a time
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr float START = -0x1p20f, HUGE_X = 0x1p20f;   // maxima in between take the fast sums
constexpr float FAR = -150.f;                      // 2^FAR is 0 in fp32

// logits ordered as unsigned integers: -0 = +0, a NaN above everything, and none all ones (a key that every other one
// is below starts the search by rounds)
constexpr uint32_t ORDER_NAN = 0xfffffffeu;
__device__ inline uint32_t order32(float f) {
  if (f != f) return ORDER_NAN;
  const uint32_t u = __float_as_uint(f + 0.0f);    // -0 + 0 = +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ inline float unorder32(uint32_t k) {
  if (k == ORDER_NAN) return __uint_as_float(0x7fc00000u);
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
__device__ inline uint64_t make_key(float f, uint32_t idx) { return ((uint64_t)order32(f) << 32) | (uint32_t)~idx; }

// Sums over some elements: z = sum 2^y, s = sum 2^y y, while they are taken with y = x log2 e - fl(m log2 e), in the end
// (exact_sums) with y = (x - m) log2 e
struct Stat { float m, z, s; };
// (rounded, wherever it is used: a product fused into a difference would leave what the rounding took)
__device__ inline float log2_of(float m) {
#pragma clang fp contract(off)
  return m * LOG2E;
}
// the sums z, s of maximum `from` over the maximum `to` >= from instead
__device__ inline void rebase(Stat& a, float to) {
  const float d = fmaxf(log2_of(a.m) - log2_of(to), FAR), f = __builtin_amdgcn_exp2f(d);
  a.s = f * fmaf(a.z, d, a.s);
  a.z *= f;
  a.m = to;
}
// sums with y = x log2 e - fl(m log2 e) -> with y = (x - m) log2 e, less by what the rounding took
__device__ inline void exact_sums(Stat& a) {
  const float e = fmaf(a.m, LOG2E, -log2_of(a.m)), f = __builtin_amdgcn_exp2f(-e);
  a.s = f * fmaf(-e, a.z, a.s);
  a.z *= f;
}

// wave reductions by lane shifts inside rows of 16 and broadcasts between them; lane 63 ends with the result
template <int CTRL, int ROWS, typename F> __device__ inline uint32_t dpp_step(uint32_t v, uint32_t id, F f) {
  return f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)id, (int)v, CTRL, ROWS, 0xf, false));
}
template <typename F> __device__ inline uint32_t wave_reduce(uint32_t v, uint32_t id, F f) {
  v = dpp_step<0x111, 0xf>(v, id, f);
  v = dpp_step<0x112, 0xf>(v, id, f);
  v = dpp_step<0x114, 0xf>(v, id, f);
  v = dpp_step<0x118, 0xf>(v, id, f);
  v = dpp_step<0x142, 0xa>(v, id, f);
  v = dpp_step<0x143, 0xc>(v, id, f);
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ inline uint32_t wave_max32(uint32_t v) {
  return wave_reduce(v, 0u, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ inline float wave_maxf(float v) {
  return __uint_as_float(wave_reduce(__float_as_uint(v), 0xff800000u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  }));
}
__device__ inline float wave_sumf(float v) {
  return __uint_as_float(wave_reduce(__float_as_uint(v), 0u, [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ inline uint64_t wave_max64(uint64_t v) {
  const uint32_t hi = (uint32_t)(v >> 32), top = wave_max32(hi);
  return ((uint64_t)top << 32) | wave_max32(hi == top ? (uint32_t)v : 0u);
}

template <typename T> struct Piece;                // 16 bytes of logits
template <> struct Piece<float> {
  static constexpr int N = 4;
  static constexpr uint32_t BARRED = 0xff800000u;  // -inf
  static __device__ void get(uint4 v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y); f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <> struct Piece<_Float16> {
  static constexpr int N = 8;
  static constexpr uint32_t BARRED = 0xfc00fc00u;
  static __device__ void get(uint4 v, float (&f)[8]) {
    const half8 h = __builtin_bit_cast(half8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)h[e];
  }
};
template <> struct Piece<__bf16> {
  static constexpr int N = 8;
  static constexpr uint32_t BARRED = 0xff80ff80u;
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

// how many of the n keys are greater than k, read in pairs
__device__ inline int rank_of(const uint64_t* buf, int n, uint64_t k) {
  int rank = 0;
#pragma unroll 8
  for (int j = 0; j + 1 < n; j += 2) {
    const ulonglong2 t = *(const ulonglong2*)(buf + j);
    rank += (t.x > k) + (t.y > k);
  }
  return rank + ((n & 1) && buf[n - 1] > k);
}

// The results of a row with the sums st: its token's log probability, its entropy.  `xt` is the token's logit
// (token_logit), asked for when the kernel starts: two dependent reads that would otherwise end it.
template <typename T> __device__ inline float token_logit(const LogprobArgs& a, int64_t row) {
  if (!a.tok) return 0.f;
  const int64_t t = a.tok[row];
  return t >= 0 && t < a.vocab ? (float)((const T*)a.x)[row * a.xs + t] : __uint_as_float(0x7fc00000u);
}
__device__ inline float finish_row(const LogprobArgs& a, int64_t row, float xt, const Stat& st, bool nan, bool write) {
  const float none = __uint_as_float(0x7fc00000u);
  const float lnz = nan ? none : logf(st.z);
  if (write) {
    if (a.tok) a.lp[row] = (xt - st.m) - lnz;
    if (a.ent) a.ent[row] = nan ? none : lnz - LN2 * (st.s / st.z);
  }
  return lnz;
}

// TOP: alternatives are asked for
template <typename T, int NT, bool TOP> __global__ __launch_bounds__(NT) void logprobs_kernel(const LogprobArgs a) {
  constexpr int N = Piece<T>::N, NW = NT / 64;
  constexpr int CAP = TOP ? (NT * N < 4096 ? NT * N : 4096) + 64 : 1;      // one piece of every thread, of 512 at most
  __shared__ __attribute__((aligned(16))) uint64_t buf[CAP];
  __shared__ uint64_t wkey[NW];
  __shared__ Stat wstat[NW];
  __shared__ int wnan[NW];
  __shared__ int count;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = blockIdx.x / a.pieces;
  const int piece = blockIdx.x - (int)row * a.pieces;
  const T* x = (const T*)a.x + row * a.xs;
  const int lo = piece * a.piece_len, hi = min(a.vocab, lo + a.piece_len);
  // rows with fewer pieces than threads go round the waves, so that each holds some
  const int tid = hi - lo >= (NT + 1) * N ? threadIdx.x : lane * NW + wave;
  const float xt = a.pieces == 1 && tid == 0 ? token_logit<T>(a, row) : 0.f;

  // [lo, hi): a head up to the first 16-byte boundary, whole pieces, a tail;
  // the head and the tail are single elements of threads 0 .. N - 2
  const int mis = (int)(((uintptr_t)(x + lo) & 15) / sizeof(T));
  const int head = min(hi - lo, mis ? N - mis : 0);
  const int body = (hi - lo - head) / N, tail0 = lo + head + body * N;
  const T* xb = x + lo + head;
  // f(value, index) of this thread's single elements and of its pieces' p
  auto each_head = [&](auto f) {
    if (tid < head) f((float)x[lo + tid], lo + tid);
  };
  auto each_tail = [&](auto f) {
    if (tid < N && tail0 + tid < hi) f((float)x[tail0 + tid], tail0 + tid);
  };
  auto of_piece = [&](int p, auto f) {
    float v[N];
    Piece<T>::get(*(const uint4*)(xb + (int64_t)p * N), v);
#pragma unroll
    for (int e = 0; e < N; ++e) f(v[e], lo + head + p * N + e);
  };
  auto each = [&](auto f) {
    each_head(f);
#pragma unroll 1
    for (int p = tid; p < body; p += NT) of_piece(p, f);
    each_tail(f);
  };

  // pieces in the order of their indices: the head (0), the body's piece p (p + 1), the tail
  const int AT_NONE = -1, AT_HEAD = 0, AT_TAIL = body + 1;
  Stat st = {START, 0.f, 0.f};
  float ml = log2_of(START);
  bool nan = false;
  int at = AT_NONE;                                // where this thread's greatest key is; of equal ones the first met
  auto raise = [&](float cm, int where) {
    if (nan) return;
    at = where;
    nan = cm != cm;
    if (!nan) {
      rebase(st, cm);
      ml = log2_of(cm);
    }
  };
  auto add = [&](float v) {
    const float y = fmaxf(fmaf(v, LOG2E, -ml), FAR), e = __builtin_amdgcn_exp2f(y);
    st.z += e;
    st.s = fmaf(e, y, st.s);
  };
  each_head([&](float v, int) {
    if (!(v <= st.m)) raise(v, AT_HEAD);
    add(v);
  });
  // LP_BATCH of this thread's pieces from p on, all asked for at once; past the row's last one: barred logits
  constexpr int R = LP_BATCH;
  auto load = [&](uint4 (&d)[R], int p) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < R; ++u) d[u] = *(const uint4*)(xb + (int64_t)min(p + u * NT, body - 1) * N);
    if (p - tid + R * NT > body) {
#pragma unroll
      for (int u = 0; u < R; ++u)
        if (p + u * NT >= body) d[u] = make_uint4(Piece<T>::BARRED, Piece<T>::BARRED, Piece<T>::BARRED, Piece<T>::BARRED);
    }
  };
  float pm[R];
#pragma unroll
  for (int u = 0; u < R; ++u) pm[u] = 0.f;
#pragma unroll 1
  for (int p = tid; p - tid < body; p += R * NT) {
    uint4 d[R];
    load(d, p);
    float cm;                                      // a NaN stays in a maximum
#pragma unroll
    for (int u = 0; u < R; ++u) {
      float v[N];
      Piece<T>::get(d[u], v);
      pm[u] = v[0];
#pragma unroll
      for (int e = 1; e < N; ++e) pm[u] = __builtin_elementwise_maximum(pm[u], v[e]);
      cm = u == 0 ? pm[0] : __builtin_elementwise_maximum(cm, pm[u]);
    }
    if (!(cm <= st.m)) {
      int where = p;
#pragma unroll
      for (int u = R - 1; u >= 0; --u)
        if (pm[u] == cm || pm[u] != pm[u]) where = p + u * NT;
      raise(cm, where + 1);
    }
#pragma unroll
    for (int u = 0; u < R; ++u) {
      float v[N];
      Piece<T>::get(d[u], v);
#pragma unroll
      for (int e = 0; e < N; ++e) add(v[e]);
    }
  }
  each_tail([&](float v, int) {
    if (!(v <= st.m)) raise(v, AT_TAIL);
    add(v);
  });

  uint64_t best = 0;                               // this thread's coarse key; 0: it holds no element
  auto coarse = [](float v, int at) { return ((uint64_t)order32(v) << 32) | (uint32_t)~at; };
  if constexpr (TOP) {
    if (at != AT_NONE) {
      best = coarse(nan ? __uint_as_float(0x7fc00000u) : st.m, at);
    } else {                                       // nothing above START, or nothing at all
      auto better = [&](float v, int where) {
        const uint64_t k = coarse(v, where);
        best = k > best ? k : best;
      };
      each_head([&](float v, int) { better(v, AT_HEAD); });
#pragma unroll 1
      for (int p = tid; p < body; p += NT) of_piece(p, [&](float v, int) { better(v, p + 1); });
      each_tail([&](float v, int) { better(v, AT_TAIL); });
    }
    // the r-th greatest coarse key of this wave (0: fewer threads hold elements)
    const int r = (a.top + NW - 1) / NW;
    uint64_t mine = best, top = 0;
#pragma unroll 1
    for (int i = 0; i < r; ++i) {
      top = wave_max64(mine);
      if (mine == top) mine = 0;                   // keys differ, but for the empty key 0
    }
    if (lane == 0) wkey[wave] = top;
    if (tid == 0) count = 0;
  }
  // the wave's sums over its maximum
  auto wave_stat = [&]() {
    rebase(st, wave_maxf(st.m));
    st.z = wave_sumf(st.z);
    st.s = wave_sumf(st.s);
    if (lane == 0) wstat[wave] = st;
  };
  wave_stat();
  const bool wave_nan = __any(nan);
  if (lane == 0) wnan[wave] = wave_nan;
  __syncthreads();
  auto all_stat = [&]() {
    float m = wstat[0].m;
#pragma unroll
    for (int v = 1; v < NW; ++v) m = fmaxf(m, wstat[v].m);
    st = Stat{m, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      Stat t = wstat[v];
      rebase(t, m);
      st.z += t.z;
      st.s += t.s;
    }
  };
  all_stat();
  bool any_nan = false;
#pragma unroll
  for (int v = 0; v < NW; ++v) any_nan |= wnan[v] != 0;
  if (st.m > START && st.m < HUGE_X) {
    exact_sums(st);
  } else if (!any_nan) {
    // the maximum itself (START was none of the elements) and then x - m, exactly as the definition has it.  No finite
    // element: z = 0.  +inf: not a number.
    float m = -__builtin_inff();
    each([&](float v, int) { m = fmaxf(m, v); });
    m = wave_maxf(m);
    __syncthreads();                               // wstat has been read
    if (lane == 0) wstat[wave].m = m;
    __syncthreads();
#pragma unroll
    for (int v = 0; v < NW; ++v) m = fmaxf(m, wstat[v].m);
    any_nan = m == __builtin_inff();
    st = Stat{m, 0.f, 0.f};
    if (fabsf(m) < __builtin_inff())
      each([&](float v, int) {
        const float y = fmaxf((v - m) * LOG2E, FAR), e = __builtin_amdgcn_exp2f(y);
        st.z += e;
        st.s = fmaf(e, y, st.s);
      });
    st.z = wave_sumf(st.z);
    st.s = wave_sumf(st.s);
    __syncthreads();
    if (lane == 0) wstat[wave] = st;
    __syncthreads();
    st.z = st.s = 0.f;
#pragma unroll
    for (int v = 0; v < NW; ++v) { st.z += wstat[v].z; st.s += wstat[v].s; }
  }
  float lnz = 0.f;
  if (a.pieces > 1) {
    if (tid == 0) {
      float* o = a.pstat + (row * a.pieces + piece) * 4;
      o[0] = st.m; o[1] = any_nan ? __uint_as_float(0x7fc00000u) : st.z; o[2] = st.s;
    }
  } else {
    lnz = finish_row(a, row, xt, st, any_nan, tid == 0);
  }
  if constexpr (TOP) {
    uint64_t bound = wkey[0];
#pragma unroll
    for (int v = 1; v < NW; ++v) bound = wkey[v] < bound ? wkey[v] : bound;
    if (best >= bound && best != 0) {
      const float least = unorder32((uint32_t)(bound >> 32));
      auto take = [&](float v, int i, int where) {
        if (v < least) return;                     // (a NaN is not)
        if (coarse(v, where) >= bound) {
          const int to = atomicAdd(&count, 1);     // the order of the keys in the buffer does not matter
          if (to < CAP) buf[to] = make_key(v, i);
        }
      };
      each_head([&](float v, int i) { take(v, i, AT_HEAD); });
#pragma unroll 1
      for (int p = tid; p < body; p += R * NT) {
        if (body > R * NT) {                       // else the maxima of the row's only batch are still there
          uint4 d[R];
          load(d, p);
#pragma unroll
          for (int u = 0; u < R; ++u) {
            float v[N];
            Piece<T>::get(d[u], v);
            pm[u] = v[0];
#pragma unroll
            for (int e = 1; e < N; ++e) pm[u] = __builtin_elementwise_maximum(pm[u], v[e]);
          }
        }
        uint32_t hits = 0;
#pragma unroll
        for (int u = 0; u < R; ++u)
          if (!(pm[u] < least) && p + u * NT < body) hits |= 1u << u;
        while (hits) {                             // one copy of the code that takes a piece's elements
          const int q = p + (__ffs(hits) - 1) * NT;
          of_piece(q, [&](float v, int i) { take(v, i, q + 1); });
          hits &= hits - 1;
        }
      }
      each_tail([&](float v, int i) { take(v, i, AT_TAIL); });
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
    if (n <= 2 * NT) {
#pragma unroll 1
      for (int i = tid; i < n; i += NT) {
        const uint64_t k = buf[i];
        const int rank = rank_of(buf, n, k);
        if (rank < a.top) emit(rank, k);
      }
    } else {
      // `top` rounds of the greatest key below the last one, over the buffer or the row
      uint64_t prev = ~(uint64_t)0;
#pragma unroll 1
      for (int i = 0; i < have; ++i) {
        uint64_t b = 0;
        auto look = [&](uint64_t k) {
          if (k < prev && k > b) b = k;
        };
        if (n <= CAP) {
          for (int j = tid; j < n; j += NT) look(buf[j]);
        } else {
          each([&](float v, int j) { look(make_key(v, j)); });
        }
        b = wave_max64(b);
        __syncthreads();                           // the last round's wkey has been read
        if (lane == 0) wkey[wave] = b;
        __syncthreads();
        b = wkey[0];
#pragma unroll
        for (int v = 1; v < NW; ++v) b = wkey[v] > b ? wkey[v] : b;
        if (tid == 0) emit(i, b);
        prev = b;
      }
    }
    if (a.pieces > 1)
      for (int i = have + tid; i < a.top; i += NT) emit(i, 0);
  }
}

// Joins the pieces of a row: their sums, and the greatest of their keys.
template <typename T> __global__ __launch_bounds__(LP_NT) void logprobs_join_kernel(const LogprobArgs a) {
  __shared__ __attribute__((aligned(16))) uint64_t buf[LP_MAX_PIECES * STARKV_MAX_TOP];
  __shared__ int count;
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63, n = a.pieces * a.top;
  const uint64_t* pt = a.ptop + row * n;
  if (tid == 0) count = 0;
  const float xt = tid == 0 ? token_logit<T>(a, row) : 0.f;
  // every wave does the same: a lane a piece
  const bool mine = lane < a.pieces;
  const float4 ps = mine ? ((const float4*)a.pstat)[row * a.pieces + lane] : make_float4(-__builtin_inff(), 0.f, 0.f, 0.f);
  // `top` keys are at or above the q-th greatest of the pieces' r-th keys, q r >= top
  uint64_t bound = 0;
  if (a.top) {
    const int r = (a.top + a.pieces - 1) / a.pieces, q = (a.top + r - 1) / r;
    const uint64_t k = mine ? pt[lane * a.top + r - 1] : 0;
    int rank = 0;
#pragma unroll 8
    for (int p = 0; p < 64; ++p) {
      const uint64_t o = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(k >> 32), p) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)k, p);
      rank += o > k;
    }
    bound = wave_max64(rank == q - 1 ? k : 0);     // (0, and all are ranked, where that many pieces are empty)
  }
  const float m = wave_maxf(ps.x);
  Stat st = {ps.x, ps.y, ps.z};
  const bool nan = __any(st.z != st.z) || m == __builtin_inff();
  // pieces of either way of summing are given over their own maximum, x - m exactly (a piece without a finite element: 0)
  const float d = fmaxf((st.m - m) * LOG2E, FAR), f = __builtin_amdgcn_exp2f(d);
  st.s = f * fmaf(st.z, d, st.s);
  st.z *= f;
  st = Stat{m, wave_sumf(st.z), wave_sumf(st.s)};
  const float lnz = finish_row(a, row, xt, st, nan, tid == 0);
  __syncthreads();
  for (int i = tid; i < n; i += LP_NT) {
    const uint64_t k = pt[i];
    if (k >= bound && k != 0) buf[atomicAdd(&count, 1)] = k;
  }
  __syncthreads();
  const int c = count;
  for (int i = tid; i < c; i += LP_NT) {
    const uint64_t k = buf[i];
    const int rank = rank_of(buf, c, k);
    if (rank < a.top) {
      a.tlp[row * a.top + rank] = (unorder32((uint32_t)(k >> 32)) - st.m) - lnz;
      a.tid[row * a.top + rank] = (uint32_t)~(uint32_t)k;
    }
  }
}

// Workgroups per row, and threads in each (wide: LP_WIDE).  A row of up to 64 KB is one batch of 1024 threads: split
// over workgroups and joined by a second launch, 8 rows of 32000 took 10.8 us instead of 9.7; with 4 workgroups and
// more to a CU 256 threads overlap better.  Longer ones are split while rows alone do not fill the chip.
LogprobPlan plan_logprobs(int rows, int vocab, int esize, int cus) {
  const int64_t bytes = (int64_t)vocab * esize;
  LogprobPlan p = {1, bytes > 16384 && rows < 4 * cus};
  if (bytes > 65536 && rows < cus) {
    p.wide = false;
    const int64_t most = vocab / (2 * LP_NT * (16 / esize));       // at least two pieces a thread
    p.pieces = (int)std::max<int64_t>(1, std::min({(int64_t)LP_MAX_PIECES, ceil_div(4 * cus, rows), most}));
  }
  return p;
}

template <typename T, int NT> static void launch_lp(const LogprobArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.rows * a.pieces));
  if (a.top) hipLaunchKernelGGL((logprobs_kernel<T, NT, true>), grid, dim3(NT), 0, st, a);
  else hipLaunchKernelGGL((logprobs_kernel<T, NT, false>), grid, dim3(NT), 0, st, a);
}
template <typename T> static int launch_lp_t(const LogprobArgs& a, bool wide, hipStream_t st) {
  if (wide) launch_lp<T, LP_WIDE>(a, st);
  else launch_lp<T, LP_NT>(a, st);
  if (a.pieces > 1) hipLaunchKernelGGL((logprobs_join_kernel<T>), dim3((unsigned)a.rows), dim3(LP_NT), 0, st, a);
  return (int)hipGetLastError();
}

int launch_logprobs(const LogprobArgs& a, bool wide, int dtype, hipStream_t st) {
  if (a.rows == 0) return 0;
  if (dtype == STARKV_F16) return launch_lp_t<_Float16>(a, wide, st);
  if (dtype == STARKV_BF16) return launch_lp_t<__bf16>(a, wide, st);
  return launch_lp_t<float>(a, wide, st);
}

}  // namespace starkv
