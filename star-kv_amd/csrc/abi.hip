// C ABI of libstarkv: argument validation, launch planning, workspace layout.
//
// Nothing here allocates device memory or synchronises; validation runs
// before any HIP call so that every argument error is reported without a GPU.
#include <algorithm>
#include <climits>
#include <cmath>
#include <mutex>
#include <vector>

#include "common.hpp"

using namespace starkv;

namespace {

constexpr int FULL_CHIP_CUS = 256;  // an MI355X: planning default when no device can be queried
constexpr int K1_WG_PER_CU = 1;     // k_logits_kernel: one 8-wave (or 4-wave) workgroup per CU
constexpr int MAX_S = 1 << 24;
constexpr int MAX_RV = 8192;
constexpr int64_t V_MAX_PITCH = 1 << 24;   // V row pitch (bytes) of the 24-bit offset multiply in P.V
constexpr int K2_MAX_H = 64;       // P.V: up to two 32-head groups
constexpr int64_t MAX_THREADS_1D = ((int64_t)1 << 32) - 256;   // one-dimensional grids: grid x block < 2^32

int esize(int dt) {
  switch (dt) {
    case STARKV_F16: case STARKV_BF16: return 2;
    case STARKV_F32: return 4;
    case STARKV_I8: case STARKV_U8: return 1;
    default: return 0;
  }
}
bool al(const void* p, int n) { return ((uintptr_t)p % (uintptr_t)n) == 0; }
bool al64(int64_t v, int n) { return v % n == 0; }

size_t a256(size_t x) { return (x + 255) & ~(size_t)255; }

// Compute units of the current device, the unit of every launch plan below
// (rounds of resident workgroups), read once per device.  A partitioned GPU
// or another part reports fewer; with no device to ask (argument validation
// on a machine without a GPU) the plan assumes a whole MI355X.
int device_cus() {
  constexpr int MAXD = 64;
  static std::mutex mu;
  static int cus[MAXD] = {};
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= MAXD) return FULL_CHIP_CUS;
  std::lock_guard<std::mutex> lk(mu);
  if (!cus[dev]) {
    int n = 0;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n < 1)
      n = FULL_CHIP_CUS;
    cus[dev] = n;
  }
  return cus[dev];
}

// Choose how many position splits minimise the modelled time of a launch of
// `groups` independent (batch, plan) groups over `n_units` position units:
// rounds of `slots` concurrent workgroups, each costing its units plus a fixed
// `c0` units (setup, pipeline fill), times (1 + frac_per_split * splits) for
// split partials written and re-read.
int choose_splits(int64_t groups, int slots, int n_units, int max_n, double c0, double frac_per_split) {
  int best = 1;
  double best_t = 1e300;
  int last = 0;
  for (int n = 1; n <= std::max(1, std::min(max_n, n_units)); ++n) {
    const int len = (n_units + n - 1) / n;
    if (len == last) continue;                     // the same plan again
    last = len;
    const int ne = (int)ceil_div(n_units, len);
    const int64_t rounds = ceil_div(groups * ne, slots);
    const double t = (double)rounds * (len + c0) * (1.0 + frac_per_split * ne);
    if (t < best_t * 0.9999) { best_t = t; best = ne; }
  }
  return best;
}

struct KPlan {
  int n_wg = 0;
  int per_cu = K1_WG_PER_CU;   // K1 workgroups resident per CU (the grouped-query kernel: two)
  bool fast = false;
};

int validate_klayout(const starkv_klatent& k, int dtype);

int validate_klatent(const starkv_klatent& k, int Hq, int dtype, int* gs_out) {
  if (k.n_kv_heads < 1 || k.n_kv_heads > K_MAX_KV) return k.n_kv_heads < 1 ? STARKV_ERR_SHAPE : STARKV_ERR_LIMIT;
  if (Hq < 1 || Hq % k.n_kv_heads) return STARKV_ERR_SHAPE;
  if (Hq > K_MAX_QH) return STARKV_ERR_LIMIT;
  if (!k.bk_head_offset || !k.bk) return STARKV_ERR_NULL;
  if (k.bk_row_stride < HEAD_DIM) return STARKV_ERR_SHAPE;
  const int st = validate_klayout(k, dtype);
  if (st) return st;
  *gs_out = Hq / k.n_kv_heads;
  return STARKV_OK;
}

// Where the K latent lives and how it is stored (shared by the attention
// entry points and the cache writer).
int validate_klayout(const starkv_klatent& k, int dtype) {
  if (k.n_kv_heads < 1 || k.n_kv_heads > K_MAX_KV) return k.n_kv_heads < 1 ? STARKV_ERR_SHAPE : STARKV_ERR_LIMIT;
  if (!k.rank || !k.head_offset || !k.pos_stride) return STARKV_ERR_NULL;
  if (!k.data) return STARKV_ERR_NULL;
  if (k.format != STARKV_FMT_DENSE && k.format != STARKV_FMT_INT8_SYM && k.format != STARKV_FMT_INT4_REF)
    return STARKV_ERR_FORMAT;
  if (dtype != STARKV_F16 && dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  for (int h = 0; h < k.n_kv_heads; ++h)
    if (k.rank[h] < 1 || k.rank[h] > 128) return STARKV_ERR_RANK;
  if (k.stride_b < 0) return STARKV_ERR_SHAPE;
  if (k.format == STARKV_FMT_DENSE) {
    for (int h = 0; h < k.n_kv_heads; ++h)
      if (k.pos_stride[h] < k.rank[h] || k.head_offset[h] < 0) return STARKV_ERR_SHAPE;
  } else {
    // quantised: any rank and any byte layout (rows that are not aligned for
    // whole 8-byte (int8) / 4-byte (int4) chunks, or ranks that are not a
    // multiple of 8, take the unaligned-row loads: k_quant_aligned)
    if (!k.scale) return STARKV_ERR_NULL;
    const bool two = k.format == STARKV_FMT_INT4_REF && k.split > 0;
    if (two && (k.split % 16 || k.split > 128)) return STARKV_ERR_SHAPE;
    if (two && k.split_format != STARKV_FMT_INT4_REF && k.split_format != STARKV_FMT_INT8_SYM) return STARKV_ERR_FORMAT;
    const int split = two ? k.split : 128;
    const bool a8 = two ? k.split_format == STARKV_FMT_INT8_SYM : k.format == STARKV_FMT_INT8_SYM;
    if (!al(k.scale, 2)) return STARKV_ERR_ALIGN;
    if (k.scale_stride_b < 0 || k.scale_stride_h < 0) return STARKV_ERR_SHAPE;
    bool any_lo = false;
    for (int h = 0; h < k.n_kv_heads; ++h) {
      const int r = k.rank[h];
      const int ra = std::min(r, split);
      if (k.head_offset[h] < 0 || k.pos_stride[h] < (a8 ? ra : (ra + 1) / 2)) return STARKV_ERR_SHAPE;
      any_lo |= r > split;
    }
    if (any_lo) {
      if (!k.data2 || !k.scale2 || !k.head_offset2 || !k.pos_stride2) return STARKV_ERR_NULL;
      if (!al(k.scale2, 2)) return STARKV_ERR_ALIGN;
      if (k.stride2_b < 0 || k.scale2_stride_b < 0 || k.scale2_stride_h < 0) return STARKV_ERR_SHAPE;
      for (int h = 0; h < k.n_kv_heads; ++h) {
        if (k.rank[h] <= split) continue;
        if (k.head_offset2[h] < 0 || k.pos_stride2[h] < (k.rank[h] - split + 1) / 2) return STARKV_ERR_SHAPE;
      }
    }
  }
  return STARKV_OK;
}

// Quantised K whose rows take whole 8-byte (int8) / 4-byte (int4) chunk loads:
// ranks multiples of 8 and every row start aligned to the chunk size.
bool k_quant_aligned(const starkv_klatent& k) {
  const bool two = k.format == STARKV_FMT_INT4_REF && k.split > 0;
  const int split = two ? k.split : 128;
  const bool a8 = two ? k.split_format == STARKV_FMT_INT8_SYM : k.format == STARKV_FMT_INT8_SYM;
  const int al_a = a8 ? 8 : 4;
  if (!al(k.data, al_a) || !al64(k.stride_b, al_a)) return false;
  bool any_lo = false;
  for (int h = 0; h < k.n_kv_heads; ++h) {
    if (k.rank[h] % 8) return false;
    if (!al64(k.head_offset[h], al_a) || !al64(k.pos_stride[h], al_a)) return false;
    any_lo |= k.rank[h] > split;
  }
  if (any_lo) {
    if (!al(k.data2, 4) || !al64(k.stride2_b, 4)) return false;
    for (int h = 0; h < k.n_kv_heads; ++h)
      if (k.rank[h] > split && (!al64(k.head_offset2[h], 4) || !al64(k.pos_stride2[h], 4))) return false;
  }
  return true;
}

// Dense head whose rows the streaming kernels stage in whole 16-byte pieces:
// rank a multiple of 8 (or a padded copy), rows 16-byte aligned in every batch.
bool ws_rows16(const starkv_klatent& k, int h, int xe, bool padded) {
  return al(k.data, 16) && al64(k.stride_b * xe, 16) && (k.rank[h] % 8 == 0 || padded) &&
         al64(k.head_offset[h] * xe, 16) && al64(k.pos_stride[h] * xe, 16);
}
// Other dense heads with contiguous rows are staged as runs of bytes (see
// KArgs::klin) by the same kernels instead of being copied into aligned rows
// or read element by element by the register-streaming kernel (8 KV heads of
// rank 102, groups of 4, B1 S65536: 83 us a call with the copy, 55 us without;
// 32 heads of odd ranks, B3 S5003: the decode call 148 against 111 us, its K
// logits 69 us before).  Below 8 ranks a row holds no whole chunk.  The grouped-query kernel stages either
// all heads of a launch so or none, and its DMA slots hold two linear heads of
// up to 127 ranks.  decode: up to 8192 positions of one-query heads below 16
// ranks, fewer than 384 in all, stay with the register-streaming kernel, whose
// few loads start sooner (decode calls, staged against streamed, us: 32 heads
// of rank 10, S4099 37.5 / 35.3, S65536 68.6 / 73.3; of rank 14, S4099 37.8 /
// 38.3; 8 heads of rank 15, S4099 32.4 / 31.7, of rank 20 32.6 / 33.1; 31
// heads of rank 9 beside one of 127, S4099 36.6 / 42.3).
bool ws_linear(const starkv_klatent& k, int h, int gs) {
  return k.format == STARKV_FMT_DENSE && k.pos_stride[h] == k.rank[h] && k.rank[h] >= 8 && k.rank[h] <= (gs > 1 ? 127 : 128) &&
         al(k.data, 2);
}
// The heads of a dense launch staged as runs of bytes; ok: every head is
// staged in one form or the other.
struct LinPlan {
  bool ok;
  uint64_t mask;
};
LinPlan lin_plan(const starkv_klatent& k, int gs, int xe, int S, bool padded, bool decode) {
  LinPlan p = {true, 0};
  bool all = true;
  int ranks = 0, rmax = 0;
  for (int h = 0; h < k.n_kv_heads; ++h) {
    const bool l = ws_linear(k, h, gs);
    all = all && l;
    ranks += k.rank[h];
    rmax = std::max(rmax, k.rank[h]);
    if (ws_rows16(k, h, xe, padded)) continue;
    if (!l) return {false, 0};
    p.mask |= (uint64_t)1 << h;
  }
  if (p.mask && gs == 1 && decode && rmax < 16 && ranks < 384 && S <= 8192) return {false, 0};
  if (p.mask && gs > 1) {
    if (!all) return {false, 0};
    for (int h = 0; h < k.n_kv_heads; ++h) p.mask |= (uint64_t)1 << h;
  }
  return p;
}

// Warp-specialised K-logit kernel: dense latents with 16-byte aligned rows
// (ranks a multiple of 8) or contiguous ones (ws_linear), or int8 latents with one scale per (b, h, s) whose
// rows start on 16-byte boundaries (pitch a multiple of 16 bytes, so the 16-byte
// DMA pieces never straddle rows); q and B_k are read element-wise there.
// padded: dense rows hold round_up(r, 8) elements, zero past r (the K-logit
// entry's repacked copy), so a rank need not be a multiple of 8.
bool k_ws(const starkv_klatent& k, int gs, int dtype, int S, bool padded, bool decode) {
  const bool i8 = k.format == STARKV_FMT_INT8_SYM;
  if (k.format != STARKV_FMT_DENSE && !i8) return false;
  const int xe = i8 ? 1 : esize(dtype);
  if (i8 && (!al(k.data, 16) || !al64(k.stride_b * xe, 16))) return false;
  // int8: the scales of a tile are staged in 16-byte pieces (8 positions), so
  // each (b, h) scale row is read up to position round_up(S, 8) - 1, inside
  // its pitch
  if (i8 && (!al(k.scale, 16) || !al64(k.scale_stride_b * 2, 16) || !al64(k.scale_stride_h * 2, 16) ||
             k.scale_stride_h < round_up(S, 8)))
    return false;
  for (int h = 0; h < k.n_kv_heads; ++h) {
    if (i8 && (k.rank[h] % 8 || !al64(k.head_offset[h], 16) || !al64(k.pos_stride[h], 16))) return false;
    if ((int64_t)TILE * k.pos_stride[h] * xe >= ((int64_t)1 << 31)) return false;   // 32-bit per-tile DMA step
  }
  return i8 || lin_plan(k, gs, xe, S, padded, decode).ok;
}

// 16-byte LDS chunks of one 32-position tile row of a head in that kernel
int ws_row_chunks(const starkv_klatent& k, int h) {
  return (int)ceil_div(k.rank[h], k.format == STARKV_FMT_INT8_SYM ? 16 : 8);
}

// First-fit decreasing of heads hs (u[h] units each) into at most nb bins of
// cap units; false if they do not fit.
static bool ffd_bins(std::vector<int> hs, const std::vector<int>& u, int nb, int cap,
                     std::vector<std::vector<int>>* out) {
  std::stable_sort(hs.begin(), hs.end(), [&](int x, int y) { return u[x] > u[y]; });
  std::vector<std::vector<int>> bins;
  std::vector<int> load;
  for (int h : hs) {
    size_t i = 0;
    while (i < bins.size() && load[i] + u[h] > cap) ++i;
    if (i == bins.size()) {
      if ((int)bins.size() == nb) return false;
      bins.emplace_back();
      load.push_back(0);
    }
    bins[i].push_back(h);
    load[i] += u[h];
  }
  if (out) *out = bins;
  return true;
}

// MHA query heads over workgroups of up to nw bins of cap units each, so that
// the largest workgroup stages as few 16-byte chunks per tile as possible (a
// single round of workgroups runs at the pace of the heaviest): longest first
// into the least loaded workgroup where its heads still pack, then single
// moves and pairwise swaps off the heaviest workgroup while they lower its
// load.  Starts from n_min workgroups, one more while the greedy pass does not
// fit.  Results are cached per (rank vector, geometry).
static bool ws_balance(const starkv_klatent& k, int Hq, int unit, int nw, int cap, int n_min,
                       std::vector<std::vector<int>>& parts) {
  std::vector<int> u(Hq), c(Hq), order(Hq);
  std::vector<int> key = {Hq, unit, nw, cap, n_min};
  for (int h = 0; h < Hq; ++h) {
    u[h] = (int)ceil_div(k.rank[h], unit);
    c[h] = ws_row_chunks(k, h);
    order[h] = h;
    key.push_back(c[h]);
    key.push_back(u[h]);
  }
  static std::mutex mu;
  static std::vector<std::pair<std::vector<int>, std::vector<std::vector<int>>>> cache;
  {
    std::lock_guard<std::mutex> lk(mu);
    for (const auto& e : cache)
      if (e.first == key) { parts = e.second; return true; }
  }
  std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return c[x] > c[y]; });
  auto fits = [&](const std::vector<int>& hs) { return ffd_bins(hs, u, nw, cap, nullptr); };
  for (int n = std::max(n_min, 1); n * nw <= K_MAX_WAVES; ++n) {
    parts.assign(n, {});
    std::vector<int> load(n, 0);
    bool ok = true;
    for (int h : order) {
      int best = -1;
      for (int g = 0; g < n; ++g) {
        if (best >= 0 && load[g] >= load[best]) continue;
        std::vector<int> t = parts[g];
        t.push_back(h);
        if (fits(t)) best = g;
      }
      if (best < 0) { ok = false; break; }
      parts[best].push_back(h);
      load[best] += c[h];
    }
    if (!ok) continue;
    for (int iter = 0; iter < 256; ++iter) {
      const int g = (int)(std::max_element(load.begin(), load.end()) - load.begin());
      bool moved = false;
      for (int o = 0; o < n && !moved; ++o) {
        if (o == g) continue;
        for (size_t i = 0; i < parts[g].size() && !moved; ++i) {
          const int h = parts[g][i];
          std::vector<int> rest = parts[g];
          rest.erase(rest.begin() + i);
          std::vector<int> grown = parts[o];
          grown.push_back(h);
          if (load[o] + c[h] < load[g] && fits(grown)) {           // move h to o
            parts[g] = rest; parts[o] = grown;
            load[g] -= c[h]; load[o] += c[h];
            moved = true;
            break;
          }
          for (size_t j = 0; j < parts[o].size(); ++j) {           // swap h with a lighter head of o
            const int h2 = parts[o][j], d = c[h] - c[h2];
            if (d <= 0 || load[o] + d >= load[g]) continue;
            std::vector<int> a2 = rest, b2 = parts[o];
            a2.push_back(h2);
            b2[j] = h;
            if (fits(a2) && fits(b2)) {
              parts[g] = a2; parts[o] = b2;
              load[g] -= d; load[o] += d;
              moved = true;
              break;
            }
          }
        }
      }
      if (!moved) break;
    }
    std::lock_guard<std::mutex> lk(mu);
    if (cache.size() >= 64) cache.erase(cache.begin());
    cache.emplace_back(key, parts);
    return true;
  }
  return false;
}

// Pack (query head, 32-rank M-tile) items into waves of up to 2 or 4 items
// (first fit decreasing, whole heads per wave; 4 once any head has rank > 64)
// and deal the waves round-robin over workgroups of 8 waves (2-item waves) or
// 4 waves (4-item waves).
int build_k_plan(const starkv_klatent& k, int Hq, int gs, int dtype, int S, KArgs& a, KPlan& plan,
                 bool padded, bool decode) {
  const bool ws = k_ws(k, gs, dtype, S, padded, decode);
  const int unit = 32;                        // ranks per item
  struct QH { int qh, kv, ni; };              // ni: items of the head
  std::vector<QH> heads;
  int max_items = 1;
  for (int qh = 0; qh < Hq; ++qh) {
    const int kv = qh / gs;
    max_items = std::max(max_items, (int)ceil_div(k.rank[kv], 32));
    heads.push_back({qh, kv, (int)ceil_div(k.rank[kv], unit)});
  }
  const int maxi = ws || max_items > 2 ? 4 : 2;   // items per (consumer) wave
  const int nw = maxi == 2 ? 8 : 4;
  const int cap = maxi * 32 / unit;               // units per wave
  // Bins of up to cap units (whole query heads), first-fit decreasing.  With
  // GQA the query heads of one KV head are packed together (KV-major), so the
  // workgroup that stages or streams that head's latent serves all of them.
  std::vector<std::vector<QH>> bins;
  std::vector<int> load;
  auto pack = [&](const std::vector<QH>& hs) {
    const size_t first = bins.size();
    for (const QH& h : hs) {
      size_t i = first;
      for (; i < bins.size(); ++i) if (load[i] + h.ni <= cap) break;
      if (i == bins.size()) { bins.emplace_back(); load.push_back(0); }
      bins[i].push_back(h);
      load[i] += h.ni;
    }
  };
  if (gs == 1) {
    std::stable_sort(heads.begin(), heads.end(), [](const QH& x, const QH& y) { return x.ni > y.ni; });
    pack(heads);
  } else {
    for (int kv = 0; kv < k.n_kv_heads; ++kv) {
      std::vector<QH> grp;
      for (const QH& h : heads) if (h.kv == kv) grp.push_back(h);
      pack(grp);
    }
  }
  int n_waves = (int)bins.size();
  plan.n_wg = (int)ceil_div(n_waves, nw);
  if (plan.n_wg * nw > K_MAX_WAVES) return STARKV_ERR_LIMIT;
  // bin -> (workgroup, wave).  MHA: the heaviest bins (latent rank sum) first,
  // each into the least loaded workgroup with a free wave, so workgroups
  // stream similar byte counts.  GQA: consecutive bins share a workgroup.
  // Warp-specialised MHA: heads are partitioned over the workgroups first
  // (ws_balance), then packed into bins per workgroup.
  std::vector<int> wg_of(n_waves), wave_of(n_waves);
  std::vector<std::vector<int>> parts;
  if (ws && gs == 1 && ws_balance(k, Hq, unit, nw, cap, plan.n_wg, parts)) {
    bins.clear();
    wg_of.clear();
    wave_of.clear();
    for (int g = 0; g < (int)parts.size(); ++g) {
      std::vector<int> u(Hq, 0);
      for (int h : parts[g]) u[h] = (int)ceil_div(k.rank[h], unit);
      std::vector<std::vector<int>> wb;
      ffd_bins(parts[g], u, nw, cap, &wb);
      for (int w = 0; w < (int)wb.size(); ++w) {
        std::vector<QH> bin;
        for (int h : wb[w]) bin.push_back({h, h, u[h]});
        bins.push_back(bin);
        wg_of.push_back(g);
        wave_of.push_back(w);
      }
    }
    n_waves = (int)bins.size();
    plan.n_wg = (int)parts.size();
  } else if (gs == 1) {
    std::vector<int> order(n_waves), rsum(n_waves, 0);
    for (int bi = 0; bi < n_waves; ++bi) {
      order[bi] = bi;
      for (const QH& h : bins[bi]) rsum[bi] += k.rank[h.kv];
    }
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return rsum[x] > rsum[y]; });
    std::vector<int64_t> wload(plan.n_wg, 0);
    std::vector<int> used(plan.n_wg, 0);
    for (int bi : order) {
      int best = -1;
      for (int g = 0; g < plan.n_wg; ++g)
        if (used[g] < nw && (best < 0 || wload[g] < wload[best])) best = g;
      wg_of[bi] = best;
      wave_of[bi] = used[best]++;
      wload[best] += rsum[bi];
    }
  } else {
    for (int bi = 0; bi < n_waves; ++bi) { wg_of[bi] = bi / nw; wave_of[bi] = bi % nw; }
  }
  for (int w = 0; w < K_MAX_WAVES; ++w)
    for (int i = 0; i < K_MAXI; ++i) a.items[w][i] = 0;
  for (int bi = 0; bi < n_waves; ++bi) {
    std::vector<QH> v = bins[bi];
    std::sort(v.begin(), v.end(), [](const QH& x, const QH& y) { return x.qh < y.qh; });
    uint32_t* row = a.items[wg_of[bi] * nw + wave_of[bi]];
    int i = 0;
    for (const QH& h : v) {
      const int r = k.rank[h.kv];
      for (int mt = 0; mt < h.ni; ++mt) row[i++] = item_pack(h.qh, h.kv, mt, std::min(32, r - 32 * mt), mt == h.ni - 1);
    }
  }
  // grouped-query heads (k_logits_gqa.hip): K reconstructed once per KV
  // head; two KV heads per workgroup (the largest rank with the smallest),
  // each run by two consumer waves (dims halves p = 0, 1)
  const bool gqa = ws && gs > 1 && gs <= 8 && k.format == STARKV_FMT_DENSE;
  if (gqa) {
    const int n = k.n_kv_heads;
    std::vector<int> order(n);
    for (int h = 0; h < n; ++h) order[h] = h;
    std::stable_sort(order.begin(), order.end(), [&](int x, int y) { return k.rank[x] > k.rank[y]; });
    plan.n_wg = (int)ceil_div(n, 2);
    plan.per_cu = 2;
    if (plan.n_wg * 4 > K_MAX_WAVES) return STARKV_ERR_LIMIT;
    for (int w = 0; w < K_MAX_WAVES; ++w)
      for (int i = 0; i < K_MAXI; ++i) a.items[w][i] = 0;
    for (int g = 0; g < plan.n_wg; ++g) {
      const int h0 = order[g], h1 = n - 1 - g > g ? order[n - 1 - g] : -1;
      for (int p = 0; p < 2; ++p) {
        a.items[g * 4 + p][0] = item_pack(h0 * gs, h0, p, 0, 1);
        if (h1 >= 0) a.items[g * 4 + 2 + p][0] = item_pack(h1 * gs, h1, p, 0, 1);
      }
    }
  }
  a.gqa = gqa;
  a.gs = gs;
  a.klin = ws && k.format == STARKV_FMT_DENSE ? lin_plan(k, gs, esize(dtype), S, padded, decode).mask : 0;
  for (int h = 0; h < K_MAX_KV; ++h) a.krank[h] = (int16_t)(h < k.n_kv_heads ? k.rank[h] : 0);
  const bool two = k.format == STARKV_FMT_INT4_REF && k.split > 0;
  a.ksplit = two ? k.split : 128;
  a.k_a_int8 = two ? k.split_format == STARKV_FMT_INT8_SYM : k.format == STARKV_FMT_INT8_SYM;
  a.x2 = k.data2; a.x2_sb = k.stride2_b;
  a.xscale2 = k.scale2; a.xs2_sb = k.scale2_stride_b; a.xs2_sh = k.scale2_stride_h;
  for (int h = 0; h < k.n_kv_heads; ++h) {
    a.xoff[h] = k.head_offset[h];
    a.xpitch[h] = (int)k.pos_stride[h];
    a.bkoff[h] = k.bk_head_offset[h];
    const bool lo = two && k.rank[h] > k.split;
    a.xoff2[h] = lo ? k.head_offset2[h] : 0;
    a.xpitch2[h] = lo ? (int)k.pos_stride2[h] : 0;
  }
  a.n_wg = plan.n_wg;
  a.maxi = maxi;
  a.ws = ws;
  a.ws_i8 = ws && k.format == STARKV_FMT_INT8_SYM;
  a.ws_stage = a.ws_nst = 0;
  if (ws) {
    // stage = the largest workgroup's latent tile (16-byte chunks of its
    // distinct KV heads, whole 1 KB DMA pieces) [+ 1 KB of int8 scales:
    // 32 positions of up to 16 heads] + the 8 KB RoPE operand
    int max_chunks = 0;
    for (int g = 0; g < plan.n_wg; ++g) {
      bool seen[K_MAX_KV] = {};
      int chunks = 0;
      for (int w = 0; w < nw; ++w)
        for (int i = 0; i < K_MAXI; ++i) {
          const uint32_t it = a.items[g * nw + w][i];
          const int kv = (it >> 8) & 0xff;
          if (!((it >> 27) & 1) || seen[kv]) continue;
          seen[kv] = true;
          chunks += (a.klin >> kv) & 1 ? (gqa ? (int)round_up(lin_chunks(k.rank[kv]), 64) : lin_chunks(k.rank[kv])) : 32 * ws_row_chunks(k, kv);
        }
      max_chunks = std::max(max_chunks, chunks);
    }
    a.ws_stage = (int)round_up(max_chunks, 64) * 16 + 8192 + (a.ws_i8 ? 1024 : 0);
    a.ws_nst = gqa ? std::min(6, K1_GQ_RING_BYTES / a.ws_stage) : std::min(4, (a.ws_i8 ? K1_WS_RING_I8_BYTES : K1_WS_RING_BYTES) / a.ws_stage);
  }
  return STARKV_OK;
}

// Vector-load variant: B_k and q rows 8-byte aligned, and latent rows aligned
// for whole-chunk loads with ranks a multiple of 8 (dense: 16-byte rows;
// quantised: k_quant_aligned).
bool k_fast(const starkv_klatent& k, int dtype, const void* q, int64_t q_sb, int64_t q_sh) {
  const bool dense = k.format == STARKV_FMT_DENSE;
  const int xe = esize(dtype);
  if (!dense && !k_quant_aligned(k)) return false;
  if (dense && (!al(k.data, 16) || !al64(k.stride_b * xe, 16))) return false;
  for (int h = 0; h < k.n_kv_heads; ++h) {
    if (dense && k.rank[h] % 8) return false;
    if (dense && (!al64(k.head_offset[h] * xe, 16) || !al64(k.pos_stride[h] * xe, 16))) return false;
    if (!al64(k.bk_head_offset[h] * 2, 8)) return false;
  }
  if (!al(k.bk, 8) || !al64(k.bk_row_stride * 2, 8)) return false;
  if (!al(q, 8) || !al64(q_sb * 2, 8) || !al64(q_sh * 2, 8)) return false;
  return true;
}

int check_mask(const void* mask, int mask_dtype) {
  if (!mask) return STARKV_OK;
  if (mask_dtype != STARKV_F32 && mask_dtype != STARKV_F16 && mask_dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  return STARKV_OK;
}


// ---- P.V geometry: workgroup = 4 waves x NTW column tiles of one position chunk
struct PVGeom {
  int Rvp, n_cb, n_c2, c2_len, n_grp;   // n_grp > 1: two-level split reduction
  int ntw;                              // column tiles per wave
};

// row_bytes: the largest row pitch (bytes) of the V latent's streams; the
// kernel addresses a chunk with 32-bit offsets, so a chunk stays below 2 GB
// ntw: column tiles per wave (0: as the storage kind asks; given behind a shared prefix, where a partial costs four times
// as much: the join reads it again with few workgroups, 8 x 333 of bf16 27 us -> 24, 4 x 1024 22 -> 20, twelve times 24 and 22)
PVGeom pv_geometry(int B, int S, int Rv, bool fused, int vq, int64_t row_bytes, int ntw = 0) {
  PVGeom g;
  g.Rvp = (int)round_up(Rv, 32);
  const double part_cost = ntw ? 4.0 : 1.0;
  if (!ntw) ntw = pv_tiles_per_wave(g.Rvp, fused, vq);
  g.ntw = ntw;
  // one 8-wave workgroup for all columns (its 24-bit row offsets need
  // every pitch below 16 MB)
  const bool wide = pv_wide_tiles(g.Rvp, fused, vq) > 0 && row_bytes < V_MAX_PITCH;
  // fused group-64 V of up to 16 tiles: the 4-wave raw-nibble kernel, three per CU
  const bool nib4 = fused && vq == VQ_G64 && g.Rvp <= 512;
  // the block formats' raw kernel: all columns, one 8-wave workgroup per CU
  const bool raw = vq == VQ_RAW;
  g.n_cb = wide || raw ? 1 : (int)ceil_div(g.Rvp / 32, 4 * ntw);
  const int wg_per_cu = wide || raw ? 1 : nib4 ? 3 : pv_wg_per_cu(ntw, vq);
  const int n_ks = (int)ceil_div(S, KSTEP);
  // each extra split writes and re-reads one fp32 partial of 32 x Rvp per
  // column block, against the X_v bytes and logits the split streams
  const double vbytes = vq == VQ_DENSE ? 2.0 * Rv : Rv / 2.0 + 4.0 * ceil_div(Rv, 64);
  // (below ~8K positions the launch is latency-bound and partials are cheap)
  const double frac = 32.0 * g.Rvp * 8.0 / g.n_cb / ((double)std::max(S, 8192) * (vbytes / g.n_cb + 128.0));
  int n = choose_splits((int64_t)B * g.n_cb, device_cus() * wg_per_cu, n_ks, 512, 4.0, part_cost * frac);
  const int64_t max_ks = std::max<int64_t>(1, ((int64_t)1 << 31) / std::max<int64_t>(row_bytes, 1) / KSTEP);
  n = std::max<int64_t>(n, ceil_div(n_ks, max_ks));
  g.c2_len = (int)ceil_div(n_ks, n) * KSTEP;
  // the all-columns and raw-nibble kernels take whole 32-position steps (a
  // chunk still below 2 GB)
  if (wide || nib4 || raw) g.c2_len = (int)std::min<int64_t>(round_up(g.c2_len, 2 * KSTEP), std::max<int64_t>(2 * KSTEP, max_ks * KSTEP / (2 * KSTEP) * (2 * KSTEP)));
  g.n_c2 = (int)ceil_div(S, g.c2_len);
  g.n_grp = g.n_c2 > PV_RG ? (int)ceil_div(g.n_c2, PV_RG) : 0;
  return g;
}

// ---- decode workspace layout (shared by the size query and the call)
int head_groups(int H) { return (int)ceil_div(H, 32); }   // P.V passes of 32 heads

struct DecodeLayout {
  int S_pad, n_c1, tiles_per_chunk, n_hg, sw, n_sl, n_cs;
  PVGeom pv;
  bool part16;
  size_t off_logits, off_cmax, off_part, off_psum, off_ypart, total;
};

// f16: fp16 model.  Short P.V chunks (<= 512 positions) then keep their
// partials in fp16, each divided by its chunk's softmax sum (a convex
// combination of V rows: bounded by max |V|): there the partials are a large
// share of the P.V traffic (at 272 positions about as many bytes as the
// int4 V latent) and halving them pays for the per-chunk rescale in the
// up-projection.  With long chunks the time comes out even (measured); group-64
// V keeps them in fp16 there too, halving the partials' share of its traffic
// (55 of 613 MB at B16 S32768), dense V in fp32.
DecodeLayout decode_layout(int B, int Hq, int Hkv, int S, int Rv, int n_wg, int k1pc, int vq, int64_t v_row_bytes,
                           bool f16, int pv_ntw = 0) {
  DecodeLayout L;
  L.S_pad = (int)round_up(S, 64);
  const int n_tiles = (int)ceil_div(S, TILE);
  const int cus = device_cus();
  L.n_c1 = choose_splits((int64_t)B * n_wg, cus * k1pc, n_tiles, 256, 3.0, 0.0);
  L.tiles_per_chunk = (int)ceil_div(n_tiles, L.n_c1);
  L.n_c1 = (int)ceil_div(n_tiles, L.tiles_per_chunk);
  L.n_hg = head_groups(Hq);
  L.pv = pv_geometry(B * L.n_hg, S, Rv, true, vq, v_row_bytes, pv_ntw);
  L.sw = up_slice_width(Hkv, Rv, cus);
  L.n_sl = (int)ceil_div(Rv, L.sw);
  L.n_cs = up_chunk_sets(Hkv, L.n_sl, L.pv.n_c2, cus);
  const int Rvp = L.pv.Rvp, n_c2 = L.pv.n_c2;
  const size_t BQ = (size_t)B * L.n_hg;
  size_t o = 0;
  L.off_logits = o; o = a256(o + (size_t)B * Hq * L.S_pad * 4);
  L.off_cmax = o; o = a256(o + (size_t)B * Hq * L.n_c1 * 4);
  const bool part16 = f16 && (L.pv.c2_len <= 512 || vq == VQ_G64);
  L.part16 = part16;
  L.off_part = o; o = a256(o + BQ * n_c2 * 32 * Rvp * (part16 ? 2 : 4));
  L.off_psum = o; o = a256(o + BQ * n_c2 * 32 * 4);
  L.off_ypart = o; o = a256(o + (size_t)Hkv * L.n_sl * L.n_cs * ((size_t)B * (Hq / Hkv)) * HEAD_DIM * 4);
  L.total = o;
  return L;
}

// V latent: validate the description and fill the P.V kernel's storage
// fields (x / x2 / scales / zero points, split, bytes per row); *vq = its
// storage kind.  Quantised formats take any rank and byte layout (the
// per-token block formats need a split that is a multiple of 8, so an 8-rank
// chunk never straddles it); pa.qfast tells whether every row is aligned for
// whole 4-byte (int4) / 8-byte (int8) chunk loads with ranks (and the lower
// block) a multiple of 8, else the P.V kernel reads unaligned rows.
int validate_v(const starkv_vlatent& v, PVArgs& pa, int* vq) {
  if (!v.data) return STARKV_ERR_NULL;
  if (v.rank < 1 || v.rank > MAX_RV) return STARKV_ERR_RANK;
  if (v.stride_b < 0 || v.stride_s < 0) return STARKV_ERR_SHAPE;
  pa.x = v.data; pa.x_sb = v.stride_b; pa.x_ss = v.stride_s;
  switch (v.format) {
    case STARKV_FMT_DENSE:
      if (v.stride_s < v.rank) return STARKV_ERR_SHAPE;
      *vq = VQ_DENSE;
      return STARKV_OK;
    case STARKV_FMT_INT4_REF:
    case STARKV_FMT_INT8_SYM: {
      if (!v.scale) return STARKV_ERR_NULL;
      const bool two = v.format == STARKV_FMT_INT4_REF && v.split > 0 && v.split < v.rank;
      if (two && v.split_format != STARKV_FMT_INT4_REF && v.split_format != STARKV_FMT_INT8_SYM)
        return STARKV_ERR_FORMAT;
      const int split = two ? v.split : v.rank;
      const bool a8 = two ? v.split_format == STARKV_FMT_INT8_SYM : v.format == STARKV_FMT_INT8_SYM;
      if (two && split % 8) return STARKV_ERR_SHAPE;
      const int al_a = a8 ? 8 : 4;
      const int nb = a8 ? split : (split + 1) / 2;
      if (v.stride_s < nb) return STARKV_ERR_SHAPE;
      if (!al(v.scale, 2)) return STARKV_ERR_ALIGN;
      if (v.scale_stride_b < 0 || v.scale_stride_s < 0) return STARKV_ERR_SHAPE;
      pa.split = split; pa.a_int8 = a8; pa.xnb = nb;
      pa.xs = v.scale; pa.xs_sb = v.scale_stride_b; pa.xs_ss = v.scale_stride_s;
      bool fast = split % 8 == 0 && al(v.data, al_a) && al64(v.stride_s, al_a) && al64(v.stride_b, al_a);
      if (two) {
        const int nb2 = (v.rank - split + 1) / 2;
        if (!v.data2 || !v.scale2) return STARKV_ERR_NULL;
        if (v.stride2_s < nb2 || v.stride2_b < 0 || v.scale2_stride_b < 0 || v.scale2_stride_s < 0)
          return STARKV_ERR_SHAPE;
        if (!al(v.scale2, 2)) return STARKV_ERR_ALIGN;
        pa.x2 = v.data2; pa.x2_sb = v.stride2_b; pa.x2_ss = v.stride2_s; pa.x2nb = nb2;
        pa.xs2 = v.scale2; pa.xs2_sb = v.scale2_stride_b; pa.xs2_ss = v.scale2_stride_s;
        fast = fast && (v.rank - split) % 8 == 0 && al(v.data2, 4) && al64(v.stride2_s, 4) && al64(v.stride2_b, 4);
      }
      pa.qfast = fast;
      *vq = VQ_BLOCK;
      return STARKV_OK;
    }
    case STARKV_FMT_INT4_G64: {
      if (!v.scale || !v.zero) return STARKV_ERR_NULL;
      const int nb = (v.rank + 1) / 2;
      if (v.stride_s < nb || v.scale_stride_s < (v.rank + 63) / 64 || v.scale_stride_b < 0)
        return STARKV_ERR_SHAPE;
      if (!al(v.scale, 2) || !al(v.zero, 2)) return STARKV_ERR_ALIGN;
      if (v.stride_s >= V_MAX_PITCH || v.scale_stride_s * 2 >= V_MAX_PITCH) return STARKV_ERR_LIMIT;
      pa.xs = v.scale; pa.xs_sb = v.scale_stride_b; pa.xs_ss = v.scale_stride_s;
      pa.xz = v.zero; pa.xnb = nb;
      pa.qfast = v.rank % 8 == 0 && al(v.data, 4) && al64(v.stride_s, 4) && al64(v.stride_b, 4);
      *vq = VQ_G64;
      return STARKV_OK;
    }
    default:
      return STARKV_ERR_FORMAT;
  }
}

// the P.V kernel's aligned-row variant: dense rows 16-byte aligned with the
// rank a multiple of 8; quantised rows as validate_v found them (pa.qfast)
bool v_fast(const starkv_vlatent& v, const PVArgs& pa) {
  if (v.format != STARKV_FMT_DENSE) return pa.qfast != 0;
  return al(v.data, 16) && al64(v.stride_s * 2, 16) && al64(v.stride_b * 2, 16) && v.rank % 8 == 0 &&
         v.stride_s * 2 < V_MAX_PITCH;
}

// largest row pitch in bytes over the V latent's streams (dense: 16-bit elements)
int64_t v_row_bytes(const starkv_vlatent& v) {
  if (v.format == STARKV_FMT_DENSE) return v.stride_s * 2;
  return std::max({v.stride_s, v.scale_stride_s * 2, v.stride2_s, v.scale2_stride_s * 2});
}

// The unaligned dense P.V rows of a 16-position step are addressed with 32-bit
// byte offsets from its first one (64-bit products cost the drop-in P.V up to
// 8 %: rank 514, B1 S4099 20.7 against 22.4 us).  Steps of fewer bytes than
// 4 GB: every pitch below 286 MB.
int check_v_step(const starkv_vlatent& v, int S) {
  if (v.format != STARKV_FMT_DENSE) return STARKV_OK;
  const int64_t rows = std::min(S, KSTEP) - 1;
  return rows > 0 && v.stride_s > (((int64_t)1 << 31) - v.rank) / rows ? STARKV_ERR_LIMIT : STARKV_OK;
}

// the P.V kernels' storage kind of a validated latent
int pv_storage(const PVArgs& pa, int vq, int rank, bool fused, int S) {
  return vq == VQ_BLOCK && pv_block_ok(pa, rank, fused, S) ? VQ_RAW : vq;
}

int validate_decode(const starkv_decode_desc* d, int* gs, int* n_wg, int* k1pc, int* vq) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->seq_len < 1 || d->seq_len > MAX_S) return STARKV_ERR_SHAPE;
  if (d->head_dim != HEAD_DIM) return STARKV_ERR_SHAPE;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  if (d->n_q_heads > K2_MAX_H) return STARKV_ERR_LIMIT;
  int st = validate_klatent(d->k, d->n_q_heads, d->dtype, gs);
  if (st) return st;
  PVArgs vtmp = {};
  if ((st = validate_v(d->v, vtmp, vq)) || (st = check_v_step(d->v, d->seq_len))) return st;
  *vq = pv_storage(vtmp, *vq, d->v.rank, true, d->seq_len);
  if (!d->q || !d->uv || !d->out || !d->rope_table) return STARKV_ERR_NULL;
  if (d->seq_len > d->rope_max_positions) return STARKV_ERR_SHAPE;
  if (d->uv_row_stride < d->v.rank) return STARKV_ERR_SHAPE;
  if ((st = check_mask(d->mask, d->mask_dtype))) return st;
  if (d->out_dtype != 0 && d->out_dtype != d->dtype && d->out_dtype != STARKV_F32) return STARKV_ERR_DTYPE;
  KArgs tmp;
  KPlan plan;
  if ((st = build_k_plan(d->k, d->n_q_heads, *gs, d->dtype, d->seq_len, tmp, plan, false, true))) return st;
  *n_wg = plan.n_wg;
  *k1pc = plan.per_cu;
  return STARKV_OK;
}

// Prefill inputs the reconstruction kernels cannot read in place -- latent
// ranks that are not a multiple of 8, latent rows not aligned for their chunk
// loads, or U_v rows that are not 16-byte aligned whole multiples of 8
// columns -- are repacked into aligned copies in the workspace first
// (RepackArgs).  The workspace holds the reconstructed K and V, then these
// copies.
struct PrefillPlan {
  int64_t S = 0, S_pad = 0;
  bool rk = false, rv = false, ru = false;          // repack the K latent, the V latent, U_v
  int k_kind1 = 0, k_kind2 = 0, v_kind1 = 0, v_kind2 = 0;
  int k_p1 = 0, k_p2 = 0, v_p1 = 0, v_p2 = 0, u_p = 0;   // repacked row pitches, bytes
  size_t kvb = 0, off_k1 = 0, off_k2 = 0, off_v1 = 0, off_v2 = 0, off_u = 0, total = 0;
};

int pitch16(int64_t bytes) { return (int)round_up(std::max<int64_t>(bytes, 1), 16); }
// bytes of n elements of a repack kind, n padded to 8
int64_t rp_bytes(int kind, int n) {
  const int64_t n8 = round_up(n, 8);
  return kind == RP_HALF ? 2 * n8 : kind == RP_BYTE ? n8 : n8 / 2;
}

// Prefill: any K latent format and rank (dense, int8 or the reference split
// format), any V latent format and rank (dense, group-64 int4 or per-token
// blocks), q 16-byte aligned.  Positions reconstructed: pos0 + n_tokens,
// padded to 64 in the workspace.
int validate_prefill(const starkv_prefill_desc* d, int* gs, PrefillPlan* P) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->batch > 65535 || d->n_tokens < 1 || d->pos0 < 0) return STARKV_ERR_SHAPE;
  if ((int64_t)d->pos0 + d->n_tokens > MAX_S) return STARKV_ERR_LIMIT;
  if (d->head_dim != HEAD_DIM) return STARKV_ERR_SHAPE;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  int st = validate_klatent(d->k, d->n_q_heads, d->dtype, gs);
  if (st) return st;
  const starkv_klatent& k = d->k;
  PVArgs vb = {};
  int vq = 0;
  if ((st = validate_v(d->v, vb, &vq))) return st;
  if (!d->q || !d->uv || !d->out || !d->rope_table) return STARKV_ERR_NULL;
  if ((int64_t)d->pos0 + d->n_tokens > d->rope_max_positions) return STARKV_ERR_SHAPE;
  if (d->uv_row_stride < d->v.rank) return STARKV_ERR_SHAPE;
  if (d->q_stride_b < 0 || d->q_stride_h < 0 || d->q_stride_t < 0) return STARKV_ERR_SHAPE;
  if (!al(d->q, 16) || !al64(d->q_stride_b, 8) || !al64(d->q_stride_h, 8) || !al64(d->q_stride_t, 8))
    return STARKV_ERR_ALIGN;
  if (d->out_stride_b < 0 || d->out_stride_h < 0 || d->out_stride_t < 0) return STARKV_ERR_SHAPE;
  // one-dimensional grids of the three launches (workgroup counts, ints in the kernels)
  const int64_t S = (int64_t)d->pos0 + d->n_tokens, Hkv = d->k.n_kv_heads;
  const int64_t g_k = round_up((int64_t)d->batch * ceil_div(S, PF_K_POS), 8) * Hkv;
  const int64_t nhp = (Hkv + 1) / 2;
  const int64_t g_v = nhp >= 8 ? 8 * ceil_div(nhp, 8) * d->batch * ceil_div(S, PF_V_POS)
                               : round_up((int64_t)d->batch * ceil_div(S, PF_V_POS), 8) * nhp;
  const int64_t g_a = round_up((int64_t)d->batch * Hkv, 8) * *gs * ceil_div(d->n_tokens, PF_Q_POS);
  if (std::max({g_k, g_v, g_a}) > INT32_MAX) return STARKV_ERR_LIMIT;

  PrefillPlan& p = *P;
  p = PrefillPlan{};
  p.S = S;
  p.S_pad = round_up(S, 64);
  // K latent
  int rmax = 0;
  for (int h = 0; h < k.n_kv_heads; ++h) rmax = std::max(rmax, k.rank[h]);
  const int rmax8 = (int)round_up(rmax, 8);
  if (k.format == STARKV_FMT_DENSE) {
    p.rk = !al(k.data, 16) || !al64(k.stride_b, 8);
    for (int h = 0; h < k.n_kv_heads; ++h)
      p.rk |= k.rank[h] % 8 || !al64(k.head_offset[h], 8) || !al64(k.pos_stride[h], 8);
    p.k_kind1 = RP_HALF;
    p.k_p1 = pitch16(rp_bytes(RP_HALF, rmax8));
  } else {
    p.rk = !k_quant_aligned(k);
    const bool two = k.format == STARKV_FMT_INT4_REF && k.split > 0;
    const bool a8 = two ? k.split_format == STARKV_FMT_INT8_SYM : k.format == STARKV_FMT_INT8_SYM;
    const int split = two ? k.split : 128;
    p.k_kind1 = a8 ? RP_BYTE : RP_NIB;
    p.k_p1 = pitch16(rp_bytes(p.k_kind1, std::min(rmax8, split)));
    if (rmax > split) {
      p.k_kind2 = RP_NIB;
      p.k_p2 = pitch16(rp_bytes(RP_NIB, rmax8 - split));
    }
  }
  // V latent
  const int Rv = d->v.rank;
  if (vq == VQ_DENSE) {
    p.rv = !(al(d->v.data, 16) && al64(d->v.stride_s, 8) && al64(d->v.stride_b, 8) && Rv % 8 == 0);
    p.v_kind1 = RP_HALF;
    p.v_p1 = pitch16(rp_bytes(RP_HALF, Rv));
  } else if (vq == VQ_G64) {
    p.rv = !vb.qfast;
    p.v_kind1 = RP_NIB;
    p.v_p1 = pitch16(rp_bytes(RP_NIB, Rv));
  } else {
    p.rv = !vb.qfast;
    p.v_kind1 = vb.a_int8 ? RP_BYTE : RP_NIB;
    p.v_p1 = pitch16(rp_bytes(p.v_kind1, vb.split));
    if (Rv > vb.split) {
      p.v_kind2 = RP_NIB;
      p.v_p2 = pitch16(rp_bytes(RP_NIB, Rv - vb.split));
    }
  }
  // U_v: 16-byte rows of whole 8-column chunks (the DMA's 16-byte pieces)
  p.ru = !(al(d->uv, 16) && al64(d->uv_row_stride, 8) && Rv % 8 == 0);
  p.u_p = pitch16(rp_bytes(RP_HALF, Rv));

  const size_t B = d->batch;
  p.kvb = a256((size_t)B * Hkv * p.S_pad * HEAD_DIM * 2);
  size_t o = 2 * p.kvb;
  if (p.rk) {
    p.off_k1 = o; o += a256(B * Hkv * S * p.k_p1);
    p.off_k2 = o; o += a256(B * Hkv * S * p.k_p2);
  }
  if (p.rv) {
    p.off_v1 = o; o += a256(B * S * p.v_p1);
    p.off_v2 = o; o += a256(B * S * p.v_p2);
  }
  if (p.ru) {
    p.off_u = o; o += a256((size_t)Hkv * HEAD_DIM * p.u_p);
  }
  p.total = o;
  return STARKV_OK;
}

}  // namespace

extern "C" {

int starkv_abi_version(void) { return STARKV_ABI_VERSION; }

const char* starkv_status_string(int s) {
  switch (s) {
    case STARKV_OK: return "ok";
    case STARKV_ERR_NULL: return "a required pointer is NULL";
    case STARKV_ERR_SHAPE: return "inconsistent or unsupported sizes";
    case STARKV_ERR_DTYPE: return "unsupported element type";
    case STARKV_ERR_ALIGN: return "pointer or stride misaligned";
    case STARKV_ERR_RANK: return "latent rank out of range";
    case STARKV_ERR_WORKSPACE: return "workspace missing or too small";
    case STARKV_ERR_LIMIT: return "exceeds a compiled limit";
    case STARKV_ERR_FORMAT: return "unknown quantisation format";
    default: return s > 0 ? hipGetErrorString((hipError_t)s) : "unknown error";
  }
}

size_t starkv_rope_table_bytes(int max_positions) {
  if (max_positions < 1) return 0;
  return (size_t)rope_table_tiles(max_positions) * 512 * 16;
}

int starkv_rope_build(const float* inv_freq_host, float attention_scaling, int max_positions,
                      void* table, size_t table_bytes, void* stream) {
  if (!inv_freq_host || !table) return STARKV_ERR_NULL;
  if (max_positions < 1 || max_positions > MAX_S) return STARKV_ERR_SHAPE;
  if (table_bytes < starkv_rope_table_bytes(max_positions)) return STARKV_ERR_WORKSPACE;
  if (!al(table, 16)) return STARKV_ERR_ALIGN;
  float f[64];
  for (int i = 0; i < 64; ++i) f[i] = inv_freq_host[i];
  return launch_rope_table(f, max_positions, attention_scaling, table, (hipStream_t)stream);
}

// Dense K whose rows the warp-specialised and grouped-query K-logit kernels
// cannot stream (rows that are neither 16-byte aligned multiples of 8 ranks
// nor contiguous, or fewer than 8 ranks) is first copied into the workspace as
// rows of round_up(r, 8) elements, zero past r, one 16-byte pitch for all
// heads ([B][Hkv][S][pitch]); the kernels then read that copy.  Every latent
// without aligned rows of whole 8-rank chunks asks for the copy's workspace,
// whether its kernel uses it or not.
struct KRepack {
  bool need = false;          // ask for the workspace
  bool on = false;            // make the copy
  int pitch = 0;              // bytes
  size_t bytes = 0;
};

KRepack k_repack_plan(const starkv_klatent& k, int gs, int dtype, int B, int S) {
  KRepack r;
  if (k.format != STARKV_FMT_DENSE) return r;
  const bool ws = k_ws(k, gs, dtype, S, false, false);
  bool rows16 = ws;
  for (int h = 0; h < k.n_kv_heads; ++h) rows16 = rows16 && ws_rows16(k, h, esize(dtype), false);
  if (rows16) return r;
  int rmax = 8;
  for (int h = 0; h < k.n_kv_heads; ++h) rmax = std::max(rmax, k.rank[h]);
  r.pitch = (int)round_up((int64_t)round_up(rmax, 8) * esize(dtype), 16);
  if ((int64_t)TILE * r.pitch >= ((int64_t)1 << 31)) return r;
  r.bytes = a256((size_t)B * k.n_kv_heads * S * r.pitch);
  r.need = true;
  r.on = !ws;
  return r;
}

size_t starkv_k_logits_workspace_bytes(const starkv_klogits_desc* d) {
  int gs = 0;
  if (!d || d->batch < 1 || d->seq_len < 1 || d->seq_len > MAX_S || validate_klatent(d->k, d->n_q_heads, d->dtype, &gs))
    return 0;
  return k_repack_plan(d->k, gs, d->dtype, d->batch, d->seq_len).bytes;
}

int starkv_k_logits(const starkv_klogits_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->seq_len < 1 || d->seq_len > MAX_S || d->head_dim != HEAD_DIM) return STARKV_ERR_SHAPE;
  int gs = 0, st;
  if ((st = validate_klatent(d->k, d->n_q_heads, d->dtype, &gs))) return st;
  if (!d->q || !d->out || !d->rope_table) return STARKV_ERR_NULL;
  if (d->seq_len > d->rope_max_positions) return STARKV_ERR_SHAPE;
  if (d->out_dtype != STARKV_F32 && d->out_dtype != STARKV_F16 && d->out_dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  if ((st = check_mask(d->mask, d->mask_dtype))) return st;
  const KRepack rp = k_repack_plan(d->k, gs, d->dtype, d->batch, d->seq_len);
  starkv_klatent k = d->k;
  int64_t rp_hoff[K_MAX_KV], rp_pstr[K_MAX_KV];   // the repacked copy's head offsets and row pitches
  if (rp.need) {
    if (!workspace || workspace_bytes < rp.bytes) return STARKV_ERR_WORKSPACE;
    if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
  }
  if (rp.on) {
    const int H = k.n_kv_heads, S = d->seq_len, xe = esize(d->dtype);
    RepackArgs ra = {};
    ra.src = (const uint8_t*)k.data; ra.src_sb = k.stride_b * xe;
    for (int h = 0; h < H; ++h) {
      ra.src_off[h] = k.head_offset[h] * xe;
      ra.src_pitch[h] = k.pos_stride[h] * xe;
      ra.nel[h] = k.rank[h];
    }
    ra.dst = (uint8_t*)workspace; ra.dst_sb = (int64_t)H * S * rp.pitch; ra.pitch = rp.pitch;
    ra.kind = RP_HALF; ra.H = H; ra.S = S;
    if ((st = launch_repack(ra, d->batch, (hipStream_t)stream))) return st;
    k.data = workspace;
    k.stride_b = (int64_t)H * S * rp.pitch / xe;
    for (int h = 0; h < H; ++h) {
      rp_hoff[h] = (int64_t)h * S * rp.pitch / xe;
      rp_pstr[h] = rp.pitch / xe;
    }
    k.head_offset = rp_hoff;
    k.pos_stride = rp_pstr;
  }
  KArgs a;
  KPlan plan;
  if ((st = build_k_plan(k, d->n_q_heads, gs, d->dtype, d->seq_len, a, plan, rp.on, false))) return st;
  a.q = d->q; a.q_sb = d->q_stride_b; a.q_sh = d->q_stride_h;
  a.x = k.data; a.x_sb = k.stride_b;
  a.xscale = d->k.scale; a.xs_sb = d->k.scale_stride_b; a.xs_sh = d->k.scale_stride_h;
  a.bk = d->k.bk; a.bk_rs = d->k.bk_row_stride;
  a.rope = (const uint4*)d->rope_table;
  a.mask = d->mask; a.m_sb = d->mask_stride_b; a.m_sh = d->mask_stride_h; a.mask_dtype = d->mask_dtype;
  a.last_pos = nullptr;
  a.out = d->out; a.o_sb = d->out_stride_b; a.o_st = TILE; a.o_sh = d->out_stride_h;   // rows
  a.chunkmax = nullptr;
  a.S = d->seq_len; a.Hq = d->n_q_heads; a.wscale = d->scale;
  const int n_tiles = (int)ceil_div(d->seq_len, TILE);
  // the K-logit kernels address one batch's logits with 32-bit element offsets
  if ((int64_t)(d->n_q_heads - 1) * d->out_stride_h + (int64_t)n_tiles * TILE >= ((int64_t)1 << 32))
    return STARKV_ERR_LIMIT;
  int nc = choose_splits((int64_t)d->batch * plan.n_wg, device_cus() * plan.per_cu, n_tiles, 256, 3.0, 0.0);
  a.tiles_per_chunk = (int)ceil_div(n_tiles, nc);
  a.n_chunks = (int)ceil_div(n_tiles, a.tiles_per_chunk);
  const bool fast = k_fast(k, d->dtype, d->q, d->q_stride_b, d->q_stride_h);
  return launch_k_logits(a, d->dtype, k.format, d->out_dtype == STARKV_F32, d->out_dtype, fast, d->batch, (hipStream_t)stream);
}

size_t starkv_pv_latent_workspace_bytes(const starkv_pv_desc* d) {
  if (!d || d->batch < 1 || d->seq_len < 1 || d->v.rank < 1) return 0;
  PVArgs tmp = {};
  int vq = 0;
  if (validate_v(d->v, tmp, &vq) || check_v_step(d->v, d->seq_len)) return 0;
  vq = pv_storage(tmp, vq, d->v.rank, false, d->seq_len);
  const int BQ = d->batch * head_groups(d->n_heads);
  const PVGeom g = pv_geometry(BQ, d->seq_len, d->v.rank, false, vq, v_row_bytes(d->v));
  return a256((size_t)BQ * g.n_c2 * 32 * g.Rvp * 4) + a256((size_t)BQ * g.n_grp * 32 * g.Rvp * 4);
}

int starkv_pv_latent(const starkv_pv_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->seq_len < 1 || d->seq_len > MAX_S || d->n_heads < 1) return STARKV_ERR_SHAPE;
  if (d->n_heads > K2_MAX_H) return STARKV_ERR_LIMIT;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  int st, vq = 0;
  PVArgs a = {};
  if ((st = validate_v(d->v, a, &vq)) || (st = check_v_step(d->v, d->seq_len))) return st;
  vq = pv_storage(a, vq, d->v.rank, false, d->seq_len);
  if (!d->p || !d->out) return STARKV_ERR_NULL;
  const size_t need = starkv_pv_latent_workspace_bytes(d);
  if (!workspace || workspace_bytes < need) return STARKV_ERR_WORKSPACE;
  if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
  const int n_hg = head_groups(d->n_heads), BQ = d->batch * n_hg;
  const PVGeom g = pv_geometry(BQ, d->seq_len, d->v.rank, false, vq, v_row_bytes(d->v));
  a.n_hg = n_hg;
  a.Rv = d->v.rank; a.Rvp = g.Rvp; a.n_cb = g.n_cb; a.n_c2 = g.n_c2; a.c2_len = g.c2_len; a.n_grp = g.n_grp;
  a.p = d->p; a.p_sb = d->p_stride_b; a.p_sh = d->p_stride_h;
  a.p_vec = al(d->p, 16) && al64(d->p_stride_b * 2, 16) && al64(d->p_stride_h * 2, 16);
  a.part = (float*)workspace;
  a.part2 = (float*)((char*)workspace + a256((size_t)BQ * g.n_c2 * 32 * g.Rvp * 4));
  a.out = d->out; a.o_sb = d->out_stride_b; a.o_sh = d->out_stride_h;
  a.S = d->seq_len; a.H = d->n_heads;
  return launch_pv(a, d->dtype, vq, false, v_fast(d->v, a), d->batch, (hipStream_t)stream);
}

size_t starkv_decode_workspace_bytes(const starkv_decode_desc* d) {
  int gs = 0, n_wg = 0, k1pc = 1, vq = 0;
  if (validate_decode(d, &gs, &n_wg, &k1pc, &vq)) return 0;
  return decode_layout(d->batch, d->n_q_heads, d->k.n_kv_heads, d->seq_len, d->v.rank, n_wg, k1pc, vq, v_row_bytes(d->v),
                    d->dtype == STARKV_F16).total;
}

// the logits of a validated decode call, into its workspace
static int decode_logits(const starkv_decode_desc* d, const DecodeLayout& L, int gs, char* ws, hipStream_t s) {
  const int B = d->batch, Hq = d->n_q_heads;
  int st;
  KArgs ka;
  KPlan plan;
  if ((st = build_k_plan(d->k, Hq, gs, d->dtype, d->seq_len, ka, plan, false, true))) return st;
  ka.q = d->q; ka.q_sb = d->q_stride_b; ka.q_sh = d->q_stride_h;
  ka.x = d->k.data; ka.x_sb = d->k.stride_b;
  ka.xscale = d->k.scale; ka.xs_sb = d->k.scale_stride_b; ka.xs_sh = d->k.scale_stride_h;
  ka.bk = d->k.bk; ka.bk_rs = d->k.bk_row_stride;
  ka.rope = (const uint4*)d->rope_table;
  ka.mask = d->mask; ka.m_sb = d->mask_stride_b; ka.m_sh = d->mask_stride_h; ka.mask_dtype = d->mask_dtype;
  ka.last_pos = d->last_pos_device;
  // logits in 32-position tiles of all heads: a tile's 4 KB is written together
  // by the workgroups of one chunk and read contiguously by P.V
  ka.out = ws + L.off_logits; ka.o_sb = (int64_t)Hq * L.S_pad; ka.o_st = (int64_t)Hq * TILE; ka.o_sh = TILE;
  ka.chunkmax = (float*)(ws + L.off_cmax);
  ka.S = d->seq_len; ka.Hq = Hq; ka.n_chunks = L.n_c1; ka.tiles_per_chunk = L.tiles_per_chunk;
  ka.wscale = d->scale;
  const bool kfast = k_fast(d->k, d->dtype, d->q, d->q_stride_b, d->q_stride_h);
  return launch_k_logits(ka, d->dtype, d->k.format, true, STARKV_F32, kfast, B, s);
}

// P.V over them
static int decode_pv(const starkv_decode_desc* d, const DecodeLayout& L, char* ws, hipStream_t s, PVArgs& pa) {
  const int B = d->batch, Hq = d->n_q_heads;
  int vq = 0, st;
  pa = PVArgs{};
  if ((st = validate_v(d->v, pa, &vq))) return st;
  vq = pv_storage(pa, vq, d->v.rank, true, d->seq_len);
  pa.logits = (const float*)(ws + L.off_logits); pa.l_sb = (int64_t)Hq * L.S_pad; pa.l_st = (int64_t)Hq * TILE; pa.l_sh = TILE;
  pa.chunkmax = (const float*)(ws + L.off_cmax); pa.n_chunk1 = L.n_c1;
  pa.part = (float*)(ws + L.off_part); pa.psum = (float*)(ws + L.off_psum); pa.part16 = L.part16;
  pa.S = d->seq_len; pa.H = Hq; pa.n_hg = L.n_hg; pa.Rv = d->v.rank; pa.Rvp = L.pv.Rvp;
  pa.n_cb = L.pv.n_cb; pa.n_c2 = L.pv.n_c2; pa.c2_len = L.pv.c2_len; pa.ntw = L.pv.ntw;
  return launch_pv(pa, d->dtype, vq, true, v_fast(d->v, pa), B, s);
}

// weights of a decode call's logits by position, from its maxima and sums
static int decode_scores(const starkv_decode_desc* d, const DecodeLayout& L, const char* ws, const float* rmax, int n_max,
                         const float* rsum, int n_sum, float* scores, int64_t stride, hipStream_t s) {
  ScoreArgs a = {};
  a.x = ws + L.off_logits; a.x_sb = (int64_t)d->n_q_heads * L.S_pad; a.x_st = (int64_t)d->n_q_heads * TILE; a.x_sh = TILE;
  a.B = d->batch; a.H = d->n_q_heads; a.S = d->seq_len; a.add = 1;
  a.rmax = rmax; a.n_max = n_max; a.rsum = rsum; a.n_sum = n_sum; a.n_hg = L.n_hg;
  a.out = scores; a.o_sb = stride;
  return launch_decode_scores(a, s);
}

static int check_scores(const starkv_decode_desc* d, const float* scores, int64_t stride) {
  if (!al(scores, 4)) return STARKV_ERR_ALIGN;
  if (d->batch > 65535) return STARKV_ERR_LIMIT;
  return d->batch > 1 && stride < d->seq_len ? STARKV_ERR_SHAPE : STARKV_OK;
}

static int decode_impl(const starkv_decode_desc* d, void* workspace, size_t workspace_bytes, void* stream,
                       void* const* events, float* scores = nullptr, int64_t scores_stride = 0) {
  int gs = 0, n_wg = 0, k1pc = 1, vq = 0, st;
  if ((st = validate_decode(d, &gs, &n_wg, &k1pc, &vq))) return st;
  if (scores && (st = check_scores(d, scores, scores_stride))) return st;
  const DecodeLayout L =
      decode_layout(d->batch, d->n_q_heads, d->k.n_kv_heads, d->seq_len, d->v.rank, n_wg, k1pc, vq, v_row_bytes(d->v),
                    d->dtype == STARKV_F16);
  if (!workspace || workspace_bytes < L.total) return STARKV_ERR_WORKSPACE;
  if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
  char* ws = (char*)workspace;
  hipStream_t s = (hipStream_t)stream;
  const int B = d->batch, Hq = d->n_q_heads;
  PVArgs pa;
  if (events && (st = (int)hipEventRecord((hipEvent_t)events[0], s))) return st;
  if ((st = decode_logits(d, L, gs, ws, s))) return st;
  if (events && (st = (int)hipEventRecord((hipEvent_t)events[1], s))) return st;
  if ((st = decode_pv(d, L, ws, s, pa))) return st;
  if (events && (st = (int)hipEventRecord((hipEvent_t)events[2], s))) return st;

  UPArgs ua;
  ua.part = pa.part; ua.psum = pa.psum; ua.part16 = L.part16; ua.n_c2 = L.pv.n_c2; ua.Rvp = L.pv.Rvp;
  ua.n_hg = L.n_hg;
  ua.uv = d->uv; ua.uv_rs = d->uv_row_stride;
  ua.out = d->out; ua.o_sb = d->out_stride_b; ua.o_sh = d->out_stride_h;
  ua.B = B; ua.Hq = Hq; ua.gs = gs; ua.Rv = d->v.rank;
  ua.sw = L.sw; ua.n_sl = L.n_sl; ua.n_cs = L.n_cs; ua.ypart = (float*)(ws + L.off_ypart);
  ua.out_f32 = d->out_dtype == STARKV_F32;
  const bool ufast = al(d->uv, 16) && al64(d->uv_row_stride * 2, 16);
  if ((st = launch_up_proj(ua, d->dtype, ufast, s))) return st;
  if (events && (st = (int)hipEventRecord((hipEvent_t)events[3], s))) return st;
  if (scores) return decode_scores(d, L, ws, pa.chunkmax, L.n_c1, pa.psum, L.pv.n_c2, scores, scores_stride, s);
  return STARKV_OK;
}

int starkv_decode_attention(const starkv_decode_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  return decode_impl(d, workspace, workspace_bytes, stream, nullptr);
}

int starkv_decode_attention_timed(const starkv_decode_desc* d, void* workspace, size_t workspace_bytes,
                                  void* stream, void* const* events) {
  if (!events || !events[0] || !events[1] || !events[2] || !events[3]) return STARKV_ERR_NULL;
  return decode_impl(d, workspace, workspace_bytes, stream, events);
}

}  // extern "C"

// ---------------------------------------------------------------------------
// Allocation-free decode: the workspace is a file-scope device array of
// STARKV_NOALLOC_SCRATCH_BYTES that every GPU the library runs on holds until
// the process ends.  Its device address is looked up once per device (the
// array's name is only a host-side stand-in) and kept; calls on one GPU share
// it, so calls that overlap on one GPU race.  The decode kernels write every
// workspace element they read (nothing needs clearing between calls).
// ---------------------------------------------------------------------------
namespace {

__device__ __align__(256) char scratch[STARKV_NOALLOC_SCRATCH_BYTES];

constexpr int NOALLOC_MAX_DEVICES = 64;
std::mutex g_scratch_mu;
void* g_scratch_ptr[NOALLOC_MAX_DEVICES] = {};

// the current device's address of `scratch` (looked up on its first use)
int scratch_address(void** out) {
  int dev = 0;
  int st = (int)hipGetDevice(&dev);
  if (st) return st;
  if (dev < 0 || dev >= NOALLOC_MAX_DEVICES) return STARKV_ERR_LIMIT;
  std::lock_guard<std::mutex> lock(g_scratch_mu);
  if (!g_scratch_ptr[dev]) {
    void* p = nullptr;
    if ((st = (int)hipGetSymbolAddress(&p, HIP_SYMBOL(scratch)))) return st;
    if (!p) return (int)hipErrorInvalidSymbol;
    g_scratch_ptr[dev] = p;
  }
  *out = g_scratch_ptr[dev];
  return STARKV_OK;
}

}  // namespace

extern "C" {

int starkv_decode_attention_noalloc(const starkv_decode_desc* d, void* stream) {
  int gs = 0, n_wg = 0, k1pc = 1, vq = 0, st;
  if ((st = validate_decode(d, &gs, &n_wg, &k1pc, &vq))) return st;
  const size_t need =
      decode_layout(d->batch, d->n_q_heads, d->k.n_kv_heads, d->seq_len, d->v.rank, n_wg, k1pc, vq, v_row_bytes(d->v),
                    d->dtype == STARKV_F16).total;
  if (need > (size_t)STARKV_NOALLOC_SCRATCH_BYTES) return STARKV_ERR_LIMIT;
  void* ws = nullptr;
  if ((st = scratch_address(&ws))) return st;
  return decode_impl(d, ws, STARKV_NOALLOC_SCRATCH_BYTES, stream, nullptr);
}

static int build_rope_apply(const starkv_rope_apply_desc* d, RopeApplyArgs& a) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->n_heads < 1 || d->n_tokens < 0 || d->pos0 < 0) return STARKV_ERR_SHAPE;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  if (!d->x || !d->rope_table) return STARKV_ERR_NULL;
  if (d->stride_b < 0 || d->stride_h < 0 || d->stride_t < 0) return STARKV_ERR_SHAPE;
  if (!d->pos0_device && (int64_t)d->pos0 + d->n_tokens > d->rope_max_positions) return STARKV_ERR_SHAPE;
  // one thread per (row, frequency); HIP keeps grid x block below 2^32
  if ((int64_t)d->batch * d->n_heads * d->n_tokens * 64 > MAX_THREADS_1D) return STARKV_ERR_LIMIT;
  a = RopeApplyArgs{};
  a.x = d->x; a.sb = d->stride_b; a.sh = d->stride_h; a.st = d->stride_t;
  a.B = d->batch; a.H = d->n_heads; a.T = d->n_tokens; a.pos0 = d->pos0; a.max_pos = d->rope_max_positions;
  a.pos0_dev = d->pos0_device; a.err = d->error_flag; a.table = d->rope_table;
  return STARKV_OK;
}

int starkv_rope_apply(const starkv_rope_apply_desc* d, void* stream) {
  RopeApplyArgs a;
  const int st = build_rope_apply(d, a);
  return st ? st : launch_rope_apply(a, d->dtype, (hipStream_t)stream);
}

static int build_k_append(const starkv_k_append_desc* d, KAppendArgs& a) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->n_tokens < 0 || d->pos0 < 0 || d->capacity < 1 || d->capacity > MAX_S) return STARKV_ERR_SHAPE;
  if (!d->pos0_device && (int64_t)d->pos0 + d->n_tokens > d->capacity) return STARKV_ERR_SHAPE;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  const starkv_klatent& k = d->k;
  int st = validate_klayout(k, d->dtype);
  if (st) return st;
  if (!d->src) return STARKV_ERR_NULL;
  if (d->src_stride_b < 0 || d->src_stride_h < 0 || d->src_stride_t < 0) return STARKV_ERR_SHAPE;
  // one wave (64 threads) per row
  if ((int64_t)d->batch * k.n_kv_heads * d->n_tokens * 64 > MAX_THREADS_1D) return STARKV_ERR_LIMIT;
  a = KAppendArgs{};
  a.src = d->src; a.src_sb = d->src_stride_b; a.src_sh = d->src_stride_h; a.src_st = d->src_stride_t;
  a.B = d->batch; a.H = k.n_kv_heads; a.T = d->n_tokens; a.pos0 = d->pos0; a.cap = d->capacity;
  a.pos0_dev = d->pos0_device; a.err = d->error_flag;
  a.fmt = k.format;
  a.data = (void*)k.data; a.stride_b = k.stride_b;
  a.scale = (void*)k.scale; a.sc_sb = k.scale_stride_b; a.sc_sh = k.scale_stride_h; a.sc_ss = 1;
  const bool two = k.format == STARKV_FMT_INT4_REF && k.split > 0;
  a.split = two ? k.split : 128;
  a.a_int8 = two ? k.split_format == STARKV_FMT_INT8_SYM : k.format == STARKV_FMT_INT8_SYM;
  a.data2 = (void*)k.data2; a.stride2_b = k.stride2_b;
  a.scale2 = (void*)k.scale2; a.sc2_sb = k.scale2_stride_b; a.sc2_sh = k.scale2_stride_h; a.sc2_ss = 1;
  for (int h = 0; h < k.n_kv_heads; ++h) {
    a.rank[h] = k.rank[h];
    a.off[h] = k.head_offset[h]; a.pitch[h] = k.pos_stride[h];
    const bool lo = two && k.rank[h] > k.split;
    a.off2[h] = lo ? k.head_offset2[h] : 0; a.pitch2[h] = lo ? k.pos_stride2[h] : 0;
    a.src_off[h] = d->src_head_offset ? d->src_head_offset[h] : h * d->src_stride_h;
    if (a.src_off[h] < 0) return STARKV_ERR_SHAPE;
  }
  return STARKV_OK;
}

int starkv_k_append(const starkv_k_append_desc* d, void* stream) {
  KAppendArgs a;
  const int st = build_k_append(d, a);
  return st ? st : launch_k_append(a, d->dtype, (hipStream_t)stream);
}

static int build_v_append(const starkv_v_append_desc* d, VAppendArgs& a) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->n_tokens < 0 || d->pos0 < 0 || d->capacity < 1 || d->capacity > MAX_S) return STARKV_ERR_SHAPE;
  if (!d->pos0_device && (int64_t)d->pos0 + d->n_tokens > d->capacity) return STARKV_ERR_SHAPE;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  PVArgs pa = {};
  int vq = 0, st;
  if ((st = validate_v(d->v, pa, &vq))) return st;
  if (!d->src) return STARKV_ERR_NULL;
  if (d->src_stride_b < 0 || d->src_stride_t < 0) return STARKV_ERR_SHAPE;
  // one wave per row (group-64: per row and group of 64 ranks)
  const int64_t waves_per_row = vq == VQ_G64 ? ceil_div(d->v.rank, 64) : 1;
  if ((int64_t)d->batch * d->n_tokens * waves_per_row * 64 > MAX_THREADS_1D) return STARKV_ERR_LIMIT;
  a = VAppendArgs{};
  a.src = d->src; a.src_sb = d->src_stride_b; a.src_st = d->src_stride_t;
  a.B = d->batch; a.T = d->n_tokens; a.pos0 = d->pos0; a.cap = d->capacity; a.R = d->v.rank; a.vq = vq;
  a.pos0_dev = d->pos0_device; a.err = d->error_flag;
  a.data = (void*)pa.x; a.stride_b = pa.x_sb; a.stride_s = pa.x_ss;
  a.scale = (void*)pa.xs; a.sc_sb = pa.xs_sb; a.sc_ss = pa.xs_ss;
  a.zero = (void*)pa.xz;
  a.split = pa.split; a.a_int8 = pa.a_int8;
  a.data2 = (void*)pa.x2; a.stride2_b = pa.x2_sb; a.stride2_s = pa.x2_ss;
  a.scale2 = (void*)pa.xs2; a.sc2_sb = pa.xs2_sb; a.sc2_ss = pa.xs2_ss;
  return STARKV_OK;
}

int starkv_v_append(const starkv_v_append_desc* d, void* stream) {
  VAppendArgs a;
  const int st = build_v_append(d, a);
  return st ? st : launch_v_append(a, d->dtype, (hipStream_t)stream);
}

int starkv_decode_append(const starkv_k_append_desc* k, const starkv_v_append_desc* v,
                         const starkv_rope_apply_desc* q, void* stream) {
  StepAppendArgs a = {};
  int st;
  if ((st = build_k_append(k, a.k)) || (st = build_v_append(v, a.v))) return st;
  if (q && (st = build_rope_apply(q, a.r))) return st;
  if (v->dtype != k->dtype || (q && q->dtype != k->dtype)) return STARKV_ERR_DTYPE;
  a.has_rope = q != nullptr;
  const int64_t nb = ceil_div((int64_t)k->batch * k->k.n_kv_heads * k->n_tokens, 4) +
                     ceil_div((int64_t)v->batch * v->n_tokens * ceil_div(v->v.rank, 64), 4) +
                     (q ? ceil_div((int64_t)q->batch * q->n_heads * q->n_tokens * 64, 256) : 0);
  if (nb > INT32_MAX) return STARKV_ERR_LIMIT;
  return launch_step_append(a, k->dtype, (hipStream_t)stream);
}

// rows of act-dtype values: data 16-byte aligned, strides multiples of 8 elements
static bool rows16(const void* p, int64_t stride) { return al(p, 16) && stride >= 0 && stride % 8 == 0; }

int starkv_rms_norm(const starkv_rms_norm_desc* d, void* stream) {
  if (!d) return STARKV_ERR_NULL;
  if (d->rows < 0 || d->hidden < 8 || d->hidden % 8) return STARKV_ERR_SHAPE;
  if (d->hidden > NORM_MAX_HIDDEN) return STARKV_ERR_LIMIT;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  if (!d->x || !d->weight || !d->out || (d->residual_out && !d->residual)) return STARKV_ERR_NULL;
  if (!(d->eps >= 0.f)) return STARKV_ERR_SHAPE;
  if (!rows16(d->x, d->x_stride) || !rows16(d->out, d->out_stride) || !al(d->weight, 16) ||
      (d->residual && !rows16(d->residual, d->residual_stride)) ||
      (d->residual_out && !rows16(d->residual_out, d->residual_out_stride)))
    return STARKV_ERR_ALIGN;
  NormArgs a = {};
  a.x = d->x; a.xs = d->x_stride;
  a.res = d->residual; a.rs = d->residual_stride;
  a.res_out = d->residual_out; a.ros = d->residual_out_stride;
  a.w = d->weight; a.out = d->out; a.os = d->out_stride;
  a.rows = d->rows; a.H = d->hidden; a.eps = d->eps;
  return launch_rms_norm(a, d->dtype, (hipStream_t)stream);
}

int starkv_silu_mul(const starkv_silu_mul_desc* d, void* stream) {
  if (!d) return STARKV_ERR_NULL;
  if (d->rows < 0 || d->width < 8 || d->width % 8) return STARKV_ERR_SHAPE;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  if (!d->gate || !d->up || !d->out) return STARKV_ERR_NULL;
  if (!rows16(d->gate, d->gate_stride) || !rows16(d->up, d->up_stride) || !rows16(d->out, d->out_stride))
    return STARKV_ERR_ALIGN;
  if ((int64_t)d->rows * (d->width / 8) > MAX_THREADS_1D) return STARKV_ERR_LIMIT;
  SiluMulArgs a = {};
  a.g = d->gate; a.gs = d->gate_stride; a.u = d->up; a.us = d->up_stride;
  a.out = d->out; a.os = d->out_stride; a.rows = d->rows; a.W = d->width;
  return launch_silu_mul(a, d->dtype, (hipStream_t)stream);
}

int starkv_skinny_gemm(const starkv_skinny_gemm_desc* d, void* stream) {
  if (!d) return STARKV_ERR_NULL;
  if (d->m < 1 || d->k < 64 || d->k % 64 || d->n < 16 || d->n % 16) return STARKV_ERR_SHAPE;
  if (d->m > GEMM_MAX_M) return STARKV_ERR_LIMIT;
  if (d->epilogue < GEMM_STORE || d->epilogue > GEMM_SILU_MUL) return STARKV_ERR_SHAPE;
  if (d->epilogue == GEMM_SILU_MUL && d->n % 32) return STARKV_ERR_SHAPE;
  if (d->dtype != STARKV_F16 && d->dtype != STARKV_BF16) return STARKV_ERR_DTYPE;
  if (!d->x || !d->w || !d->out) return STARKV_ERR_NULL;
  if (d->x_stride < d->k || (!d->w_packed && d->w_stride < d->k)) return STARKV_ERR_SHAPE;
  const int n_out = d->epilogue == GEMM_SILU_MUL ? d->n / 2 : d->n;
  if (d->out_stride < n_out) return STARKV_ERR_SHAPE;
  if (!rows16(d->x, d->x_stride) || !al(d->w, 16) || (!d->w_packed && !rows16(d->w, d->w_stride)) || !al(d->out, 2))
    return STARKV_ERR_ALIGN;
  GemmArgs a = {};
  a.x = d->x; a.xs = d->x_stride; a.w = d->w; a.ws = d->w_stride; a.out = d->out; a.os = d->out_stride;
  a.wpk = d->w_packed != 0;
  if (d->rms && !(d->rms_eps >= 0.f)) return STARKV_ERR_SHAPE;
  a.rms = d->rms != 0; a.rms_eps = d->rms_eps;
  a.M = d->m; a.N = d->n; a.K = d->k; a.half_rows = d->n / 2;
  return launch_skinny_gemm(a, d->dtype, d->epilogue, (hipStream_t)stream);
}

}  // extern "C"

extern "C" {

size_t starkv_prefill_workspace_bytes(const starkv_prefill_desc* d) {
  int gs = 0;
  PrefillPlan P;
  if (validate_prefill(d, &gs, &P)) return 0;
  return P.total;
}

// Launch the repacks the plan asks for and point the kernel arguments at the
// aligned copies (latent offsets: elements for dense, bytes for quantised).
static int prefill_repack(const starkv_prefill_desc* d, const PrefillPlan& P, PFArgs& a, char* ws, hipStream_t s) {
  const starkv_klatent& k = d->k;
  const int Hkv = k.n_kv_heads, B = d->batch, S = (int)P.S;
  int st;
  auto set = [&](RepackArgs& r, int kind, const void* src, int64_t src_sb, int H, int S_, char* dst, int pitch) {
    r = RepackArgs{};
    r.kind = kind; r.src = (const uint8_t*)src; r.src_sb = src_sb; r.H = H; r.S = S_;
    r.dst = (uint8_t*)dst; r.pitch = pitch; r.dst_sb = (int64_t)H * S_ * pitch;
  };
  if (P.rk) {
    const bool dense = k.format == STARKV_FMT_DENSE;
    const int es = dense ? 2 : 1;
    const bool two = k.format == STARKV_FMT_INT4_REF && k.split > 0;
    const int split = dense ? 128 : (two ? k.split : 128);
    RepackArgs r;
    set(r, P.k_kind1, k.data, k.stride_b * es, Hkv, S, ws + P.off_k1, P.k_p1);
    for (int h = 0; h < Hkv; ++h) {
      r.src_off[h] = k.head_offset[h] * es; r.src_pitch[h] = k.pos_stride[h] * es;
      r.nel[h] = std::min(k.rank[h], split);
    }
    if ((st = launch_repack(r, B, s))) return st;
    a.kx = r.dst; a.kx_sb = r.dst_sb / es;
    for (int h = 0; h < Hkv; ++h) { a.kxoff[h] = (int64_t)h * S * P.k_p1 / es; a.kxpitch[h] = P.k_p1 / es; }
    if (P.k_p2) {
      set(r, RP_NIB, k.data2, k.stride2_b, Hkv, S, ws + P.off_k2, P.k_p2);
      for (int h = 0; h < Hkv; ++h) {
        const bool lo = k.rank[h] > split;
        r.src_off[h] = lo ? k.head_offset2[h] : 0; r.src_pitch[h] = lo ? k.pos_stride2[h] : 0;
        r.nel[h] = lo ? k.rank[h] - split : 0;
      }
      if ((st = launch_repack(r, B, s))) return st;
      a.kx2 = r.dst; a.kx2_sb = r.dst_sb;
      for (int h = 0; h < Hkv; ++h) { a.kxoff2[h] = (int64_t)h * S * P.k_p2; a.kxpitch2[h] = P.k_p2; }
    }
  }
  if (P.rv) {
    const starkv_vlatent& v = d->v;
    const bool dense = v.format == STARKV_FMT_DENSE;
    const int es = dense ? 2 : 1;
    PVArgs vb = {};
    int vq = 0;
    if ((st = validate_v(v, vb, &vq))) return st;
    RepackArgs r;
    set(r, P.v_kind1, v.data, v.stride_b * es, 1, S, ws + P.off_v1, P.v_p1);
    r.src_off[0] = 0; r.src_pitch[0] = v.stride_s * es;
    r.nel[0] = vq == VQ_BLOCK ? vb.split : v.rank;
    if ((st = launch_repack(r, B, s))) return st;
    a.vx = r.dst; a.vx_sb = r.dst_sb / es; a.vx_ss = P.v_p1 / es;
    if (P.v_p2) {
      set(r, RP_NIB, v.data2, v.stride2_b, 1, S, ws + P.off_v2, P.v_p2);
      r.src_off[0] = 0; r.src_pitch[0] = v.stride2_s;
      r.nel[0] = v.rank - vb.split;
      if ((st = launch_repack(r, B, s))) return st;
      a.vx2 = r.dst; a.vx2_sb = r.dst_sb; a.vx2_ss = P.v_p2;
    }
  }
  if (P.ru) {
    RepackArgs r;
    set(r, RP_HALF, d->uv, 0, 1, Hkv * HEAD_DIM, ws + P.off_u, P.u_p);
    r.src_off[0] = 0; r.src_pitch[0] = d->uv_row_stride * 2;
    r.nel[0] = d->v.rank;
    if ((st = launch_repack(r, 1, s))) return st;
    a.uv = r.dst; a.uv_rs = P.u_p / 2;
  }
  return STARKV_OK;
}

static int prefill_impl(const starkv_prefill_desc* d, void* workspace, size_t workspace_bytes, void* stream,
                        void* const* events) {
  int gs = 0, st;
  PrefillPlan P;
  if ((st = validate_prefill(d, &gs, &P))) return st;
  const size_t kvb = P.kvb;
  if (!workspace || workspace_bytes < P.total) return STARKV_ERR_WORKSPACE;
  if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
  const starkv_klatent& k = d->k;
  PFArgs a = {};
  a.S = d->pos0 + d->n_tokens; a.S_pad = (int)P.S_pad;
  a.Hkv = k.n_kv_heads; a.Hq = d->n_q_heads; a.gs = gs; a.T = d->n_tokens; a.pos0 = d->pos0;
  a.kx = k.data; a.kx_sb = k.stride_b; a.k_i8 = k.format == STARKV_FMT_INT8_SYM;
  a.kscale = k.scale; a.ks_sb = k.scale_stride_b; a.ks_sh = k.scale_stride_h;
  // reference split format: ranks [0, ksplit) int8 or int4 in data, the rest int4 in data2
  const bool ktwo = k.format == STARKV_FMT_INT4_REF && k.split > 0;
  a.k_ref = k.format == STARKV_FMT_INT4_REF;
  a.ksplit = ktwo ? k.split : 128;
  a.k_a8 = ktwo && k.split_format == STARKV_FMT_INT8_SYM;
  a.kx2 = k.data2; a.kx2_sb = k.stride2_b;
  a.kscale2 = k.scale2; a.ks2_sb = k.scale2_stride_b; a.ks2_sh = k.scale2_stride_h;
  for (int h = 0; h < k.n_kv_heads; ++h) {
    a.krank[h] = k.rank[h];
    a.kxoff[h] = k.head_offset[h]; a.kxpitch[h] = k.pos_stride[h];
    const bool lo = ktwo && k.rank[h] > k.split;
    a.kxoff2[h] = lo ? k.head_offset2[h] : 0; a.kxpitch2[h] = lo ? k.pos_stride2[h] : 0;
    a.bkoff[h] = k.bk_head_offset[h];
  }
  a.bk = k.bk; a.bk_rs = k.bk_row_stride;
  const starkv_vlatent& v = d->v;
  a.vx = v.data; a.vx_sb = v.stride_b; a.vx_ss = v.stride_s;
  a.v_g64 = v.format == STARKV_FMT_INT4_G64; a.Rv = v.rank;
  a.vscale = v.scale; a.vzero = v.zero; a.vs_sb = v.scale_stride_b; a.vs_ss = v.scale_stride_s;
  {
    // per-token blocks: the split and block formats as validate_v reads them
    PVArgs vb = {};
    int vq = 0;
    if ((st = validate_v(v, vb, &vq))) return st;
    a.v_blk = vq == VQ_BLOCK;
    a.vsplit = vb.split; a.v_a8 = vb.a_int8;
    a.vx2 = vb.x2; a.vx2_sb = vb.x2_sb; a.vx2_ss = vb.x2_ss;
    a.vscale2 = vb.xs2; a.vs2_sb = vb.xs2_sb; a.vs2_ss = vb.xs2_ss;
  }
  a.uv = d->uv; a.uv_rs = d->uv_row_stride;
  a.rope = d->rope_table;
  a.kbuf = workspace; a.vbuf = (char*)workspace + kvb;
  a.q = d->q; a.q_sb = d->q_stride_b; a.q_sh = d->q_stride_h; a.q_st = d->q_stride_t;
  a.scale_log2 = d->scale * 1.4426950408889634f;
  a.out = d->out; a.o_sb = d->out_stride_b; a.o_sh = d->out_stride_h; a.o_st = d->out_stride_t;
  hipStream_t s = (hipStream_t)stream;
  if (events && (st = (int)hipEventRecord((hipEvent_t)events[0], s))) return st;
  if ((st = prefill_repack(d, P, a, (char*)workspace, s))) return st;
  if ((st = launch_prefill(a, d->dtype, d->batch, s, events ? (hipEvent_t)events[1] : nullptr))) return st;
  if (events && (st = (int)hipEventRecord((hipEvent_t)events[2], s))) return st;
  return STARKV_OK;
}

int starkv_prefill_attention(const starkv_prefill_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  return prefill_impl(d, workspace, workspace_bytes, stream, nullptr);
}

int starkv_prefill_attention_timed(const starkv_prefill_desc* d, void* workspace, size_t workspace_bytes,
                                   void* stream, void* const* events) {
  if (!events || !events[0] || !events[1] || !events[2]) return STARKV_ERR_NULL;
  return prefill_impl(d, workspace, workspace_bytes, stream, events);
}

}  // extern "C"

extern "C" {

static int scale_size(int dt) { return dt == STARKV_E8M0 ? 1 : dt == STARKV_F32 ? 4 : 0; }
// e4m3 rows: 16-byte aligned pieces
static bool rows_e4m3(const void* p, int64_t stride) { return al(p, 16) && stride % 16 == 0; }
static bool act16(int dt) { return dt == STARKV_F16 || dt == STARKV_BF16; }

int starkv_fp8_quantize(const starkv_fp8_quantize_desc* d, void* stream) {
  if (!d) return STARKV_ERR_NULL;
  if (d->rows < 0 || d->k < 1) return STARKV_ERR_SHAPE;
  if (!act16(d->dtype) || !scale_size(d->scale_dtype)) return STARKV_ERR_DTYPE;
  if (d->rows == 0) return STARKV_OK;
  if (!d->x || !d->q || !d->scale) return STARKV_ERR_NULL;
  if ((d->rows > 1 && (d->x_stride < d->k || d->q_stride < round_up(d->k, 16))) || d->scale_stride_r < 0 ||
      d->scale_stride_b < 0)
    return STARKV_ERR_SHAPE;
  if (!al(d->x, 2) || !rows_e4m3(d->q, d->q_stride) || !al(d->scale, scale_size(d->scale_dtype))) return STARKV_ERR_ALIGN;
  Fp8QuantArgs a = {};
  a.x = d->x; a.xs = d->x_stride; a.q = (uint8_t*)d->q; a.qs = d->q_stride;
  a.s = d->scale; a.ssr = d->scale_stride_r; a.ssb = d->scale_stride_b;
  a.rows = d->rows; a.k = d->k; a.kb = (int)ceil_div(d->k, FP8_BLOCK);
  a.vec = al(d->x, 16) && d->x_stride % 8 == 0;
  if (ceil_div((int64_t)a.rows * a.kb, 32) > INT32_MAX / 256) return STARKV_ERR_LIMIT;
  return launch_fp8_quant(a, d->dtype, d->scale_dtype, (hipStream_t)stream);
}

// workspace of a product: quantised activations, their scales (block-major),
// row factors
struct Fp8Space { Fp8Plan plan; size_t off_s, off_r, total; };

static int plan_fp8(const starkv_fp8_gemm_desc* d, Fp8Space& s) {
  if (!d) return STARKV_ERR_NULL;
  if (d->m < 0 || d->n < 1 || d->k < 1) return STARKV_ERR_SHAPE;
  const bool q = d->dtype != STARKV_E4M3;
  if ((q && !act16(d->dtype)) || !scale_size(d->scale_dtype)) return STARKV_ERR_DTYPE;
  if (!act16(d->out_dtype) && d->out_dtype != STARKV_F32) return STARKV_ERR_DTYPE;
  if (d->silu_mul && (d->n % 256 || d->residual)) return STARKV_ERR_SHAPE;
  if (d->rms && (!q || !(d->rms_eps >= 0.f))) return STARKV_ERR_SHAPE;
  if (d->k > (1 << 24) || d->n > (1 << 30) || d->m > (1 << 30)) return STARKV_ERR_LIMIT;
  s = Fp8Space{};
  const int64_t kb = ceil_div(d->k, FP8_BLOCK);
  if (q && d->m > 0) {
    s.off_s = a256((size_t)d->m * round_up(d->k, 16));
    s.off_r = s.off_s + a256((size_t)d->m * kb * scale_size(d->scale_dtype));
    s.total = s.off_r + a256((size_t)d->m * 4);
  }
  s.plan = plan_fp8_gemm(d->m, d->n, (int)kb, d->silu_mul != 0, d->out_dtype == STARKV_F32,
                         d->scale_dtype == STARKV_E8M0, device_cus());
  // grids of at most 2^22 workgroups (2^31 threads), rows' blocks below 2^31
  if ((ceil_div(d->m, s.plan.bm) + 1) * (ceil_div(d->n, s.plan.bn) + 8) > (1 << 22) || (int64_t)d->m * kb > INT32_MAX / 8)
    return STARKV_ERR_LIMIT;
  return STARKV_OK;
}

size_t starkv_fp8_gemm_workspace_bytes(const starkv_fp8_gemm_desc* d) {
  Fp8Space s;
  return plan_fp8(d, s) ? 0 : s.total;
}

int starkv_fp8_gemm(const starkv_fp8_gemm_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  Fp8Space sp;
  int st = plan_fp8(d, sp);
  if (st) return st;
  if (d->m == 0) return STARKV_OK;
  const bool q = d->dtype != STARKV_E4M3;
  const int n_out = d->silu_mul ? d->n / 2 : d->n, os = esize(d->out_dtype), ss = scale_size(d->scale_dtype);
  if (!d->x || !d->w || !d->w_scale || !d->out || (!q && !d->x_scale)) return STARKV_ERR_NULL;
  if ((d->m > 1 && (d->x_stride < d->k || d->out_stride < n_out || (d->residual && d->residual_stride < n_out))) ||
      (d->n > 1 && d->w_stride < d->k) || d->w_scale_stride_r < 0 || d->w_scale_stride_b < 0 ||
      (!q && (d->x_scale_stride_r < 0 || d->x_scale_stride_b < 0)))
    return STARKV_ERR_SHAPE;
  if (!rows_e4m3(d->w, d->w_stride) || (q ? !al(d->x, 2) : !rows_e4m3(d->x, d->x_stride)) || !al(d->out, os) ||
      !al(d->residual, os) || !al(d->w_scale, ss) || (!q && !al(d->x_scale, ss)))
    return STARKV_ERR_ALIGN;
  if (sp.total) {
    if (!workspace || workspace_bytes < sp.total) return STARKV_ERR_WORKSPACE;
    if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
  }
  // tiles in LDS: a tile's rows (256, the up rows half a weight further) and their scales at 32-bit offsets
  if (!sp.plan.few) {
    const int64_t lim = ((int64_t)1 << 32) - 1, wr = 256 + (d->silu_mul ? d->n / 2 : 0);
    if ((q ? round_up(d->k, 16) : d->x_stride) > (lim - d->k) / 256 || d->w_stride > (lim - d->k) / wr ||
        (!q && d->x_scale_stride_r > lim / 1024) || (d->silu_mul && d->w_scale_stride_r > lim / (d->n / 256 + 8)))
      return STARKV_ERR_LIMIT;
  }
  Fp8GemmArgs a = {};
  a.x = d->x; a.xs = d->x_stride; a.sx = d->x_scale; a.sxr = d->x_scale_stride_r; a.sxb = d->x_scale_stride_b;
  a.w = (const uint8_t*)d->w; a.ws = d->w_stride; a.sw = d->w_scale; a.swr = d->w_scale_stride_r; a.swb = d->w_scale_stride_b;
  a.res = d->residual; a.rs = d->residual_stride; a.out = d->out; a.os = d->out_stride;
  a.m = d->m; a.n = d->n; a.k = d->k; a.kb = (int)ceil_div(d->k, FP8_BLOCK); a.half = d->n / 2;
  hipStream_t s = (hipStream_t)stream;
  if (q) {
    char* ws = (char*)workspace;
    Fp8QuantArgs qa = {};
    qa.x = d->x; qa.xs = d->x_stride; qa.q = (uint8_t*)ws; qa.qs = round_up(d->k, 16);
    qa.s = ws + sp.off_s; qa.ssr = 1; qa.ssb = d->m;
    if (d->rms) { qa.rscale = (float*)(ws + sp.off_r); qa.rms_eps = d->rms_eps; }
    qa.rows = d->m; qa.k = d->k; qa.kb = a.kb; qa.vec = al(d->x, 16) && d->x_stride % 8 == 0;
    if ((st = launch_fp8_quant(qa, d->dtype, d->scale_dtype, s))) return st;
    a.x = qa.q; a.xs = qa.qs; a.sx = qa.s; a.sxr = 1; a.sxb = d->m; a.rscale = qa.rscale;
  }
  if (sp.plan.few) return launch_fp8_few(a, sp.plan, d->out_dtype, d->scale_dtype, d->silu_mul != 0, s);
  return launch_fp8_gemm(a, sp.plan, d->out_dtype, d->scale_dtype, d->silu_mul != 0, s);
}

static int plan_lp(const starkv_logprobs_desc* d, LogprobArgs& a, bool& wide, size_t& bytes) {
  if (!d) return STARKV_ERR_NULL;
  if (d->rows < 0 || d->vocab < 1 || d->top < 0 || d->top > d->vocab) return STARKV_ERR_SHAPE;
  if (d->top > STARKV_MAX_TOP || d->vocab > (1 << 24)) return STARKV_ERR_LIMIT;
  if (!act16(d->dtype) && d->dtype != STARKV_F32) return STARKV_ERR_DTYPE;
  a = LogprobArgs{};
  a.rows = d->rows; a.vocab = d->vocab; a.top = d->top;
  const LogprobPlan p = plan_logprobs(std::max(d->rows, 1), d->vocab, esize(d->dtype), device_cus());
  a.pieces = p.pieces;
  wide = p.wide;
  a.piece_len = (int)round_up(ceil_div(d->vocab, a.pieces), 1024);
  a.pieces = (int)ceil_div(d->vocab, a.piece_len);
  if ((int64_t)d->rows * a.pieces > INT32_MAX / 1024) return STARKV_ERR_LIMIT;
  const size_t stat = a256((size_t)d->rows * a.pieces * 16);
  bytes = a.pieces > 1 ? stat + (size_t)d->rows * a.pieces * d->top * 8 : 0;
  return STARKV_OK;
}

size_t starkv_token_logprobs_workspace_bytes(const starkv_logprobs_desc* d) {
  LogprobArgs a;
  bool wide;
  size_t bytes = 0;
  return plan_lp(d, a, wide, bytes) ? 0 : bytes;
}

int starkv_token_logprobs(const starkv_logprobs_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  LogprobArgs a;
  bool wide;
  size_t bytes = 0;
  const int st = plan_lp(d, a, wide, bytes);
  if (st) return st;
  if (d->rows == 0) return STARKV_OK;
  if (!d->logits || (d->tokens && !d->logprob) || (d->top && (!d->top_logprob || !d->top_id))) return STARKV_ERR_NULL;
  if (d->rows > 1 && d->stride < d->vocab) return STARKV_ERR_SHAPE;
  if (!al(d->logits, esize(d->dtype)) || !al(d->tokens, 8) || !al(d->logprob, 4) || !al(d->entropy, 4) ||
      !al(d->top_logprob, 4) || !al(d->top_id, 8))
    return STARKV_ERR_ALIGN;
  if (bytes) {
    if (!workspace || workspace_bytes < bytes) return STARKV_ERR_WORKSPACE;
    if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
    a.pstat = (float*)workspace;
    a.ptop = (uint64_t*)((char*)workspace + a256((size_t)d->rows * a.pieces * 16));
  }
  a.x = d->logits; a.xs = d->stride; a.tok = d->tokens;
  a.lp = d->logprob; a.ent = d->entropy; a.tlp = d->top_logprob; a.tid = d->top_id;
  return launch_logprobs(a, wide, d->dtype, (hipStream_t)stream);
}


// ---------------------------------------------------------------------------
// Bounded caches
// ---------------------------------------------------------------------------
static int check_scores_desc(const starkv_scores_desc* d) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->n_heads < 1 || d->seq_len < 1) return STARKV_ERR_SHAPE;
  if (d->batch > 65535 || d->n_heads > SCORE_MAX_H || d->seq_len > MAX_S) return STARKV_ERR_LIMIT;
  if (!act16(d->dtype) && d->dtype != STARKV_F32) return STARKV_ERR_DTYPE;
  // one workgroup of 256 threads a piece
  if ((int64_t)d->batch * d->n_heads * score_pieces(d->seq_len) * 256 > MAX_THREADS_1D) return STARKV_ERR_LIMIT;
  return STARKV_OK;
}

size_t starkv_attention_scores_workspace_bytes(const starkv_scores_desc* d) {
  return check_scores_desc(d) ? 0 : (size_t)d->batch * d->n_heads * score_pieces(d->seq_len) * 8;
}

int starkv_attention_scores(const starkv_scores_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = check_scores_desc(d);
  if (st) return st;
  if (!d->logits || !d->scores) return STARKV_ERR_NULL;
  if (d->stride_b < 0 || d->stride_h < 0 || (d->batch > 1 && d->scores_stride_b < d->seq_len)) return STARKV_ERR_SHAPE;
  if (!al(d->logits, esize(d->dtype)) || !al(d->scores, 4)) return STARKV_ERR_ALIGN;
  if (!workspace || workspace_bytes < starkv_attention_scores_workspace_bytes(d)) return STARKV_ERR_WORKSPACE;
  if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
  ScoreArgs a = {};
  a.x = d->logits; a.x_sb = d->stride_b; a.x_st = 32; a.x_sh = d->stride_h;
  a.B = d->batch; a.H = d->n_heads; a.S = d->seq_len; a.add = d->add != 0;
  a.stat = (float2*)workspace; a.n_max = score_pieces(d->seq_len);
  a.out = d->scores; a.o_sb = d->scores_stride_b;
  return launch_scores(a, d->dtype, (hipStream_t)stream);
}

int starkv_decode_attention_scores(const starkv_decode_desc* d, float* scores, int64_t scores_stride_b, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  if (!scores) return STARKV_ERR_NULL;
  return decode_impl(d, workspace, workspace_bytes, stream, nullptr, scores, scores_stride_b);
}

static int check_select(const starkv_select_desc* d, SelectArgs& a, size_t& bytes) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 0 || d->length < 0 || d->sinks < 0 || d->recent < 0 || d->keep > d->length ||
      (int64_t)d->sinks + d->recent > d->keep)
    return STARKV_ERR_SHAPE;
  if (d->length > MAX_S || d->batch > 65535) return STARKV_ERR_LIMIT;
  a = SelectArgs{d->scores, d->scores_stride_b, d->positions, d->positions_stride_b, d->length, d->keep, d->sinks, d->recent, d->batch};
  const int fixed = d->sinks + d->recent, n = d->length - fixed;
  a.piece_len = select_piece(n, d->keep - fixed);
  bytes = 0;
  if (!a.piece_len || !d->batch) return STARKV_OK;
  a.pieces = (int)ceil_div(n, a.piece_len);
  bytes = a256((size_t)3 * d->batch * a.pieces * 2048 * 4) + (size_t)d->batch * 3 * 8;
  return STARKV_OK;
}

size_t starkv_select_positions_workspace_bytes(const starkv_select_desc* d) {
  SelectArgs a;
  size_t bytes;
  return check_select(d, a, bytes) ? 0 : bytes;
}

int starkv_select_positions(const starkv_select_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  SelectArgs a;
  size_t bytes;
  const int st = check_select(d, a, bytes);
  if (st) return st;
  if (d->batch == 0 || d->keep == 0) return STARKV_OK;
  if (!d->scores || !d->positions) return STARKV_ERR_NULL;
  if (d->batch > 1 && (d->scores_stride_b < 0 || d->positions_stride_b < d->keep)) return STARKV_ERR_SHAPE;
  if (!al(d->scores, 4) || !al(d->positions, 4)) return STARKV_ERR_ALIGN;
  if (bytes) {
    if (!workspace || workspace_bytes < bytes) return STARKV_ERR_WORKSPACE;
    if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
    a.hist = (uint32_t*)workspace;
    a.state = (int2*)((char*)workspace + a256((size_t)3 * a.B * a.pieces * 2048 * 4));
  }
  return launch_select(a, (hipStream_t)stream);
}

// Whether rows 0 .. L - 1 of `nb[h]` bytes of all heads and sequences lie apart (pitch[h] >= nb[h]): a move in place writes
// each of them once.
static bool rows_apart(int H, const int64_t* off, const int64_t* pitch, const int* nb, int B, int64_t sb, int L) {
  auto end = [&](int h) { return off[h] + (L - 1) * pitch[h] + nb[h]; };
  int64_t lo = INT64_MAX, hi = 0, row = 0;
  bool even = true, stacked = true, inside = true;   // one pitch; heads one behind another; heads side by side in a row
  int last = -1;
  for (int h = 0; h < H; ++h) {
    if (!nb[h]) continue;
    if (last >= 0) {
      even &= pitch[h] == pitch[last];
      stacked &= off[h] >= end(last);
      inside &= off[h] >= off[last] + nb[last];
    }
    last = h;
    lo = std::min(lo, off[h]); hi = std::max(hi, end(h)); row = std::max(row, off[h] + nb[h]);
  }
  if (last < 0) return true;
  row -= lo;
  inside &= even && row <= pitch[last];
  if (!stacked && !inside) {
    for (int g = 0; g < H; ++g)
      for (int h = 0; h < H; ++h) {                // off[g] <= off[h]; at equal pitch only the nearest rows can meet
        if (g == h || !nb[g] || !nb[h] || off[g] > off[h] || (off[g] == off[h] && g > h)) continue;
        const int64_t d = off[h] - off[g], p = pitch[g];
        if (pitch[h] != p) {
          if (off[h] < end(g)) return false;
        } else if ((d / p < L && d % p < nb[g]) || (d / p + 1 < L && p - d % p < nb[h])) {
          return false;
        }
      }
  }
  if (B == 1 || sb >= hi - lo || (inside && sb >= row && pitch[last] >= (B - 1) * sb + row)) return true;
  // sequences side by side within a head's row: heads beside one another in a position's row, or one behind another
  bool rows = true, beside = even, behind = true;
  int prev = -1;
  for (int h = 0; h < H; ++h) {
    if (!nb[h]) continue;
    rows &= sb >= nb[h] && pitch[h] >= (B - 1) * sb + nb[h];
    if (prev >= 0) {
      beside &= off[h] >= off[prev] + (B - 1) * sb + nb[prev];
      behind &= off[h] >= end(prev) + (B - 1) * sb;
    }
    beside &= off[h] + (B - 1) * sb + nb[h] - lo <= pitch[h];
    prev = h;
  }
  if (rows && (beside || behind)) return true;
  // each head's sequences one behind another, and the heads' ranges apart
  for (int g = 0; g < H; ++g) {
    if (!nb[g]) continue;
    if (sb < end(g) - off[g]) return false;
    for (int h = 0; h < H; ++h)
      if (g != h && nb[h] && off[g] <= off[h] && off[h] < end(g) + (B - 1) * sb) return false;
  }
  return true;
}

int starkv_keep_positions(const starkv_keep_desc* d, void* stream) {
  if (!d) return STARKV_ERR_NULL;
  if (d->batch < 1 || d->length < 0 || d->keep < 0 || d->keep > d->length) return STARKV_ERR_SHAPE;
  if (d->length > MAX_S || d->batch > 65535) return STARKV_ERR_LIMIT;
  const starkv_klatent& k = d->k;
  const starkv_vlatent& v = d->v;
  PVArgs pv = {};
  int vq = 0, st;
  if ((st = validate_klayout(k, d->dtype)) || (st = validate_v(v, pv, &vq))) return st;
  if (d->length == 0) return STARKV_OK;
  if (!d->positions && d->keep) return STARKV_ERR_NULL;
  const bool many = d->batch > 1, dense = k.format == STARKV_FMT_DENSE, two = k.format == STARKV_FMT_INT4_REF && k.split > 0;
  if (many && (d->positions_stride_b < d->keep || (d->scores && d->scores_stride_b < d->length))) return STARKV_ERR_SHAPE;
  if (!al(d->positions, 4) || !al(d->scores, 4)) return STARKV_ERR_ALIGN;
  MoveArgs a = {};
  a.pos = d->positions; a.p_sb = d->positions_stride_b; a.keep = d->keep; a.length = d->length; a.err = d->error_flag;
  const int es = dense ? 2 : 1, H = k.n_kv_heads, split = two ? k.split : 128;
  const bool a8 = two ? k.split_format == STARKV_FMT_INT8_SYM : k.format == STARKV_FMT_INT8_SYM;
  a.k1 = (uint8_t*)k.data; a.k1_sb = k.stride_b * es;
  a.k2 = (uint8_t*)k.data2; a.k2_sb = k.stride2_b;
  bool lower = false;
  for (int h = 0; h < H; ++h) {
    const int r = k.rank[h], up = std::min(r, split);
    a.off1[h] = k.head_offset[h] * es; a.pitch1[h] = k.pos_stride[h] * es;
    a.nb1[h] = dense ? 2 * r : a8 ? up : (up + 1) / 2;
    if (!two || r <= split) continue;
    lower = true;
    a.off2[h] = k.head_offset2[h]; a.pitch2[h] = k.pos_stride2[h]; a.nb2[h] = (r - split + 1) / 2;
  }
  a.Hk = H;
  if (!dense) {
    a.ks1 = (uint8_t*)k.scale; a.ks1_sb = 2 * k.scale_stride_b; a.ks1_sh = 2 * k.scale_stride_h;
    a.units[MOVE_KS1] = H;
  }
  if (lower) {
    a.ks2 = (uint8_t*)k.scale2; a.ks2_sb = 2 * k.scale2_stride_b; a.ks2_sh = 2 * k.scale2_stride_h;
    a.units[MOVE_KS2] = H;
  }
  const int B = d->batch, L = d->length;
  if (!rows_apart(H, a.off1, a.pitch1, a.nb1, B, a.k1_sb, L) || !rows_apart(H, a.off2, a.pitch2, a.nb2, B, a.k2_sb, L))
    return STARKV_ERR_SHAPE;
  int64_t s_off[2][K_MAX_KV], s_pitch[K_MAX_KV];
  int s_nb[2][K_MAX_KV];
  for (int h = 0; h < H; ++h) {
    s_off[0][h] = h * a.ks1_sh; s_off[1][h] = h * a.ks2_sh; s_pitch[h] = 2;
    s_nb[0][h] = dense ? 0 : 2; s_nb[1][h] = lower ? 2 : 0;
  }
  if (!rows_apart(H, s_off[0], s_pitch, s_nb[0], B, a.ks1_sb, L) || !rows_apart(H, s_off[1], s_pitch, s_nb[1], B, a.ks2_sb, L))
    return STARKV_ERR_SHAPE;
  // V rows, the lower block's, their scales and zero points
  const int vs = vq == VQ_DENSE ? 2 : 1, groups = vq == VQ_G64 ? (v.rank + 63) / 64 : 1;
  a.v[0] = {(uint8_t*)v.data, v.stride_b * vs, v.stride_s * vs, vq == VQ_DENSE ? 2 * v.rank : pv.xnb};
  if (pv.x2) a.v[1] = {(uint8_t*)v.data2, v.stride2_b, v.stride2_s, pv.x2nb};
  if (vq != VQ_DENSE) a.v[2] = {(uint8_t*)v.scale, 2 * v.scale_stride_b, 2 * v.scale_stride_s, 2 * groups};
  if (pv.x2) a.v[3] = {(uint8_t*)v.scale2, 2 * v.scale2_stride_b, 2 * v.scale2_stride_s, 2};
  if (vq == VQ_G64) a.v[4] = {(uint8_t*)v.zero, 2 * v.scale_stride_b, 2 * v.scale_stride_s, 2 * groups};
  int nk1 = 0, nk2 = 0;
  for (int h = 0; h < H; ++h) { nk1 = std::max(nk1, a.nb1[h]); nk2 = std::max(nk2, a.nb2[h]); }
  a.units[MOVE_K1] = H * (int)ceil_div(nk1, MOVE_SLICE);
  a.units[MOVE_K2] = lower ? H * (int)ceil_div(nk2, MOVE_SLICE) : 0;
  for (int i = 0; i < MOVE_SCORES - MOVE_V; ++i) a.units[MOVE_V + i] = (int)ceil_div(a.v[i].nb, MOVE_SLICE);
  for (int i = 0; i < MOVE_SCORES - MOVE_V; ++i) {
    const int64_t at = 0, pitch = a.v[i].pitch;
    if (a.v[i].nb && (pitch < a.v[i].nb || !rows_apart(1, &at, &pitch, &a.v[i].nb, B, a.v[i].sb, L))) return STARKV_ERR_SHAPE;
  }
  if (d->scores) { a.scores = d->scores; a.scores_sb = d->scores_stride_b; a.units[MOVE_SCORES] = 1; }
  a.B = B;
  for (int k = 0; k < MOVE_KINDS; ++k) a.per_row += a.units[k];
  if ((int64_t)a.per_row * B > MAX_THREADS_1D / 1024 - 8) return STARKV_ERR_LIMIT;       // workgroups of 1024 threads
  return launch_move(a, (hipStream_t)stream);
}

// ---------------------------------------------------------------------------
// Decode over a shared prefix
// ---------------------------------------------------------------------------
namespace {

// Up to so many own positions P V takes four column tiles a wave: more column blocks and fewer splits, whose partials are
// most of what short ones move (with the join, 8 x 333 of bf16, Rv 1228: 27 us, as decode has it 33; 16 x 512 of fp16, Rv
// 1640: 34, 41; 16 x 2048: 49, 53; 16 x 8192: 118, 112)
constexpr int PX_OWN_SHORT = 4096;
constexpr int64_t PX_MAX_ROWS = 1 << 20;           // (sequence, query head) rows of a call

// offsets of a packed prefix
struct PrefixSpace {
  int strips, Rvp, ks_max;
  int64_t xkoff[K_MAX_KV], xboff[K_MAX_KV];
  size_t off_xk, off_xb, off_xv, total;
};

int prefix_space(int n_kv, const int* rank, int Rv, int P, PrefixSpace& s) {
  if (n_kv < 1 || P < 1) return STARKV_ERR_SHAPE;
  if (n_kv > K_MAX_KV || P > MAX_S) return STARKV_ERR_LIMIT;
  if (!rank) return STARKV_ERR_NULL;
  if (Rv < 1 || Rv > MAX_RV) return STARKV_ERR_RANK;
  s = PrefixSpace{};
  s.strips = (int)ceil_div(P, PX_STRIP);
  s.Rvp = (int)round_up(Rv, 32);
  int64_t k = 0, b = 0;
  for (int h = 0; h < n_kv; ++h) {
    if (rank[h] < 1 || rank[h] > 128) return STARKV_ERR_RANK;
    s.xkoff[h] = k; s.xboff[h] = b;
    const int nc = (rank[h] + 7) / 8;
    k += (int64_t)s.strips * 2 * nc * 512;
    b += (int64_t)((nc + 1) / 2) * 4096;
    s.ks_max = std::max(s.ks_max, (nc + 1) / 2);
  }
  s.off_xk = PX_HEAD_BYTES;
  s.off_xb = s.off_xk + (size_t)k;
  s.off_xv = s.off_xb + (size_t)b;
  s.total = s.off_xv + (size_t)s.strips * PX_STRIP * s.Rvp * 2;
  return STARKV_OK;
}

int check_pack(const starkv_prefix_pack_desc* d, PrefixSpace& s) {
  if (!d) return STARKV_ERR_NULL;
  if (!act16(d->dtype)) return STARKV_ERR_DTYPE;
  if (d->k.format != STARKV_FMT_DENSE || d->v.format != STARKV_FMT_DENSE) return STARKV_ERR_FORMAT;
  PVArgs pv = {};
  int vq = 0, st;
  if ((st = validate_klayout(d->k, d->dtype)) || (st = validate_v(d->v, pv, &vq))) return st;
  if (!d->k.bk || !d->k.bk_head_offset) return STARKV_ERR_NULL;
  if (d->k.bk_row_stride < HEAD_DIM) return STARKV_ERR_SHAPE;
  return prefix_space(d->k.n_kv_heads, d->k.rank, d->v.rank, d->length, s);
}

// Whether a call's own logits are formed beside the prefix's
bool own_logits_here(const starkv_decode_desc& o) { return o.k.format == STARKV_FMT_DENSE; }

struct PrefixLayout {
  DecodeLayout own;
  PrefixSpace space;
  bool has_own, own_here;
  int oc_len, gs, M, Mp, bm, tiles_m, tiles_n, n_split, sp_len, n_ch, ch_len, n_hg, sc, n_sl;
  size_t off_p, off_stat, off_cmax, off_rmax, off_part, off_lsum, off_jsum, off_jmax, off_ypart, total;
};

// Strips per P V split: the least modelled time in strips (about 1 us each), rounds of one workgroup a CU, each its strips
// and a fixed time, and 0.12 for each split that the join adds up.  A round of workgroups that is hardly begun costs as
// much as a full one (65536 positions of 512 rows in 19 splits of 14 tiles: 198 us, in 36 161, in 18 152); 16384 of 128 rows
// in 128 splits of 2 tiles: 13.8 us and 15 for the join, in 64 14.6 and 11.3.
int prefix_split_len(int tiles, int cus, int strips) {
  int best = 0;
  double least = 0;
  // as many splits as whole rounds hold, and halves and quarters of a round
  for (int quarters = 1; quarters <= 32; quarters = quarters < 4 ? 2 * quarters : quarters + 4) {
    const int want = (int)std::max<int64_t>(1, std::min<int64_t>((int64_t)quarters * cus / 4 / tiles, PX_MAX_SPLITS));
    const int len = (int)ceil_div(strips, want);
    const int64_t n = ceil_div(strips, len);
    const double t = (double)ceil_div(tiles * n, cus) * (len + 3.0) + 0.12 * (double)n;
    if (!best || t < least * 0.9999) { best = len; least = t; }
  }
  return best;
}

int prefix_layout(const starkv_prefix_decode_desc* d, PrefixLayout& L) {
  if (!d) return STARKV_ERR_NULL;
  const starkv_decode_desc& o = d->own;
  L = PrefixLayout{};
  int st;
  if ((st = prefix_space(d->n_kv_heads, d->rank, d->v_rank, d->length, L.space))) return st;
  L.has_own = o.seq_len != 0;
  if (L.has_own) {
    int n_wg = 0, k1pc = 1, vq = 0;
    if ((st = validate_decode(&o, &L.gs, &n_wg, &k1pc, &vq))) return st;
    if (o.k.n_kv_heads != d->n_kv_heads || o.v.rank != d->v_rank) return STARKV_ERR_SHAPE;
    for (int h = 0; h < d->n_kv_heads; ++h)
      if (o.k.rank[h] != d->rank[h]) return STARKV_ERR_SHAPE;
    L.own = decode_layout(o.batch, o.n_q_heads, d->n_kv_heads, o.seq_len, o.v.rank, n_wg, k1pc, vq, v_row_bytes(o.v),
                          o.dtype == STARKV_F16, vq == VQ_DENSE && o.seq_len <= PX_OWN_SHORT ? 4 : 0);
    L.own_here = own_logits_here(o);
    if (L.own_here) {
      // chunks of at least one tile a wave, two workgroups a CU
      const int tiles = (int)ceil_div(o.seq_len, TILE);
      const int64_t want = std::max<int64_t>(1, 2 * device_cus() / ((int64_t)o.batch * d->n_kv_heads));
      L.oc_len = (int)round_up(ceil_div(tiles, want), 8);
      L.own.n_c1 = (int)ceil_div(tiles, L.oc_len);
    }
  } else {
    if (o.batch < 1 || o.head_dim != HEAD_DIM || o.n_q_heads < 1 || o.n_q_heads % d->n_kv_heads) return STARKV_ERR_SHAPE;
    if (!act16(o.dtype)) return STARKV_ERR_DTYPE;
    if (o.n_q_heads > K2_MAX_H) return STARKV_ERR_LIMIT;
    if (!o.q || !o.uv || !o.out || !o.rope_table) return STARKV_ERR_NULL;
    if (o.uv_row_stride < d->v_rank) return STARKV_ERR_SHAPE;
    if (o.out_dtype != 0 && o.out_dtype != o.dtype && o.out_dtype != STARKV_F32) return STARKV_ERR_DTYPE;
    L.gs = o.n_q_heads / d->n_kv_heads;
  }
  const int B = o.batch, Hq = o.n_q_heads, cus = device_cus(), strips = L.space.strips, Rvp = L.space.Rvp;
  if ((int64_t)B * Hq > PX_MAX_ROWS || B > 65535) return STARKV_ERR_LIMIT;
  L.M = B * Hq;
  L.bm = L.M <= 64 ? 64 : L.M <= 128 ? 128 : 256;
  L.tiles_m = (int)ceil_div(L.M, L.bm);
  L.Mp = L.tiles_m * L.bm;
  L.tiles_n = (int)ceil_div(Rvp, PX_BN);
  const int tiles = L.tiles_m * L.tiles_n;
  L.sp_len = prefix_split_len(tiles, cus, strips);
  L.n_split = (int)ceil_div(strips, L.sp_len);
  // logits: two workgroups a CU, each of its eight waves a strip at a time
  const int zb = (int)ceil_div((int64_t)B * L.gs, 32 * PX_GROUPS);
  const int64_t want = std::max<int64_t>(1, 2 * cus / ((int64_t)d->n_kv_heads * zb));
  L.ch_len = (int)round_up(ceil_div(strips, want), 8);
  L.n_ch = (int)ceil_div(strips, L.ch_len);
  L.n_hg = head_groups(Hq);
  // columns of an up-projection workgroup: wide ones read whole lines of the partials, narrow ones fill the CUs
  const int64_t row_blocks = (int64_t)d->n_kv_heads * ceil_div((int64_t)B * L.gs, 32);
  L.sc = row_blocks * ceil_div(d->v_rank, 128) >= cus ? 128 : row_blocks * ceil_div(d->v_rank, 64) >= cus ? 64 : 32;
  L.n_sl = (int)ceil_div(d->v_rank, L.sc);
  const size_t BQ = (size_t)B * L.n_hg, Mp = L.Mp;
  size_t off = L.has_own ? L.own.total : 0;
  auto take = [&](size_t& at, size_t n) { at = off; off = a256(off + n); };
  if (L.own_here) take(L.own.off_cmax, (size_t)B * Hq * L.own.n_c1 * 4);
  take(L.off_p, (size_t)strips * 8 * Mp * 16);
  take(L.off_stat, (size_t)strips * Mp * 8);
  take(L.off_cmax, (size_t)L.n_ch * Mp * 4);
  take(L.off_rmax, Mp * 4);
  take(L.off_part, (size_t)L.n_split * L.M * Rvp * 4);
  take(L.off_lsum, (size_t)L.n_split * Mp * 4);
  take(L.off_jsum, BQ * 32 * 4);
  take(L.off_jmax, (size_t)L.M * 4);
  take(L.off_ypart, (size_t)L.n_sl * L.M * HEAD_DIM * 4);
  L.total = off;
  return STARKV_OK;
}

}  // namespace

size_t starkv_prefix_bytes(const starkv_prefix_pack_desc* d) {
  PrefixSpace s;
  return check_pack(d, s) ? 0 : s.total;
}

int starkv_prefix_pack(const starkv_prefix_pack_desc* d, void* stream) {
  PrefixSpace s;
  const int st = check_pack(d, s);
  if (st) return st;
  if (!d->prefix) return STARKV_ERR_NULL;
  if (d->prefix_bytes < s.total) return STARKV_ERR_WORKSPACE;
  if (!al(d->prefix, 256) || !al(d->k.data, 2) || !al(d->v.data, 2) || !al(d->k.bk, 2)) return STARKV_ERR_ALIGN;
  PrefixPackArgs a = {};
  a.k = d->k.data; a.bk = d->k.bk; a.v = d->v.data;
  a.bk_rs = d->k.bk_row_stride; a.v_ss = d->v.stride_s;
  a.Hkv = d->k.n_kv_heads; a.P = d->length; a.strips = s.strips; a.Rv = d->v.rank; a.Rvp = s.Rvp;
  a.scale_v = d->dtype == STARKV_BF16;
  int rmax = 1;
  for (int h = 0; h < a.Hkv; ++h) {
    a.koff[h] = d->k.head_offset[h]; a.kpitch[h] = d->k.pos_stride[h]; a.bkoff[h] = d->k.bk_head_offset[h];
    a.rank[h] = d->k.rank[h]; a.xkoff[h] = s.xkoff[h]; a.xboff[h] = s.xboff[h];
    rmax = std::max(rmax, a.rank[h]);
  }
  a.bound = 1.4143 * rmax * std::max(1.0, std::fabs((double)d->attention_scaling));
  char* p = (char*)d->prefix;
  a.head = (float*)p; a.xk = (uint8_t*)p + s.off_xk; a.xb = (uint8_t*)p + s.off_xb; a.xv = (uint4*)(p + s.off_xv);
  return launch_prefix_pack(a, d->dtype, (hipStream_t)stream);
}

size_t starkv_prefix_decode_workspace_bytes(const starkv_prefix_decode_desc* d) {
  PrefixLayout L;
  return prefix_layout(d, L) ? 0 : L.total;
}

int starkv_prefix_decode(const starkv_prefix_decode_desc* d, void* workspace, size_t workspace_bytes, void* stream) {
  PrefixLayout L;
  int st = prefix_layout(d, L);
  if (st) return st;
  const starkv_decode_desc& o = d->own;
  if (!d->prefix || !d->turn_cos || !d->turn_sin) return STARKV_ERR_NULL;
  if (d->prefix_bytes < L.space.total || round_up(d->length, PX_STRIP) > o.rope_max_positions) return STARKV_ERR_SHAPE;
  if (!al(d->prefix, 256) || !al(o.q, 2)) return STARKV_ERR_ALIGN;
  const bool score = d->scores && L.has_own;
  if (score && (st = check_scores(&o, d->scores, d->scores_stride_b))) return st;
  if (!workspace || workspace_bytes < L.total) return STARKV_ERR_WORKSPACE;
  if (!al(workspace, 256)) return STARKV_ERR_ALIGN;
  char* ws = (char*)workspace;
  hipStream_t s = (hipStream_t)stream;
  PrefixLogitsArgs a = {};
  const char* p = (const char*)d->prefix;
  a.head = (const float*)p; a.xk = (const uint8_t*)p + L.space.off_xk; a.xb = (const uint8_t*)p + L.space.off_xb;
  a.xv = (const uint4*)(p + L.space.off_xv);
  for (int h = 0; h < d->n_kv_heads; ++h) {
    a.xkoff[h] = L.space.xkoff[h]; a.xboff[h] = L.space.xboff[h]; a.rank[h] = d->rank[h];
  }
  for (int i = 0; i < 64; ++i) { a.cos_p[i] = d->turn_cos[i]; a.sin_p[i] = d->turn_sin[i]; }
  a.rope = (const uint4*)o.rope_table;
  a.q = o.q; a.q_sb = o.q_stride_b; a.q_sh = o.q_stride_h;
  a.scale = o.scale;
  a.P = d->length; a.strips = L.space.strips; a.B = o.batch; a.Hq = o.n_q_heads; a.Hkv = d->n_kv_heads; a.gs = L.gs;
  a.Rvp = L.space.Rvp; a.ks_max = L.space.ks_max; a.M = L.M; a.Mp = L.Mp;
  a.p = (uint4*)(ws + L.off_p); a.stat = (float2*)(ws + L.off_stat);
  a.cmax = (float*)(ws + L.off_cmax); a.n_ch = L.n_ch; a.ch_len = L.ch_len; a.rmax = (float*)(ws + L.off_rmax);
  a.bm = L.bm; a.tiles_m = L.tiles_m; a.tiles_n = L.tiles_n; a.n_split = L.n_split; a.sp_len = L.sp_len;
  a.part = (float*)(ws + L.off_part); a.lsum = (float*)(ws + L.off_lsum);
  a.n_hg = L.n_hg; a.jsum = (float*)(ws + L.off_jsum);
  a.uv = o.uv; a.uv_rs = o.uv_row_stride; a.Rv = d->v_rank; a.sc = L.sc; a.n_sl = L.n_sl; a.ypart = (float*)(ws + L.off_ypart);
  a.out = o.out; a.o_sb = o.out_stride_b; a.o_sh = o.out_stride_h;
  a.jmax = score ? (float*)(ws + L.off_jmax) : nullptr;
  if (L.has_own) {
    a.own_max = (float*)(ws + L.own.off_cmax); a.own_sum = (const float*)(ws + L.own.off_psum);
    a.own_part = ws + L.own.off_part;
    a.n_c1 = L.own.n_c1; a.n_c2 = L.own.pv.n_c2; a.own_Rvp = L.own.pv.Rvp; a.own_part16 = L.own.part16;
    a.S = o.seq_len;
    a.mask = o.mask; a.m_sb = o.mask_stride_b; a.m_sh = o.mask_stride_h; a.mask_dtype = o.mask_dtype;
    a.ol = (float*)(ws + L.own.off_logits); a.ol_sb = (int64_t)o.n_q_heads * L.own.S_pad; a.ol_st = (int64_t)o.n_q_heads * TILE;
    if (L.own_here) {
      a.oc_len = L.oc_len;
      a.ox = o.k.data; a.ox_sb = o.k.stride_b;
      for (int h = 0; h < d->n_kv_heads; ++h) { a.oxoff[h] = o.k.head_offset[h]; a.oxpitch[h] = o.k.pos_stride[h]; }
      a.last_pos = o.last_pos_device;
    } else if ((st = decode_logits(&o, L.own, L.gs, ws, s))) {
      return st;
    }
  }
  if ((st = launch_prefix_logits(a, o.dtype, L.own_here, s))) return st;
  PVArgs pa;
  if (L.has_own && (st = decode_pv(&o, L.own, ws, s, pa))) return st;
  if ((st = launch_prefix_pv(a, s)) || (st = launch_prefix_up(a, o.dtype, o.out_dtype == STARKV_F32, s))) return st;
  if (score) return decode_scores(&o, L.own, ws, a.jmax, 1, a.jsum, 1, d->scores, d->scores_stride_b, s);
  return STARKV_OK;
}

}  // extern "C"
