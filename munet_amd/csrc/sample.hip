// The next token of each row of logits, drawn with given uniform numbers.
//
// Tokens are ordered by value (down), then index (up); z = (x - max) / T and
// w = e^z.  Each filter keeps a prefix of that order: top-k the first k, top-p
// the fewest whose weights reach p of the weight that top-k leaves, min-p those
// with w >= min_p.  The shortest prefix is kept (one token at least), and the
// token drawn is the first, in index order, at which the kept weights' running
// sum passes u times their sum.
//
// A prefix is a threshold: every value above it, and the first few (in index
// order) equal to it.  Nothing is sorted: the threshold is found by a histogram
// of counts and weights over the values, refined where the prefix ends.
//
// Weights are 64-bit whole numbers, round(w 2^S) with S = 44 up to 2^19 tokens: whole
// sums do not depend on their order, so a call's result does not depend on how its
// threads meet, and 2^-45 of the largest weight is lost per token, where fp32
// sums over 10^5 tokens would move one draw in a hundred to a neighbour.
#include "mh_common.hpp"
#include "mh_kernels.hpp"

namespace mh {
namespace {

constexpr int kBins = 2048;
constexpr int kMaxGroups = 1024;

// Float -> unsigned key with the same order; -0 takes +0's key (the two tie).
__device__ __forceinline__ uint32_t value_key(float v) {
  uint32_t u = __float_as_uint(v);
  if (u == 0x80000000u) u = 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}

// 2^(S + y), y = (x - max) log2(e) / T <= 0, and rounded to a whole number.  With
// 128 (S + y) = n + r, n whole and |r| <= 1/2: 2^(n >> 7) times the table's 2^(n mod 128
// / 128) times e^(r ln 2 / 128) by its series to the third power (the next term is
// below 2^-38: one in 10^8 draws from 10^5 equal tokens could move).  Eleven 64-bit
// operations, where the series without a table takes twenty (sums of 131072
// weights in 200 rows 92 us | 77).
constexpr int kTable = 128;
struct Weigh {
  const double *table;  // 2^(j / 128)
  double max, per;      // y = (x - max) * per
  float least;          // logits below weigh nothing
  int S;
  bool inf;  // the largest logit is infinite: it weighs 1, all others nothing
  __device__ __forceinline__ void start(float xmax, float T) {
    max = double(xmax);
    per = 1.4426950408889634074 / double(T);
    inf = xmax == __builtin_inff();
    // (-inf weighs nothing at any temperature)
    least = inf ? xmax : fmaxf(float(max - double(S) / per), -3.402823466e38f);
  }
  __device__ __forceinline__ double scaled(float x) const {
    constexpr double round = 6755399441055744.0;  // 1.5 * 2^52: a sum's low bits are the number rounded
    constexpr double c1 = 0.69314718055994530942 / kTable, c2 = c1 * c1 / 2, c3 = c1 * c1 * c1 / 6;
    const double t = inf ? double(kTable) * S : fma(double(x) - max, per * kTable, double(kTable) * S), m = t + round;
    const int n = int(uint32_t(__double_as_longlong(m)));
    const double r = t - (m - round), e = r * fma(r, fma(r, c3, c2), c1), b = table[n & (kTable - 1)];
    const uint64_t v = uint64_t(__double_as_longlong(fma(b, e, b))) + (uint64_t(uint32_t(n >> 7)) << 52);
    return x >= least ? __longlong_as_double((long long)v) : 0.0;
  }
  static __device__ __forceinline__ uint64_t whole(double v) {
    // (below 2^52: the sum's low bits are the number rounded to nearest)
    return uint64_t(__double_as_longlong(v + 4503599627370496.0)) & ((uint64_t(1) << 52) - 1);
  }
  __device__ __forceinline__ uint64_t operator()(float x) const { return whole(scaled(x)); }
  // the table's entry j: e^(j ln 2 / 128) by its series
  static __device__ __forceinline__ double entry(int j) {
    const double t = j * (0.69314718055994530942 / kTable);
    double r = 1.0;
#pragma unroll
    for (int i = 20; i > 0; --i) r = fma(r, t / i, 1.0);
    return r;
  }
};

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((unsigned long long)v, o, 64);
  return v;
}
// inclusive sums over the lanes
template <class V> __device__ __forceinline__ V wave_scan(V v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const V u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

// A logit as the draw takes it: NaN never wins and weighs nothing, as -inf.
template <int DT> __device__ __forceinline__ float logit(typename Store<DT>::T v) {
  const float x = Store<DT>::dec(v);
  return x == x ? x : -__builtin_inff();
}

// f(logit, index) over a row, in any order: whole 16-byte chunks where the row's start
// allows it, single values before and after.
template <int DT, int NT, class F> __device__ __forceinline__ void each_value(const typename Store<DT>::T *row, int cols, F f) {
  typedef typename Store<DT>::T T;
  constexpr int E = 16 / sizeof(T);
  const int tid = threadIdx.x;
  const int head = min(int((16 - (uintptr_t(row) & 15)) & 15) / int(sizeof(T)), cols), chunks = (cols - head) / E;
  if (tid < head) f(logit<DT>(row[tid]), tid);
  const uint4 *c = reinterpret_cast<const uint4 *>(row + head);
#pragma unroll 4
  for (int i = tid; i < chunks; i += NT) {
    const uint4 w = c[i];
    float v[E];
    if constexpr (DT == F32) {
      v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    } else {
      dec8<DT>(w, v);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f(v[e] == v[e] ? v[e] : -__builtin_inff(), head + i * E + e);
  }
  const int tail = head + chunks * E + tid;
  if (tail < cols) f(logit<DT>(row[tail]), tail);
}

// A prefix of the order: values above K, and the first `ties` equal to it.
struct Cut {
  uint32_t K;
  uint32_t ties;
};

// One workgroup per row.
//  1. The largest logit, and the largest of each thread's own.
//  2. Top-k: the k-th of the threads' largest bounds the k-th logit from below: what
//     passes it, the top k and little more, goes into a list in LDS.  No weights
//     but those of the list.  Min-p alone: what passes its least weight.
//     Top-p of all tokens: a histogram of their weights; the tokens of the bin in
//     which the prefix ends go into the list.
//  3. The threshold by histograms over the list.
//  4. The draw: from the list by histograms of weight over its indexes, or, where more
//     is kept than the list, by the weights of groups of consecutive tokens (top-p:
//     added up while the list is gathered).
// Where a list does not hold what it should (thousands of equal logits), its histograms
// run over the row in memory instead.
template <int DT, int NT>
__global__ void __launch_bounds__(NT) sample_kernel(Sampling p, int S) {
  typedef typename Store<DT>::T T;
  constexpr int NW = NT / 64, kList = 4096;
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned int count[kBins];
  __shared__ unsigned long long group_mass[kMaxGroups];
  __shared__ unsigned int red[2][NW];
  __shared__ unsigned long long red64[NW];
  __shared__ uint32_t list_key[kList];
  __shared__ int list_at[kList];
  __shared__ int listed;
  __shared__ double table[kTable];
  __shared__ unsigned long long scan_mass[NW];
  __shared__ unsigned int scan_count[NW];
  __shared__ struct {
    uint32_t bin;
    uint32_t count;  // tokens above the bin
    unsigned long long mass;
  } at;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = blockIdx.x, V = p.cols;
  const T *row = static_cast<const T *>(p.logits) + long(r) * p.ld;
  const float T_ = p.temperature ? p.temperature[r] : 1.f;
  const bool greedy = !(T_ > 0.f);
  const int k = p.top_k ? p.top_k[r] : 0;
  const float tp = p.top_p ? p.top_p[r] : 1.f, mp = p.min_p ? p.min_p[r] : 0.f;
  const bool by_k = k > 0 && k < V, by_p = tp < 1.f, by_m = mp > 0.f;

  // ---- the largest value; with temperature 0 its first index too
  uint32_t own = 0;
  unsigned long long first = 0;  // (key, ~index)
  if (greedy) {
    each_value<DT, NT>(row, V, [&](float x, int i) {
      const unsigned long long c = (static_cast<unsigned long long>(value_key(x)) << 32) | (0xffffffffu - uint32_t(i));
      first = c > first ? c : first;
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const unsigned long long c = __shfl_xor(first, o, 64);
      first = c > first ? c : first;
    }
    if (lane == 0) red64[wave] = first;
    __syncthreads();
    for (int w = 0; w < NW; ++w) first = red64[w] > first ? red64[w] : first;
    if (tid == 0) {
      const bool none = uint32_t(first >> 32) <= value_key(-__builtin_inff());
      p.ids[r] = none ? -1 : int(0xffffffffu - uint32_t(first));
      if (p.logprob) p.logprob[r] = none ? -__builtin_inff() : 0.f;
    }
    return;
  }
  each_value<DT, NT>(row, V, [&](float x, int) { own = max(own, value_key(x)); });
  uint32_t top = own;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, uint32_t(__shfl_xor(top, o, 64)));
  if (lane == 0) red[0][wave] = top;
  if (tid < kTable) table[tid] = Weigh::entry(tid);
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NW; ++w) top = max(top, red[0][w]);
  const float xmax = key_value(top);
  if (top <= value_key(-__builtin_inff())) {  // nothing to draw from
    if (tid == 0) {
      p.ids[r] = -1;
      if (p.logprob) p.logprob[r] = -__builtin_inff();
    }
    return;
  }
  Weigh w;
  w.table = table;
  w.S = S;
  w.start(xmax, T_);
  // min-p: a weight below this (times 2^S) is dropped
  const double least = by_m ? double(fminf(mp, 1.f)) * __builtin_ldexp(1.0, S) : 0.0;
  // bins of equal width in z over the S bits that weigh anything
  const float per_bin = float(kBins) / float(S + 1), slope = fminf(float(w.per) * per_bin, 1e30f);
  auto bin_of = [&](float x) -> uint32_t { return x == xmax ? 0u : uint32_t(fminf((xmax - x) * slope, float(kBins - 1))); };

  auto clear = [&] {
    for (int i = tid; i < kBins; i += NT) {
      mass[i] = 0;
      count[i] = 0;
    }
    __syncthreads();
  };
  // Where a prefix of `goal` tokens or weight of the bins ends, and what lies above:
  // kBins / NT bins to a thread, its wave's sums before it, the waves' before those.
  auto find = [&](bool by_mass, uint64_t goal) {
    constexpr int PB = kBins / NT;
    __syncthreads();
    uint64_t bm[PB], m = 0;
    uint32_t bc[PB], c = 0;
#pragma unroll
    for (int i = 0; i < PB; ++i) {
      m += bm[i] = mass[tid * PB + i];
      c += bc[i] = count[tid * PB + i];
    }
    uint64_t ms = wave_scan((unsigned long long)m, lane);
    uint32_t cs = wave_scan(c, lane);
    if (lane == 63) {
      scan_mass[wave] = ms;
      scan_count[wave] = cs;
    }
    __syncthreads();
    for (int v = 0; v < wave; ++v) {
      ms += scan_mass[v];
      cs += scan_count[v];
    }
    const uint64_t up = by_mass ? ms : uint64_t(cs), down = by_mass ? ms - m : uint64_t(cs - c);
    if ((down < goal && up >= goal) || (tid == NT - 1 && up < goal)) {
      uint64_t am = ms - m;
      uint32_t ac = cs - c;
      int b = 0;
#pragma unroll
      for (int i = 0; i + 1 < PB; ++i)
        if (b == i && (by_mass ? am + bm[i] : uint64_t(ac) + bc[i]) < goal) {
          am += bm[i];
          ac += bc[i];
          ++b;
        }
      at.bin = tid * PB + b;
      at.count = ac;
      at.mass = am;
    }
    __syncthreads();
  };
  auto sum_of = [&](uint64_t m) -> uint64_t {
    m = wave_sum_u64(m);
    if (lane == 0) red64[wave] = m;
    __syncthreads();
    uint64_t s = 0;
#pragma unroll
    for (int i = 0; i < NW; ++i) s += red64[i];
    __syncthreads();
    return s;
  };
  // bins of the tokens of `each` that `in` takes
  auto fill = [&](auto each, auto in, auto where) {
    clear();
    each([&](float x, int) {
      if (in(x)) {
        const uint32_t b = where(x);
        atomicAdd(&count[b], 1u);
        const uint64_t m = w(x);
        if (m) atomicAdd(&mass[b], (unsigned long long)m);
      }
    });
  };
  // the exact end of a prefix of `goal` tokens or weight, in bin b0, with so much above the bin
  auto end_in = [&](auto each, bool by_mass, uint64_t goal, uint32_t b0, uint64_t am, uint64_t ac, uint64_t &above_mass) -> Cut {
    // the keys of that bin
    uint32_t lo = 0xffffffffu, hi = 0;
    each([&](float x, int) {
      if (bin_of(x) == b0) {
        const uint32_t kk = value_key(x);
        lo = min(lo, kk);
        hi = max(hi, kk);
      }
    });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      lo = min(lo, uint32_t(__shfl_xor(lo, o, 64)));
      hi = max(hi, uint32_t(__shfl_xor(hi, o, 64)));
    }
    if (lane == 0) {
      red[0][wave] = lo;
      red[1][wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      lo = min(lo, red[0][i]);
      hi = max(hi, red[1][i]);
    }
    __syncthreads();
    for (;;) {
      int sh = 0;
      while (((hi - lo) >> sh) >= uint32_t(kBins)) ++sh;
      fill(each, [&](float x) { const uint32_t kk = value_key(x); return bin_of(x) == b0 && kk >= lo && kk <= hi; },
           [&](float x) { return (hi - value_key(x)) >> sh; });
      find(by_mass, by_mass ? goal - am : goal - ac);
      const uint32_t sb = at.bin;
      am += at.mass;
      ac += at.count;
      __syncthreads();
      if (sh == 0) {
        const uint32_t K = hi - sb;
        above_mass = am;
        uint64_t ties = goal - ac;
        if (by_mass) {
          const uint64_t one = w(key_value(K));
          ties = one ? (goal - am + one - 1) / one : 1;
        }
        return Cut{K, uint32_t(ties > 0xffffffffu ? 0xffffffffu : ties)};
      }
      hi -= sb << sh;
      const uint32_t span = (1u << sh) - 1u;
      lo = hi - lo > span ? hi - span : lo;
    }
  };
  auto goal_p = [&](uint64_t total) -> uint64_t {  // the weight that top-p's prefix reaches
    const double g = __builtin_ceil(double(fmaxf(tp, 0.f)) * double(total));
    return g < 1.0 ? 1 : min(uint64_t(g), total);
  };
  auto shorter = [](Cut a, Cut b) { return b.K > a.K || (b.K == a.K && b.ties < a.ties) ? b : a; };
  // top-k's prefix over `each`, and top-p's of what it leaves
  auto of_top_k = [&](auto each) -> Cut {
    fill(each, [&](float) { return true; }, bin_of);
    find(false, uint64_t(k));
    uint64_t above = 0;
    const Cut c = end_in(each, false, uint64_t(k), at.bin, at.mass, at.count, above);
    if (!by_p) return c;
    const uint64_t goal = goal_p(above + uint64_t(c.ties) * w(key_value(c.K)));
    fill(each, [&](float) { return true; }, bin_of);
    find(true, goal);
    return shorter(c, end_in(each, true, goal, at.bin, at.mass, at.count, above));
  };
  // The index at which the running sum of `weight` over `each`, in index order,
  // passes goal: bins of consecutive indexes, refined to one.
  auto select = [&](auto each, uint64_t goal, auto weight) -> int {
    int lo = 0, bits = 0;
    while ((int64_t(kBins) << bits) < V) ++bits;
    for (;; bits = bits > 11 ? bits - 11 : 0) {
      __syncthreads();
      clear();
      each([&](float x, int i) {
        const int b = (i - lo) >> bits;
        if (i >= lo && b < kBins) {
          const uint64_t v = weight(x, i);
          if (v) atomicAdd(&mass[b], (unsigned long long)v);
        }
      });
      find(true, goal + 1);
      lo += int(at.bin) << bits;
      goal -= at.mass;
      if (bits == 0) return lo;
    }
  };
  // The threshold, and the index of its last tie that is kept.
  Cut cut{0u, 0xffffffffu};
  int last_tie = V;
  auto weight = [&](float x, int i) -> uint64_t {
    const uint32_t kk = value_key(x);
    if (kk < cut.K || (kk == cut.K && i > last_tie)) return 0;
    const double s = w.scaled(x);
    return s < least ? 0 : Weigh::whole(s);
  };
  auto cut_ties = [&](auto each) {
    uint32_t ties = 0;
    each([&](float x, int) { ties += value_key(x) == cut.K; });
    if (sum_of(ties) > cut.ties)
      last_tie = select(each, uint64_t(cut.ties) - 1, [&](float x, int) { return uint64_t(value_key(x) == cut.K); });
  };
  auto put = [&](int i, float x, uint64_t total) {
    p.ids[r] = i;
    // log(w / sum) from the logit itself: the whole weight has few bits where w is small
    if (p.logprob)
      p.logprob[r] = float((double(x) == w.max ? 0.0 : (double(x) - w.max) / double(T_)) - log(double(total) * __builtin_ldexp(1.0, -S)));
  };
  float u = p.u[r];
  u = u > 0.f ? u : 0.f;
  auto goal_of = [&](uint64_t total) -> uint64_t {
    const uint64_t g = uint64_t(double(u) * double(total));
    return g < total ? g : total - 1;  // u = 1: the last kept token
  };

  auto over_row = [&](auto f) { each_value<DT, NT>(row, V, f); };
  // A list of one token per thread is ordered by counting, for each, those before
  // it: a few steps over LDS where the histograms take a dozen barriers each
  // (top 50 of 131072: 57 us | 52).
  constexpr int kShort = NT < 512 ? NT : 512;
  // inclusive sums over the threads, and the last one's
  auto scan = [&](uint64_t v, uint64_t &total) -> uint64_t {
    uint64_t run = wave_scan((unsigned long long)v, lane);
    if (lane == 63) scan_mass[wave] = run;
    __syncthreads();
    total = 0;
    for (int i = 0; i < NW; ++i) {
      if (i < wave) run += scan_mass[i];
      total += scan_mass[i];
    }
    __syncthreads();
    return run;
  };
  // The list's token that ends the prefix: of k tokens; then of weight `goal`, with
  // `above` before the list (0: top-p's share of those k).
  auto short_cut = [&](int n, uint32_t k_, uint64_t above, uint64_t goal) {
    uint32_t rank = 0;
    if (tid < n) {
      const uint32_t kk = list_key[tid];
      const int i = list_at[tid];
      for (int j = 0; j < n; ++j) rank += list_key[j] > kk || (list_key[j] == kk && list_at[j] < i);
      mass[rank] = w(key_value(kk));
      count[rank] = uint32_t(tid);
    }
    __syncthreads();
    const uint64_t mine = uint32_t(tid) < k_ ? mass[tid] : 0;
    uint64_t total;
    const uint64_t run = scan(mine, total);
    if (goal == 0) goal = goal_p(total);
    const uint64_t need = goal > above + total ? total : goal - above;  // (~0: all k)
    if (tid == int(k_) - 1) at.bin = k_ - 1;
    __syncthreads();
    if (uint32_t(tid) < k_ && goal != ~uint64_t(0) && run >= need && run - mine < need) at.bin = uint32_t(tid);
    __syncthreads();
    const int last = int(count[at.bin]);
    cut.K = list_key[last];
    last_tie = list_at[last];
    __syncthreads();
  };
  auto draw_short = [&](int n) {
    if (tid < n) {
      const int i = list_at[tid];
      uint32_t rank = 0;
      for (int j = 0; j < n; ++j) rank += list_at[j] < i;
      mass[rank] = weight(key_value(list_key[tid]), i);
      count[rank] = uint32_t(tid);
    }
    __syncthreads();
    const uint64_t mine = tid < n ? mass[tid] : 0;
    uint64_t total;
    const uint64_t run = scan(mine, total), goal = goal_of(total);
    if (run > goal && run - mine <= goal) {
      const int e = int(count[tid]);
      put(list_at[e], key_value(list_key[e]), total);
    }
  };
  // Groups of consecutive tokens: f(logit, index) over one by a wave, in any order.
  int gs = 512;
  while ((V + gs - 1) / gs > kMaxGroups) gs *= 2;
  const int groups = (V + gs - 1) / gs;
  const bool chunks = ((uintptr_t(row) & 15) == 0);
  auto over_group = [&](int g, auto f) {
    const int from = g * gs, to = min(from + gs, V);
    if (chunks && to - from == gs) {
#pragma unroll 2
      for (int i = from + lane * 8; i < to; i += 512) {
        float v[8];
        if constexpr (DT == F32) {
          ld4<F32>(row + i, v);
          ld4<F32>(row + i + 4, v + 4);
        } else {
          dec8<DT>(*reinterpret_cast<const uint4 *>(row + i), v);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) f(v[e] == v[e] ? v[e] : -__builtin_inff(), i + e);
      }
    } else {
      for (int i = from + lane; i < to; i += 64) f(logit<DT>(row[i]), i);
    }
  };
  bool grouped = false;  // group_mass is filled

  // ---- the threshold
  if (by_p && !by_k) {
    clear();
    over_row([&](float x, int) {
      const uint64_t m = w(x);
      if (m) atomicAdd(&mass[bin_of(x)], (unsigned long long)m);
    });
    __syncthreads();
    uint64_t m = 0;
    for (int i = tid; i < kBins; i += NT) m += mass[i];
    const uint64_t goal = goal_p(sum_of(m));
    find(true, goal);
    const uint32_t b0 = at.bin;
    const uint64_t am = at.mass;
    if (tid == 0) listed = 0;
    __syncthreads();
    for (int g = wave; g < groups; g += NW) {
      uint64_t gm = 0;
      over_group(g, [&](float x, int i) {
        const uint32_t b = bin_of(x);
        if (b < b0) {
          const double s = w.scaled(x);
          gm += s < least ? 0 : Weigh::whole(s);
        } else if (b == b0) {
          const int n = atomicAdd(&listed, 1);
          if (n < kList) {
            list_key[n] = value_key(x);
            list_at[n] = i;
          }
        }
      });
      gm = wave_sum_u64(gm);
      if (lane == 0) group_mass[g] = gm;
    }
    __syncthreads();
    const int n = listed;
    uint64_t above = 0;
    if (n <= kList) {
      auto each = [&](auto f) {
        for (int i = tid; i < n; i += NT) f(key_value(list_key[i]), list_at[i]);
      };
      if (n <= kShort) {
        short_cut(n, uint32_t(n), am, goal);
      } else {
        cut = end_in(each, true, goal, b0, am, 0, above);
        cut_ties(each);
      }
      each([&](float x, int i) {
        const uint64_t v = weight(x, i);
        if (v) atomicAdd(&group_mass[i / gs], (unsigned long long)v);
      });
      grouped = true;
    } else {
      cut = end_in(over_row, true, goal, b0, am, 0, above);
      cut_ties(over_row);
    }
    __syncthreads();
  } else if (by_k || by_m) {
    uint32_t bound = kBins - 1;
    if (by_k && V > kShort) {
      const int owners = int(sum_of(own != 0));  // (threads with a logit)
      clear();
      // (of n threads' largest the k-th is passed by about -n log(1 - k / n) logits:
      // near n that is no bound, and the logits are counted instead)
      const bool bounded = k <= owners - owners / 10;
      if (bounded) {
        if (own) atomicAdd(&count[bin_of(key_value(own))], 1u);
      } else {
        over_row([&](float x, int) { atomicAdd(&count[bin_of(x)], 1u); });
      }
      find(false, uint64_t(k));
      bound = at.bin;
    }
    // (top-p goes by the weight of all that top-k leaves)
    if (by_m && !(by_k && by_p)) bound = min(bound, uint32_t(fminf(float(-log2(double(fminf(mp, 1.f)))) * per_bin + 2.f, float(kBins - 1))));
    if (tid == 0) listed = 0;
    __syncthreads();
    over_row([&](float x, int i) {
      if (bin_of(x) <= bound) {
        const int n = atomicAdd(&listed, 1);
        if (n < kList) {
          list_key[n] = value_key(x);
          list_at[n] = i;
        }
      }
    });
    __syncthreads();
    const int n = listed;
    // (fewer than k where min-p leaves fewer: then it decides)
    const bool holds = n <= kList && (n >= k || by_m || V <= kList);
    auto each = [&](auto f) {
      for (int i = tid; i < n; i += NT) f(key_value(list_key[i]), list_at[i]);
    };
    if (holds && n <= kShort) {
      if (by_k && n >= k) short_cut(n, uint32_t(k), 0, by_p ? 0 : ~uint64_t(0));
      draw_short(n);
      return;
    }
    if (holds) {
      if (by_k && n >= k) {
        cut = of_top_k(each);
        cut_ties(each);
      }
      uint64_t total = 0;
      each([&](float x, int i) { total += weight(x, i); });
      total = sum_of(total);
      const int id = select(each, goal_of(total), weight);
      if (tid == 0) put(id, logit<DT>(row[id]), total);
      return;
    }
    if (by_k) {
      cut = of_top_k(over_row);
      cut_ties(over_row);
    }
    __syncthreads();
  }

  // ---- the draw from the groups
  if (!grouped) {
    for (int g = wave; g < groups; g += NW) {
      uint64_t gm = 0;
      over_group(g, [&](float x, int i) { gm += weight(x, i); });
      gm = wave_sum_u64(gm);
      if (lane == 0) group_mass[g] = gm;
    }
    __syncthreads();
  }
  if (wave != 0) return;
  const int per = (groups + 63) / 64;
  uint64_t sum = 0;
  for (int i = 0; i < per; ++i)
    if (lane * per + i < groups) sum += group_mass[lane * per + i];
  const uint64_t run = wave_scan((unsigned long long)sum, lane);
  const uint64_t total = __shfl((unsigned long long)run, 63, 64);
  const uint64_t goal = goal_of(total);
  const int hl = __builtin_ctzll(__ballot(run > goal));
  int g0 = 0;
  uint64_t left = 0;
  if (lane == hl) {
    uint64_t m = run - sum;
    g0 = lane * per;
    while (m + group_mass[g0] <= goal) m += group_mass[g0++];
    left = goal - m;
  }
  g0 = __shfl(g0, hl, 64);
  left = __shfl((unsigned long long)left, hl, 64);
  uint64_t have = 0;
  for (int base = g0 * gs; base < min(g0 * gs + gs, V); base += 64) {
    const int i = base + lane;
    const float x = i < V ? logit<DT>(row[i]) : -__builtin_inff();
    const uint64_t run2 = have + uint64_t(wave_scan((unsigned long long)(i < V ? weight(x, i) : 0), lane));
    const uint64_t hit = __ballot(run2 > left);
    if (hit) {
      if (lane == __builtin_ctzll(hit)) put(i, x, total);
      return;
    }
    have = __shfl((unsigned long long)run2, 63, 64);
  }
}

}  // namespace

hipError_t sample_rows(int dt, const Sampling &p, hipStream_t st) {
  if (p.rows < 1 || p.rows >= 1 << 22 || p.cols < 1) return hipErrorInvalidValue;
  // sums of p.cols weights of at most 2^S stay below 2^63
  int bits = 0;
  while ((int64_t(1) << bits) < p.cols) ++bits;
  const int S = bits <= 19 ? 44 : 63 - bits;
#define MH_SAMPLE(DTV)                                                                                            \
  if (p.cols <= 4096)                                                                                             \
    hipLaunchKernelGGL((sample_kernel<DTV, 256>), dim3(unsigned(p.rows)), dim3(256), 0, st, p, S);                \
  else                                                                                                            \
    hipLaunchKernelGGL((sample_kernel<DTV, 1024>), dim3(unsigned(p.rows)), dim3(1024), 0, st, p, S);
  switch (dt) {
  case F32: MH_SAMPLE(F32) break;
  case F16: MH_SAMPLE(F16) break;
  case BF16: MH_SAMPLE(BF16) break;
  default: return hipErrorInvalidValue;
  }
#undef MH_SAMPLE
  return hipGetLastError();
}

}  // namespace mh
