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

// 2^y for y <= 0 as a whole multiple of 2^-S, and before that rounding (times
// 2^S): 2^y = 2^n e^(f ln 2), |f| <= 1/2, by the exponential's series to the
// twelfth power (the next term is below 2^-52).
struct Weigh {
  double max, per;  // z log2(e) = (x - max) * per
  int S;
  __device__ __forceinline__ double scaled(float x) const {
    if (double(x) == max) return __builtin_ldexp(1.0, S);
    const double y = (double(x) - max) * per;
    if (!(y > -64.0)) return 0.0;
    const double n = __builtin_rint(y), t = (y - n) * 0.69314718055994530942;
    double r = 1.0 / 479001600.0;
    r = fma(r, t, 1.0 / 39916800.0);
    r = fma(r, t, 1.0 / 3628800.0);
    r = fma(r, t, 1.0 / 362880.0);
    r = fma(r, t, 1.0 / 40320.0);
    r = fma(r, t, 1.0 / 5040.0);
    r = fma(r, t, 1.0 / 720.0);
    r = fma(r, t, 1.0 / 120.0);
    r = fma(r, t, 1.0 / 24.0);
    r = fma(r, t, 1.0 / 6.0);
    r = fma(r, t, 0.5);
    r = fma(r, t, 1.0);
    r = fma(r, t, 1.0);
    return __builtin_ldexp(r, int(n) + S);
  }
  static __device__ __forceinline__ uint64_t whole(double v) {
    // (below 2^52: the sum's low bits are the number rounded to nearest)
    return uint64_t(__double_as_longlong(v + 4503599627370496.0)) & ((uint64_t(1) << 52) - 1);
  }
  __device__ __forceinline__ uint64_t operator()(float x) const { return whole(scaled(x)); }
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

// f(logit) over a row, in any order: whole 16-byte chunks where the row's start
// allows it, single values before and after.
template <int DT, int NT, class F> __device__ __forceinline__ void each_value(const typename Store<DT>::T *row, int cols, F f) {
  typedef typename Store<DT>::T T;
  constexpr int E = 16 / sizeof(T);
  const int tid = threadIdx.x;
  const int head = min(int((16 - (uintptr_t(row) & 15)) & 15) / int(sizeof(T)), cols), chunks = (cols - head) / E;
  if (tid < head) f(logit<DT>(row[tid]));
  const uint4 *c = reinterpret_cast<const uint4 *>(row + head);
#pragma unroll 2
  for (int i = tid; i < chunks; i += NT) {
    const uint4 w = c[i];
    float v[E];
    if constexpr (DT == F32) {
      v[0] = __uint_as_float(w.x); v[1] = __uint_as_float(w.y); v[2] = __uint_as_float(w.z); v[3] = __uint_as_float(w.w);
    } else {
      dec8<DT>(w, v);
    }
#pragma unroll
    for (int e = 0; e < E; ++e) f(v[e] == v[e] ? v[e] : -__builtin_inff());
  }
  const int tail = head + chunks * E + tid;
  if (tail < cols) f(logit<DT>(row[tail]));
}

// A prefix of the order: values above K, and the first `ties` equal to it.
struct Cut {
  uint32_t K;
  uint32_t ties;
};

template <int DT, int NT>
__global__ void __launch_bounds__(NT) sample_kernel(Sampling p, int S) {
  typedef typename Store<DT>::T T;
  constexpr int NW = NT / 64;
  __shared__ unsigned long long mass[kBins];
  __shared__ unsigned int count[kBins];
  __shared__ unsigned int red[2][NW];
  __shared__ struct {
    uint32_t bin;
    uint32_t count;  // tokens above the bin
    unsigned long long mass;
  } at;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int r = blockIdx.x, V = p.cols;
  const T *row = static_cast<const T *>(p.logits) + long(r) * p.ld;

  // ---- the largest value
  uint32_t top = 0;
  each_value<DT, NT>(row, V, [&](float x) {
    top = max(top, value_key(x));
  });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) top = max(top, uint32_t(__shfl_xor(top, o, 64)));
  if (lane == 0) red[0][wave] = top;
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
  const float T_ = p.temperature ? p.temperature[r] : 1.f;
  const bool greedy = !(T_ > 0.f);
  const int k = p.top_k ? p.top_k[r] : 0;
  const float tp = p.top_p ? p.top_p[r] : 1.f, mp = p.min_p ? p.min_p[r] : 0.f;
  Weigh w;
  w.max = double(xmax);
  w.per = greedy ? 0.0 : 1.4426950408889634074 / double(T_);
  w.S = S;

  // ---- the prefix
  Cut cut{0u, 0xffffffffu};
  if (greedy) {
    cut = Cut{top, 1u};
  } else if ((k > 0 && k < V) || tp < 1.f) {
    // bins of equal width in z over the S bits that weigh anything
    const float per_bin = float(kBins) / float(S + 1), slope = fminf(float(w.per) * per_bin, 1e30f);
    auto bin_of = [&](float x) -> uint32_t {
      return x == xmax ? 0u : uint32_t(fminf((xmax - x) * slope, float(kBins - 1)));
    };
    // bins of the tokens that `in` takes, and where a prefix of `n` tokens or of
    // weight `goal` ends: the bin, and what lies above it
    auto fill = [&](auto in, auto where) {
      for (int i = tid; i < kBins; i += NT) {
        mass[i] = 0;
        count[i] = 0;
      }
      __syncthreads();
      each_value<DT, NT>(row, V, [&](float x) {
        if (in(x)) {
          const uint32_t b = where(x);
          atomicAdd(&count[b], 1u);
          const uint64_t m = w(x);
          if (m) atomicAdd(&mass[b], (unsigned long long)m);
        }
      });
      __syncthreads();
    };
    auto find = [&](bool by_mass, uint64_t goal) {
      if (wave == 0) {
        constexpr int per = kBins / 64;
        uint64_t m = 0;
        uint32_t c = 0;
        for (int i = 0; i < per; ++i) {
          m += mass[lane * per + i];
          c += count[lane * per + i];
        }
        const uint64_t ms = wave_scan((unsigned long long)m, lane);
        const uint32_t cs = wave_scan(c, lane);
        const bool hit = (by_mass ? ms : uint64_t(cs)) >= goal;
        const uint64_t hits = __ballot(hit);
        const int l = hits ? __builtin_ctzll(hits) : 63;
        if (lane == l) {
          uint64_t am = ms - m;
          uint32_t ac = cs - c;
          int b = lane * per;
          for (int i = 0; i + 1 < per; ++i) {
            if ((by_mass ? am + mass[b] : uint64_t(ac) + count[b]) >= goal) break;
            am += mass[b];
            ac += count[b];
            ++b;
          }
          at.bin = b;
          at.count = ac;
          at.mass = am;
        }
      }
      __syncthreads();
    };
    // the exact end of a prefix of `goal` tokens or weight
    auto end_of = [&](bool by_mass, uint64_t goal, uint64_t &above_mass) -> Cut {
      find(by_mass, goal);
      const uint32_t b0 = at.bin;
      uint64_t am = at.mass;
      uint64_t ac = at.count;
      // the keys of that bin
      uint32_t lo = 0xffffffffu, hi = 0;
      each_value<DT, NT>(row, V, [&](float x) {
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
        fill([&](float x) { const uint32_t kk = value_key(x); return bin_of(x) == b0 && kk >= lo && kk <= hi; },
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
    fill([&](float) { return true; }, bin_of);
    uint64_t total = 0;  // the weight that top-k leaves
    if (k > 0 && k < V) {
      uint64_t above = 0;
      cut = end_of(false, uint64_t(k), above);
      total = above + uint64_t(cut.ties) * w(key_value(cut.K));
      if (tp < 1.f) fill([&](float) { return true; }, bin_of);
    } else {
      if (wave == 0) {
        uint64_t m = 0;
        for (int i = lane; i < kBins; i += 64) m += mass[i];
        m = wave_sum_u64(m);
        if (lane == 0) at.mass = m;
      }
      __syncthreads();
      total = at.mass;
      __syncthreads();
    }
    if (tp < 1.f) {
      const double g = __builtin_ceil(double(fmaxf(tp, 0.f)) * double(total));
      const uint64_t goal = g < 1.0 ? 1 : min(uint64_t(g), total);
      uint64_t above = 0;
      const Cut c = end_of(true, goal, above);
      if (c.K > cut.K || (c.K == cut.K && c.ties < cut.ties)) cut = c;
    }
  }
  // min-p: a weight below this (times 2^S) is dropped
  const double least = mp > 0.f && !greedy ? double(fminf(mp, 1.f)) * __builtin_ldexp(1.0, S) : 0.0;

  // ---- kept weight and ties of each group of consecutive tokens
  __syncthreads();
  int gs = 512;
  while ((V + gs - 1) / gs > kMaxGroups) gs *= 2;
  const int groups = (V + gs - 1) / gs;
  // (mass / count are reused: kMaxGroups <= kBins)
  auto kept = [&](float x, uint64_t &m) -> int {  // 0 no, 1 above the threshold, 2 equal to it
    m = 0;
    const uint32_t kk = value_key(x);
    if (kk < cut.K) return 0;
    const double s = w.scaled(x);
    if (s < least) return 0;
    m = Weigh::whole(s);
    return kk > cut.K ? 1 : 2;
  };
  for (int g = wave; g < groups; g += NW) {
    uint64_t m = 0;
    uint32_t ties = 0;
    const int end = min(g * gs + gs, V);
#pragma unroll 4
    for (int i = g * gs + lane; i < end; i += 64) {
      uint64_t one;
      const int how = kept(logit<DT>(row[i]), one);
      if (how == 1) m += one;
      if (how == 2) ++ties;
    }
    m = wave_sum_u64(m);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ties += __shfl_xor(ties, o, 64);
    if (lane == 0) {
      mass[g] = m;
      count[g] = ties;
    }
  }
  __syncthreads();
  if (wave != 0) return;

  // ---- the draw (one wave)
  const uint64_t tie_weight = w(key_value(cut.K));  // (unused where nothing ties)
  const int per = (groups + 63) / 64;
  uint32_t my_ties = 0;
  for (int i = 0; i < per; ++i)
    if (lane * per + i < groups) my_ties += count[lane * per + i];
  uint64_t before = uint64_t(wave_scan((unsigned long long)my_ties, lane)) - my_ties;
  uint64_t sum = 0, left_ties = before;
  for (int i = 0; i < per; ++i) {
    const int g = lane * per + i;
    if (g >= groups) break;
    const uint64_t left = left_ties < cut.ties ? cut.ties - left_ties : 0, n = min(left, uint64_t(count[g]));
    left_ties += count[g];
    mass[g] += n * tie_weight;
    sum += mass[g];
  }
  const uint64_t run = wave_scan((unsigned long long)sum, lane);
  const uint64_t total = __shfl((unsigned long long)run, 63, 64);
  float u = p.u[r];
  u = u > 0.f ? u : 0.f;
  uint64_t goal = uint64_t(double(u) * double(total));
  if (goal >= total) goal = total - 1;  // u = 1: the last kept token
  const int hl = __builtin_ctzll(__ballot(run > goal));
  int g0 = 0;
  uint64_t g_goal = 0, g_ties = 0;
  if (lane == hl) {
    uint64_t m = run - sum;
    uint64_t ties = before;
    g0 = lane * per;
    while (m + mass[g0] <= goal) {
      m += mass[g0];
      ties += count[g0];
      ++g0;
    }
    g_goal = goal - m;
    g_ties = ties;
  }
  g0 = __shfl(g0, hl, 64);
  g_goal = __shfl((unsigned long long)g_goal, hl, 64);
  g_ties = __shfl((unsigned long long)g_ties, hl, 64);
  uint64_t have = 0, ties = g_ties;
  for (int base = g0 * gs; base < min(g0 * gs + gs, V); base += 64) {
    const int i = base + lane;
    uint64_t one = 0;
    int how = 0;
    float x = 0.f;
    if (i < V) {
      x = logit<DT>(row[i]);
      how = kept(x, one);
    }
    const uint64_t tied = __ballot(how == 2);
    if (how == 2 && ties + __builtin_popcountll(tied & ((uint64_t(1) << lane) - 1)) >= cut.ties) one = 0;
    ties += __builtin_popcountll(tied);
    const uint64_t run2 = have + uint64_t(wave_scan((unsigned long long)one, lane));
    const uint64_t hit = __ballot(run2 > g_goal);
    if (hit) {
      if (lane == __builtin_ctzll(hit)) {
        p.ids[r] = i;
        // log(w / sum) from the logit itself: the whole weight has few bits where w is small
        if (p.logprob)
          p.logprob[r] = greedy ? 0.f
                                : float((double(x) == w.max ? 0.0 : (double(x) - w.max) / double(T_)) -
                                        log(double(total) * __builtin_ldexp(1.0, -S)));
      }
      return;
    }
    have = __shfl((unsigned long long)run2, 63, 64);
  }
}

}  // namespace

hipError_t sample_rows(int dt, const Sampling &p, hipStream_t st) {
  if (p.rows < 1 || p.cols < 1) return hipErrorInvalidValue;
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
