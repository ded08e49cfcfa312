// Attention over the paged 8-bit KV cache (paged_index.hpp) for ragged batches:
// single tokens, whole prompts, and chunks of prompts behind a cached prefix.
//
// Row r = (query i, head h) of sequence b at position p = len - n + i:
//   o = sum_j w_j v_j / sum_j w_j,  w_j = 2^(c q.k_j - m),  c = scale log2(e),
// over the keys j that the row sees (j <= p if causal, j > p - window if a
// window is set); a row that sees none is zero.
//
// The rows of one key/value head are packed: its group of query heads times the
// sequence's queries are the columns of 16-wide MFMA tiles, so that a single
// token of 8 grouped heads costs what one head costs, and the cache is read once
// per key/value head.
//
// Everything stays in registers.  For a block of 64 keys a wave computes
// S^T = K Q^T as four 16 x 16 tiles; row m = 4 a + r of tile t is key
// 16 a + 4 t + r, so that lane group g (the lanes 16 g .. 16 g + 15) ends with
// the scores of the 16 consecutive keys 16 g .. 16 g + 15 of query column
// lane & 15: exactly the k-operand order in which O^T = V^T P^T takes them
// (two steps of 8 keys per lane), and exactly one 16-byte run of the transposed
// values.  A page holds at least 16 tokens, so a lane group's keys lie in one
// page and take one key scale and one value scale.
//
// Precision: e4m3 converts to fp16 exactly.  A row of q is scaled by a power of
// two to below 2^14 and is then exact in fp16 for bf16 and fp16 inputs (but for at
// most 2^-38 of the row's largest value); fp32 inputs are the sum of two fp16 parts
// (22 bits and a sign).  Scores, the running maximum, the sum and the outputs are
// fp32.  A probability enters the second product as 2^9 w times its page's value
// scale over the row's largest product of the two so far (a reference near it),
// rounded to fp16 (half a unit of 11 bits down to 2^-23 of that; outputs of 16 bits
// are rounded as much once more), or as two such parts for fp32 inputs.
#include "mh_common.hpp"
#include "mh_kernels.hpp"
#include "paged_index.hpp"

namespace mh {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

// Probabilities times value scales are taken times 2^kLift, against a reference that
// the row's largest passes by at most kRaise (log2): below 2^15 in fp16.
constexpr float kLift = 9.f, kRaise = 5.f;
// The references: mx of the scores (log2), to which the sum goes, and mx + lref of
// scores + log2 of value scales, to which the outputs go; lref is a whole number, so
// that powers of two alone lie between the two.  The first moves when a score
// passes it by kRaise, the second then too or when a product passes it: sums and
// outputs are seldom scaled.  (Against the largest value scale alone, outputs of
// small values went lost beside large ones of no weight.)
__device__ __forceinline__ bool passes(float top, float both, float &mx, float &lref, float &down, float &down_both) {
  const float m = top > mx + kRaise ? top : mx;
  const bool moved = m != mx || both > mx + lref + kRaise;
  down = down_both = 1.f;
  if (moved) {
    const float by = mx - m, l = __builtin_ceilf(fmaxf(mx + lref, both) - m);
    down = __builtin_amdgcn_exp2f(by);
    down_both = __builtin_amdgcn_exp2f(by + (lref - l));
    mx = m;
    lref = l;
  }
  return moved;
}
// A run's value scale over lref, to what the probabilities can take: at least 2^-60,
// where they are zeros in fp16, since the sum goes by them times the inverse, which has
// to stay a float (a page of zeros has scale 2^-100); and for two parts, which
// are scaled after the exponential, at most 2^110.
template <int NP> __device__ __forceinline__ float apart(float lv, float lref) {
  return __builtin_amdgcn_fmed3f(lv - lref, -60.f, NP == 2 ? 110.f : 250.f);
}

struct PagedArgs {
  const void *q;
  void *out;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  const int32_t *tables, *lens, *cu;
  float *part_o;
  float2 *part_ml;
  int *err;
  long ldq, ldo;
  int B, Hq, Hkv, G, hd, plog, n_pages, n_rows, width, causal, window, splits, chunk, tiles;
  float c;  // scale * log2(e)
};

// Barrier that waits for this wave's LDS operations and not for its loads from
// memory.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A table that the launch does not change, for loads into scalar registers at
// scalar indexes.
typedef const __attribute__((address_space(4))) int32_t *ScalarTable;
__device__ __forceinline__ ScalarTable scalar_ptr(const int32_t *p) { return (ScalarTable)(uintptr_t)p; }

// 8 e4m3 bytes -> 8 fp16 values, exact
__device__ __forceinline__ f16x8 cvt8(uint32_t lo, uint32_t hi) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return f16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// bytes [a, b) of a 16-byte chunk kept, the others zero
__device__ __forceinline__ uint4 keep_bytes(uint4 v, int a, int b) {
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int lo = min(max(a - 4 * i, 0), 4), hi = min(max(b - 4 * i, 0), 4);
    const uint32_t below_hi = hi >= 4 ? 0xffffffffu : (1u << (8 * hi)) - 1u;
    const uint32_t below_lo = lo >= 4 ? 0xffffffffu : (1u << (8 * lo)) - 1u;
    w[i] &= below_hi & ~below_lo;
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// 0x01 in every byte of w that holds an e4m3 NaN (0x7f or 0xff)
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t x = (w & 0x7f7f7f7fu) + 0x01010101u;  // 0x80 where the magnitude is 0x7f
  return (x >> 7) & 0x01010101u;
}

__device__ __forceinline__ float finite_max8(const float v[8], float big) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float m = __builtin_fabsf(v[e]);
    big = m < __builtin_inff() ? fmaxf(big, m) : big;
  }
  return big;
}
// 2^k: 2^k times a row of this largest magnitude lies below 2^14
__device__ __forceinline__ float row_lift(float big) {
  const int ex = int(__float_as_uint(big) >> 23);  // biased exponent, 0 for zero and subnormal rows
  const int k = ex == 0 ? 0 : min(13 - (ex - 127), 120);
  return __uint_as_float(uint32_t(k + 127) << 23);
}

// 1 / a row's sum; 0 where it saw no key
__device__ __forceinline__ float over(float sum) { return sum == 0.f ? 0.f : 1.f / sum; }

// The query rows of a wave: NQ tiles of 16 (column n of tile x is row r_first + 16 x
// + n of the packed rows; past the last row, that row again, not stored), their
// running softmax and their outputs O^T.
template <int DT, int HDP, int NQ> struct RowTiles {
  typedef typename Store<DT>::T T;
  static constexpr int NP = DT == F32 ? 2 : 1;  // fp16 parts of q and of the probabilities
  static constexpr int KS = HDP / 32, MT = HDP / 16, RW = 16 * NQ;
  f16x8 qf[NP][NQ][KS];
  f16x8 pf[NP][NQ][2];
  f32x4 acc[MT][NQ];
  float c_row[NQ], mx[NQ], l[NQ];
  float lref[NQ];  // outputs are in units of 2^lref
  int lo_row[NQ], hi_row[NQ];
  int every_lo, every_hi;  // keys that every row sees
  int some_lo, some_hi;    // keys that some row sees

  // head values d_of(s) .. + 7 are the operand of step s
  template <class D>
  __device__ __forceinline__ void start(const PagedArgs &a, int row0, int nq, int len, int rows, int r_first, int kvh, int n,
                                        KeyRange mine, D d_of) {
    const int i0 = r_first / a.G, i1 = (min(r_first + RW, rows) - 1) / a.G;
    const KeyRange all = seen_keys(len, nq, i0, i1, a.causal, a.window);
    every_lo = max(seen_keys(len, nq, i1, i1, a.causal, a.window).lo, mine.lo);
    every_hi = min(seen_keys(len, nq, i0, i0, a.causal, a.window).hi, mine.hi);
    some_lo = max(all.lo, mine.lo);
    some_hi = min(all.hi, mine.hi);
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int r = min(r_first + 16 * x + n, rows - 1), i = r / a.G, h = kvh * a.G + r - i * a.G;
      const T *qp = static_cast<const T *>(a.q) + long(row0 + i) * a.ldq + long(h) * a.hd;
      float v[KS][8], big = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = d_of(s);
        if (d < a.hd) {
          if constexpr (DT == F32) {
            ld4<F32>(qp + d, v[s]);
            ld4<F32>(qp + d + 4, v[s] + 4);
          } else {
            dec8<DT>(*reinterpret_cast<const uint4 *>(qp + d), v[s]);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[s][e] = 0.f;
        }
        big = finite_max8(v[s], big);
      }
      const float lift = row_lift(xor32_max(xor16_max(big))), up = __builtin_copysignf(lift, a.c);
      c_row[x] = __builtin_fabsf(a.c) / lift;  // (a power of two; the scale's sign is q's)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float w = v[s][e] * up;
          const _Float16 h0 = _Float16(w);
          qf[0][x][s][e] = h0;
          if constexpr (NP == 2) qf[1][x][s][e] = _Float16(w - float(h0));
        }
      }
      const KeyRange kr = seen_keys(len, nq, i, i, a.causal, a.window);
      lo_row[x] = max(kr.lo, mine.lo);
      hi_row[x] = min(kr.hi, mine.hi);
      mx[x] = -__builtin_inff();
      l[x] = 0.f;
      lref[x] = -126.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][x] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
  }

  // Raw scores of a block (this lane group's keys tv .. tv + 15, with their
  // page's key scale and log2 of its value scale) to probabilities pf; the sums and
  // outputs so far scaled to the new references.
  // masked: some row does not see some key.
  __device__ __forceinline__ void probabilities(f32x4 (&s)[4][NQ], float ksc, float lv, bool page_ok, int tv, bool masked) {
    float ks[NQ];
#pragma unroll
    for (int x = 0; x < NQ; ++x) ks[x] = ksc;
    if (masked) {
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        const uint32_t ok = seen(x, tv, page_ok);
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[t][x][r] = (ok >> (4 * t + r)) & 1u ? s[t][x][r] : -__builtin_inff();
        // a page of which the row sees nothing may have anything as scales
        ks[x] = ok ? ksc : 1.f;
      }
    }
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      // (c_row and a page's scale are positive: the largest raw score is the largest score)
      float f = ks[x] * c_row[x];
      f = f == 0.f ? 1e-37f : f;  // (so that a masked score stays -inf)
      float top = s[0][x][0];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][x][r]);
      const bool none = !(top > -__builtin_inff());
      top = none ? -__builtin_inff() : top * f;
      const float both = xor32_max(xor16_max(none ? top : top + lv));
      top = xor32_max(xor16_max(top));
      float down, down_both;
      if (__any(passes(top, both, mx[x], lref[x], down, down_both))) {
        l[x] *= down;
#pragma unroll
        for (int i = 0; i < MT; ++i) acc[i][x] *= down_both;
      }
      float ref = mx[x] > -__builtin_inff() ? mx[x] : 0.f;
      const float lf = apart<NP>(lv, lref[x]);
      const float unscale = __builtin_amdgcn_exp2f(-lf), lift = __builtin_amdgcn_exp2f(lf + kLift);
      // The product below is not rounded before the maximum, which is, goes off it.
      // Where that could leave much (scores past 2^16), both are rounded.
      const bool far = __builtin_fabsf(ref) > 65536.f;
      if (__any(far)) {
#pragma clang fp contract(off)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) s[t][x][r] = far ? s[t][x][r] * f - ref : s[t][x][r];
        f = far ? 1.f : f;
        ref = far ? 0.f : ref;
      }
      float sum = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float p[2];
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float raw = s[2 * u + (e >> 2)][x][(e & 3) + y];
            // fp32: the difference from the maximum is rounded once, and the
            // power of two applied to the result
            p[y] = __builtin_amdgcn_exp2f(NP == 2 ? fmaf(raw, f, -ref) : fmaf(raw, f, lf + kLift - ref));
            if constexpr (NP == 2) p[y] *= lift;
            // (not of the rounded values: those of small weights and value scales are
            // zero)
            sum += p[y];
          }
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const _Float16 h0 = _Float16(p[y]);
            pf[0][x][u][e + y] = h0;
            if constexpr (NP == 2) pf[1][x][u][e + y] = _Float16(p[y] - float(h0));
          }
        }
      l[x] = fmaf(sum, unscale, l[x]);  // (2^kLift w)
    }
  }

  // bit e: row x sees key tv + e
  __device__ __forceinline__ uint32_t seen(int x, int tv, bool page_ok) const {
    const int lo = min(max(lo_row[x] - tv, 0), 16), hi = min(max(hi_row[x] - tv, 0), 16);
    return page_ok ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
  }

  // O^T += V^T P^T for head rows 16 i .. 16 i + 15
  __device__ __forceinline__ void values(int i, f16x8 v0, f16x8 v1) {
#pragma unroll
    for (int x = 0; x < NQ; ++x)
#pragma unroll
      for (int p = NP - 1; p >= 0; --p) {
        acc[i][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[p][x][0], acc[i][x], 0, 0, 0);
        acc[i][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[p][x][1], acc[i][x], 0, 0, 0);
      }
  }

  // A NaN value that only some rows see must reach these alone, which a zero
  // probability does not give: outputs of rows that see a marked value (m0, m1:
  // 1 at a NaN value, 0 else) become NaN.
  __device__ __forceinline__ void mark_nans(int i, f16x8 m0, f16x8 m1, int tv, bool page_ok) {
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      f16x8 s0, s1;
      const uint32_t ok = seen(x, tv, page_ok);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        s0[e] = (ok >> e) & 1u ? _Float16(1.f) : _Float16(0.f);
        s1[e] = (ok >> (8 + e)) & 1u ? _Float16(1.f) : _Float16(0.f);
      }
      f32x4 hit = f32x4{0.f, 0.f, 0.f, 0.f};
      hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(m0, s0, hit, 0, 0, 0);
      hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(m1, s1, hit, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (hit[r] > 0.f) acc[i][x][r] = __builtin_nanf("");
    }
  }

  // The sums over the lane groups, the outputs over them (zero where no key was seen)
  // and in the values' scale, in this order: an output is no larger than the
  // largest value, its product with the sum may pass a float.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      l[x] = xor32_add(xor16_add(l[x]));
      const float inv = over(l[x]), up = __builtin_amdgcn_exp2f(lref[x]);
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][x] = acc[i][x] * inv * up;
    }
  }
};

// Where a packed row's output goes: to the caller, or with the share's maximum and
// sum to the join.
template <int DT> struct RowOut {
  typedef typename Store<DT>::T T;
  T *out;
  float *part;
  __device__ __forceinline__ RowOut(const PagedArgs &a, int row0, int kvh, int split, int r, float m, float sum, bool first) {
    const int i = r / a.G, h = kvh * a.G + r - i * a.G;
    out = nullptr;
    part = nullptr;
    if (a.splits == 1) {
      out = static_cast<T *>(a.out) + long(row0 + i) * a.ldo + long(h) * a.hd;
    } else {
      const long at = ((long(row0) + i) * a.Hq + h) * a.splits + split;
      if (first) a.part_ml[at] = make_float2(m, sum);
      if (!(sum == 0.f)) part = a.part_o + at * a.hd;  // (the join skips empty shares)
    }
  }
  __device__ __forceinline__ void put(int d, f32x4 o) const {
    if (out) {
      const float v[4] = {o[0], o[1], o[2], o[3]};
      st4<DT>(out + d, v);
    } else if (part) {
      *reinterpret_cast<f32x4 *>(part + d) = o;
    }
  }
};

// The part of a call that a workgroup is: request, its rows and keys (cut to the
// table and the buffer).
struct Part {
  int split, kvh, b, len, row0, nq, rows;
};
__device__ __forceinline__ bool part_of(const PagedArgs &a, int b, int kvh, Part &w) {
  w.kvh = kvh;
  w.b = b;
  const auto lens = scalar_ptr(a.lens), cu = scalar_ptr(a.cu);
  const int most = a.width << a.plog, len = lens[w.b];
  w.len = min(max(len, 0), most);
  w.row0 = cu[w.b];
  w.nq = min(cu[w.b + 1], a.n_rows) - w.row0;
  if (w.row0 < 0 || w.nq <= 0) return false;
  if (len > most && threadIdx.x == 0) atomicOr(a.err, kErrPage);
  w.rows = w.nq * a.G;
  return true;
}

// Few rows (a decode step): the four waves take the same 16 rows and every fourth
// block of the keys each.  Keys and values go from memory straight into the
// MFMA operands.
template <int DT, int HDP>
__global__ void __launch_bounds__(256) attn_paged_kernel(PagedArgs a) {
  constexpr int J = HDP / 64, MT = HDP / 16, RW = 16;
  // (the wave's number as a scalar: what follows from it are scalar tests)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 15, g = lane >> 4;
  Part w;
  // The heads of a page lie together: the workgroups that read them follow each
  // other on an XCD.
  const PairItem it = pair_item(blockIdx.x, a.B * a.splits * a.tiles, a.Hkv);
  w.split = it.pair / a.tiles % a.splits;
  if (!part_of(a, it.pair / a.tiles / a.splits, it.item, w)) return;
  const int P = 1 << a.plog;
  const int32_t *table = a.tables + long(w.b) * a.width;
  const uint8_t *kc = a.kc + page_base(0, a.Hkv, w.kvh, P, a.hd), *vc = a.vc + page_base(0, a.Hkv, w.kvh, P, a.hd);
  const int64_t stride = page_base(1, a.Hkv, 0, P, a.hd);
  // The merge of the four waves' shares: 128 head values at a time.
  constexpr int MW = HDP < 128 ? HDP : 128, LD = MW + 4;
  __shared__ __align__(16) float wo[4][RW][LD];
  __shared__ float2 wml[4][RW];

  // (more tiles than the launch was sized for are walked)
  for (int tile = it.pair % a.tiles; long(tile) * RW < w.rows; tile += a.tiles) {
    const int r_first = tile * RW;
    const int i0 = r_first / a.G, i1 = (min(r_first + RW, w.rows) - 1) / a.G;
    const KeyRange mine = key_share(seen_keys(w.len, w.nq, i0, i1, a.causal, a.window), w.split, a.splits, a.chunk);
    // A block's keys are on their way while the probabilities and values of the block
    // before are worked on, its values during its scores: they take the registers
    // that those have left.  Every load is made, at an address that exists, and
    // what should not count is masked: a load under a condition makes the compiler
    // wait for it before the next.  Keys past the range take its last page; a page
    // outside the pool holds no keys (page 0 is read); head values past hd repeat
    // earlier ones (their queries are zero, their outputs not stored).
    // The pages come by scalar loads, a block ahead: a vector load's result is waited
    // for together with all loads before it, here the block's bytes.
    const auto table_s = scalar_ptr(table);
    const int last = __builtin_amdgcn_readfirstlane(mine.hi) - 1;
    int page0 = 0, page1 = 0, page2 = 0, page3 = 0;  // of the block's runs of 16 keys
    int pv = 0;                                      // of this lane's scores and values (run g)
    bool next_ok = false;
    int missing = -1;  // last key of a run whose page is outside the pool
    uint4 kr[4][J], vr[MT];
    float ksc = 0.f, vsc = 0.f;
    auto pages = [&](int base) {
      page0 = table_s[min(base, last) >> a.plog];
      page1 = table_s[min(base + 16, last) >> a.plog];
      page2 = table_s[min(base + 32, last) >> a.plog];
      page3 = table_s[min(base + 48, last) >> a.plog];
    };
    auto of_run = [&](int c) {
      const int lo = c & 1 ? page1 : page0, hi = c & 1 ? page3 : page2;
      return c & 2 ? hi : lo;
    };
    auto load_keys = [&](int base) {
      const int tk = base + 16 * (n >> 2), tv = base + 16 * g;
      int pk = of_run(n >> 2);  // of this lane's key rows
      pv = of_run(g);
      next_ok = page_in_pool(pv, a.n_pages);
      missing = max(missing, next_ok || tv >= mine.hi ? -1 : tv + 15);
      pk = page_in_pool(pk, a.n_pages) ? pk : 0;
      pv = next_ok ? pv : 0;
      const uint8_t *kp = kc + pk * stride + (tk & (P - 1)) * a.hd;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < J; ++j)
          kr[t][j] = *reinterpret_cast<const uint4 *>(kp + (4 * t + (n & 3)) * a.hd + min(64 * j + 16 * g, a.hd - 16));
      ksc = a.ks[long(pv) * a.Hkv + w.kvh];
      vsc = a.vs[long(pv) * a.Hkv + w.kvh];
    };
    auto load_values = [&](int base) {
      const uint8_t *vp = vc + pv * stride + ((base + 16 * g) & (P - 1)) + n * P;
#pragma unroll
      for (int i = 0; i < MT; ++i) vr[i] = *reinterpret_cast<const uint4 *>(vp + min(16 * i, a.hd - 16) * P);
    };
    int base = (mine.lo & ~(kKeyBlock - 1)) + wave * kKeyBlock;
    // (the last block's successor is itself: its bytes are in the caches)
    auto after = [&](int b) { return b + 4 * kKeyBlock < mine.hi ? b + 4 * kKeyBlock : b; };
    if (base < mine.hi) {
      pages(base);
      load_keys(base);
      load_values(base);
      pages(after(base));
    }
    // (the queries' loads after the first block's: all of them are waited for at once)
    RowTiles<DT, HDP, 1> q;
    // (the order of the head values in a step is that of the 16-byte runs in which
    // a lane loads its keys)
    q.start(a, w.row0, w.nq, w.len, w.rows, r_first, w.kvh, n, mine, [&](int s) { return 64 * (s >> 1) + 16 * g + 8 * (s & 1); });
    while (base < mine.hi) {
      const int next = base + 4 * kKeyBlock, then = after(base), tv = base + 16 * g;
      const bool page_ok = next_ok;
      const float lv = page_ok ? fmaxf(__builtin_amdgcn_logf(vsc), -126.f) : -126.f, kscale = ksc;
      f32x4 s[4][1];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        s[t][0] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const f16x8 k0 = cvt8(kr[t][j].x, kr[t][j].y), k1 = cvt8(kr[t][j].z, kr[t][j].w);
#pragma unroll
          for (int p = q.NP - 1; p >= 0; --p) {
            s[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, q.qf[p][0][2 * j], s[t][0], 0, 0, 0);
            s[t][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, q.qf[p][0][2 * j + 1], s[t][0], 0, 0, 0);
          }
        }
      }
      load_keys(then);
      pages(after(then));
      __builtin_amdgcn_sched_barrier(0);
      const bool masked = base < q.every_lo || base + kKeyBlock > q.every_hi || __any(!page_ok);
      q.probabilities(s, kscale, lv, page_ok, tv, masked);

      // Keys that no row sees may hold anything, NaN among it: their bytes are
      // cleared.
      bool nans = false;
      if (masked) {
        const int lo = min(max(q.some_lo - tv, 0), 16), hi = page_ok ? min(max(q.some_hi - tv, 0), 16) : 0;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          vr[i] = keep_bytes(vr[i], lo, hi);
          any |= nan_bytes(vr[i].x) | nan_bytes(vr[i].y) | nan_bytes(vr[i].z) | nan_bytes(vr[i].w);
        }
        nans = __any(any != 0);
      }
      if (nans) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          uint32_t b[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w}, mark[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t nb = nan_bytes(b[c]);
            b[c] &= ~(nb * 0xffu);
            mark[c] = nb * 0x38u;  // e4m3 1.0
          }
          vr[i] = make_uint4(b[0], b[1], b[2], b[3]);
          q.mark_nans(i, cvt8(mark[0], mark[1]), cvt8(mark[2], mark[3]), tv, page_ok);
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) q.values(i, cvt8(vr[i].x, vr[i].y), cvt8(vr[i].z, vr[i].w));
      base = next;
      if (base < mine.hi) load_values(base);
    }
    // (told here: in the loop it took 67 scalars spilled instead of 38, 16.4 us for 15.4 in
    // 24 windows of 1000 keys, fp32; pages behind the window may be gone)
    if (missing >= q.some_lo) atomicOr(a.err, kErrPage);
    q.finish();

    // the four waves' shares of the keys, in wave order
    if (g == 0) wml[wave][n] = make_float2(q.mx[0], q.l[0]);
#pragma unroll
    for (int part = 0; part < HDP / MW; ++part) {
#pragma unroll
      for (int i = 0; i < MW / 16; ++i) *reinterpret_cast<f32x4 *>(&wo[wave][n][16 * i + 4 * g]) = q.acc[part * (MW / 16) + i][0];
      lds_barrier();  // (not for the loads of the block after the last)
      for (int e = tid; e < RW * (MW / 4); e += 256) {
        const int rr = e / (MW / 4), d = 4 * (e % (MW / 4)), r = r_first + rr;
        if (r < w.rows && part * MW + d < a.hd) {
          float top = wml[0][rr].x;
#pragma unroll
          for (int v = 1; v < 4; ++v) top = fmaxf(top, wml[v][rr].x);
          f32x4 y[4];
          float2 ml[4];  // (sum 0: this wave saw no key)
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            ml[v] = wml[v][rr];
            y[v] = *reinterpret_cast<const f32x4 *>(&wo[v][rr][d]);
          }
          float sum = 0.f;
#pragma unroll
          for (int v = 0; v < 4; ++v) {
            ml[v].y = ml[v].y == 0.f ? 0.f : ml[v].y * __builtin_amdgcn_exp2f(ml[v].x - top);
            sum += ml[v].y;
          }
          const float inv = over(sum);
          f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] = fmaf(y[v][c], ml[v].y * inv, o[c]);
          const int at = part * MW + d;
          RowOut<DT>(a, w.row0, w.kvh, w.split, r, top, sum, at == 0).put(at, o);
        }
      }
      lds_barrier();
    }
  }
}

// Many rows (prompts): 32 to a wave, on 32 x 32 MFMA tiles, four waves to a
// workgroup, which share every block of 64 keys.  The workgroup converts a block to
// fp16 once, into LDS (two buffers: the next block's bytes are on their way while
// this one is multiplied), from where each wave reads its operands.
// As above, the scores' tiles S^T = K Q^T end in the operand order of O^T = V^T P^T:
// key 16 h + i of a tile of 32 is its row 8 (i / 4) + 4 h + i % 4, so that lane half
// h holds the scores of the 16 consecutive keys 16 h .. 16 h + 15 of its column.
// LDS rows are swizzled in 16-byte chunks so that 16 lanes that read the same chunk
// of 16 rows find them in different banks: chunk c of a row of 256 bytes or more
// lies at c ^ (row & 15), of 128 bytes (values: a head value's 64 keys) at c ^
// (row / 2 & 7).
// ONE: pages of 64 tokens or more, where a block lies in one: one page number, two
// addresses and two scales, scalars that each wave has.  With smaller pages the first
// wave puts the runs' scales into LDS for the others, who wait for it (6 chunks
// of 6700 tokens in all that end at 1200 to 8000 keys, 32 heads on 8 of 128, pages of
// 64: 520 us a pass so, 452 with ONE).
// Registers bound the waves: 64 outputs, 32 of q and 32 scores a lane at hd 128
// leave two waves to a SIMD, with 11 to 21 of 256 spilled; fp32 and heads above 128
// take all registers for one.
template <int DT, int HDP, bool ONE>
__global__ void __launch_bounds__(256, DT == F32 || HDP > 128 ? 1 : 2) attn_paged_wide_kernel(PagedArgs a) {
  typedef typename Store<DT>::T T;
  constexpr int NT = 256, NW = 4, RW = 32, RB = NW * RW;
  constexpr int NP = DT == F32 ? 2 : 1;          // fp16 parts of q and of the probabilities
  constexpr int KS = HDP / 16, MT = HDP / 32;
  constexpr int XK = HDP / 16;                   // 16-byte pieces of a key in the cache
  constexpr int NK = 64 * XK, CH = 2 * NK / NT;  // pieces of a block's keys; pieces (keys and values) per thread
  constexpr int KROW = HDP * 2, KB = 64 * KROW, VB = HDP * 128;
  __shared__ __align__(16) uint8_t lds[2][KB + VB];
  // per 16 keys: key scale, log2 of the value scale, page in the pool
  __shared__ float4 info[2][4];
  // NaN values of a block at the edge of some row's mask (they are zeros in
  // LDS): bit k of nan_at, key k of the block
  __shared__ uint64_t nan_at[2][HDP];
  // the runs of 16 keys (bits 0..3) of which a wave noted some: a wave without a missing page
  // notes nothing in blocks that all rows see, and what nan_at has of its runs is old
  __shared__ uint32_t dirty[2][NW];
  // (the wave's number as a scalar: what follows from it are scalar tests)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, h = lane >> 5;
  Part w;
  const PairItem it = pair_item(blockIdx.x, a.B * a.Hkv, a.tiles * a.splits);
  w.split = it.item % a.splits;
  int b = it.pair / a.Hkv;
  if (a.B <= NT && a.B > 1) {
    // Requests from the longest to the shortest, so that none of the long ones is left
    // for the end (6 requests of 1200 to 8000 keys: the last workgroup ends 3 %
    // past the mean instead of 6 to 33 %)
    __shared__ int lens[NT], found;
    const int mine = tid < a.B ? a.lens[tid] : 0;
    lens[tid] = mine;
    __syncthreads();
    int rank = 0;
    for (int v = 0; v < a.B; ++v) rank += lens[v] > mine || (lens[v] == mine && v < tid);
    if (tid < a.B && rank == b) found = tid;
    __syncthreads();
    b = __builtin_amdgcn_readfirstlane(found);
  }
  if (!part_of(a, b, it.pair % a.Hkv, w)) return;
  const int P = 1 << a.plog;
  const int32_t *table = a.tables + long(w.b) * a.width;
  const uint8_t *kc = a.kc + page_base(0, a.Hkv, w.kvh, P, a.hd), *vc = a.vc + page_base(0, a.Hkv, w.kvh, P, a.hd);
  const int64_t stride = page_base(1, a.Hkv, 0, P, a.hd);
  auto k_at = [](int row, int c) { return row * KROW + 16 * (KROW == 128 ? c ^ ((row >> 1) & 7) : c ^ (row & 15)); };
  auto v_at = [](int row, int c) { return KB + row * 128 + 16 * (c ^ ((row >> 1) & 7)); };

  // This thread's pieces: of the keys (row, 16 head values) or the values (head
  // value, 16 keys; neighbours within a page follow each other).  The pieces of a wave
  // lie in one page, whatever the page holds: its number and the page's address
  // are scalars, and a thread adds a constant.
  static_assert(NK % NT == 0, "a thread's i-th piece is of keys or of values for the whole workgroup");
  auto of_keys = [](int i) { return NT * i < NK; };
  const int ql = min(a.plog - 4, 2);  // log2 of the runs of 16 keys per page and block
  uint32_t off[CH];                   // byte within the page's keys or values, less the scalar part
  int l0[CH];                         // LDS byte of its first chunk; the second one's is l0 ^ 16
  int grp0[CH];                       // first run of the wave's piece (scalar)
  auto value_piece = [&](int i, int &row, int &grp) {
    const int f = tid + NT * i - NK, lo = f & ((1 << ql) - 1);
    row = (f >> ql) % HDP;
    grp = ((f >> ql) / HDP << ql) + lo;
    return lo;
  };
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const int e = tid + NT * i;
    if (of_keys(i)) {
      const int row = e / XK, x = e % XK, k = row & 15, R = (row & 32) + 8 * (k >> 2) + 4 * ((row >> 4) & 1) + (k & 3);
      grp0[i] = (64 * wave + NT * i) / (16 * XK);
      off[i] = uint32_t((ONE ? row : k) * a.hd + min(16 * x, a.hd - 16));
      l0[i] = k_at(R, 2 * x);
    } else {
      int row, grp;
      const int lo = value_piece(i, row, grp);
      off[i] = uint32_t(min(row, a.hd - 1) * P + 16 * lo);
      l0[i] = v_at(row, 2 * grp);
      grp0[i] = ((64 * wave + NT * i - NK) >> ql) / HDP << ql;
    }
  }

  // (the last rows first: with causal masks they have the most keys)
  for (int tile = a.tiles - 1 - it.item / a.splits; long(tile) * RB < w.rows; tile += a.tiles) {
    const int R0 = tile * RB, r_first = R0 + wave * RW;
    const KeyRange all = seen_keys(w.len, w.nq, R0 / a.G, (min(R0 + RB, w.rows) - 1) / a.G, a.causal, a.window);
    const KeyRange mine = key_share(all, w.split, a.splits, a.chunk);
    // keys that every row of the workgroup sees, and the first that some row does
    const int all_lo = max(seen_keys(w.len, w.nq, (min(R0 + RB, w.rows) - 1) / a.G, 0, a.causal, a.window).lo, mine.lo),
              all_hi = min(seen_keys(w.len, w.nq, 0, R0 / a.G, a.causal, a.window).hi, mine.hi), any_lo = max(all.lo, mine.lo);
    const bool on = r_first < w.rows;

    // ---- this wave's rows: column n is row r_first + n (past the last, that row
    // again, not stored)
    const int row = min(r_first + n, w.rows - 1), qi = row / a.G;
    const int i0 = min(r_first, w.rows - 1) / a.G, i1 = (min(r_first + RW, w.rows) - 1) / a.G;
    const KeyRange kr = seen_keys(w.len, w.nq, qi, qi, a.causal, a.window);
    const int row_lo = max(kr.lo, mine.lo), row_hi = min(kr.hi, mine.hi);
    const KeyRange some = seen_keys(w.len, w.nq, i0, i1, a.causal, a.window);
    const int every_lo = max(seen_keys(w.len, w.nq, i1, i1, a.causal, a.window).lo, mine.lo);
    const int every_hi = min(seen_keys(w.len, w.nq, i0, i0, a.causal, a.window).hi, mine.hi);
    f16x8 qf[NP][KS];
    float c_row, mx = -__builtin_inff(), l = 0.f, lref = -126.f;
    f32x16 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) acc[i][j] = 0.f;
    {
      const T *qp = static_cast<const T *>(a.q) + long(w.row0 + qi) * a.ldq + long(w.kvh * a.G + row - qi * a.G) * a.hd;
      float v[KS][8], big = 0.f;
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = 16 * s + 8 * h, e = min(d, a.hd - 8);
        if constexpr (DT == F32) {
          ld4<F32>(qp + e, v[s]);
          ld4<F32>(qp + e + 4, v[s] + 4);
        } else {
          dec8<DT>(*reinterpret_cast<const uint4 *>(qp + e), v[s]);
        }
#pragma unroll
        for (int e8 = 0; e8 < 8; ++e8) v[s][e8] = d < a.hd ? v[s][e8] : 0.f;
        big = finite_max8(v[s], big);
      }
      const float lift = row_lift(xor32_max(big)), up = __builtin_copysignf(lift, a.c);
      c_row = __builtin_fabsf(a.c) / lift;  // (a power of two; the scale's sign is q's)
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float x = v[s][e] * up;
          const _Float16 h0 = _Float16(x);
          qf[0][s][e] = h0;
          if constexpr (NP == 2) qf[1][s][e] = _Float16(x - float(h0));
        }
    }

    // ---- the loader.  Every load is made, at an address that exists (see above).
    int page[CH], ipage = -1;  // of the block asked for
    int ip = -1, holes = 0;    // of the block fetched; holes: pieces whose page is outside the pool
    const int last = __builtin_amdgcn_readfirstlane(mine.hi) - 1;
    const auto table_s = scalar_ptr(table);
    uint4 raw[CH];
    float isc = 0.f, ivs = 0.f;
    const auto ks_s = scalar_ptr(reinterpret_cast<const int32_t *>(a.ks)), vs_s = scalar_ptr(reinterpret_cast<const int32_t *>(a.vs));
    int p_far = -1, p_near = -1;        // (one page a block) pages of the block fetched, of the block before it
    float ks_next = 0.f, vs_next = 0.f;  // scales of the block that comes next
    auto ask = [&](int base) {  // pages of the block
      if constexpr (ONE) {
        page[0] = table_s[uint32_t(min(base, last)) >> a.plog];
      } else {
#pragma unroll
        for (int i = 0; i < CH; ++i) page[i] = table_s[uint32_t(min(base + 16 * grp0[i], last)) >> a.plog];
        if (wave == 0) ipage = table[uint32_t(min(base + 16 * (tid & 3), last)) >> a.plog];
      }
    };
    auto ask_scales = [&]() {  // of the block before the one that was fetched last
      if constexpr (ONE) {
        const int64_t at = int64_t(max(p_near, 0)) * a.Hkv + w.kvh;
        ks_next = __int_as_float(ks_s[at]);
        vs_next = __int_as_float(vs_s[at]);
      }
    };
    auto load_piece = [&](int i, const uint8_t *from) {
      uint32_t o = off[i];
      asm volatile("" : "+v"(o));  // (a scalar address and 32 bits, not a 64-bit sum kept for each piece)
      raw[i] = *reinterpret_cast<const uint4 *>(from + o);
    };
    auto fetch = [&](int base) {  // its bytes and scales
      holes = 0;
      if constexpr (ONE) {
        const bool in = page_in_pool(page[0], a.n_pages);
        p_near = p_far;
        p_far = __builtin_amdgcn_readfirstlane(in ? page[0] : -1);
        const int at = base & (P - 1);
        const int64_t from = (in ? page[0] : 0) * stride;
        const uint8_t *const kb = kc + from + at * a.hd, *const vb = vc + from + at;
#pragma unroll
        for (int i = 0; i < CH; ++i) load_piece(i, of_keys(i) ? kb : vb);
        if (!in) {
          holes = -1;
          if (tid == 0) atomicOr(a.err, kErrPage);
        }
        return;
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const bool in = page_in_pool(page[i], a.n_pages);
        const int p = in ? page[i] : 0, at = (base + 16 * grp0[i]) & (P - 1);
        if (!in) holes |= 1 << i;
        load_piece(i, (of_keys(i) ? kc + at * a.hd : vc + at) + p * stride);
      }
      if (wave == 0) {
        ip = page_in_pool(ipage, a.n_pages) ? ipage : -1;
        isc = a.ks[long(max(ip, 0)) * a.Hkv + w.kvh];
        ivs = a.vs[long(max(ip, 0)) * a.Hkv + w.kvh];
      }
    };
    auto place = [&](int base, int buf) {  // into LDS as fp16
      uint32_t any = 0, runs = 0;
      if (base < all_lo || base + kKeyBlock > all_hi || holes) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          if (of_keys(i)) continue;
          int vrow, grp;
          (void)value_piece(i, vrow, grp);
          const int t = base + 16 * grp;
          raw[i] = keep_bytes(raw[i], min(max(any_lo - t, 0), 16), holes >> i & 1 ? 0 : min(max(mine.hi - t, 0), 16));
          uint32_t b[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w}, bits = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t nb = nan_bytes(b[c]);
            b[c] &= ~(nb * 0xffu);
            bits |= ((nb & 1u) | (nb >> 7 & 2u) | (nb >> 14 & 4u) | (nb >> 21 & 8u)) << (4 * c);
          }
          raw[i] = make_uint4(b[0], b[1], b[2], b[3]);
          any |= bits;
          runs |= ((1u << (1 << ql)) - 1u) << grp0[i];
          reinterpret_cast<uint16_t *>(nan_at[buf])[vrow * 4 + grp] = uint16_t(bits);
        }
        any = __any(any != 0) ? runs : 0u;
      }
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        *reinterpret_cast<f16x8 *>(&lds[buf][l0[i]]) = cvt8(raw[i].x, raw[i].y);
        *reinterpret_cast<f16x8 *>(&lds[buf][l0[i] ^ 16]) = cvt8(raw[i].z, raw[i].w);
      }
      if (lane == 0) dirty[buf][wave] = any;
      if (!ONE && wave == 0) {
        const float lv = ip >= 0 ? fmaxf(__builtin_amdgcn_logf(ivs), -126.f) : -126.f;
        if (tid < 4) {
          // (pages behind the window may be gone)
          if (ip < 0 && base + 16 * tid < mine.hi && base + 16 * tid + 16 > any_lo) atomicOr(a.err, kErrPage);
          info[buf][tid] = make_float4(isc, lv, ip >= 0 ? 1.f : 0.f, 0.f);
        }
      }
    };

    if (mine.lo < mine.hi) {
      const int first = mine.lo & ~(kKeyBlock - 1);
      ask(first);
      fetch(first);
      ask(first + kKeyBlock);
      place(first, 0);
      fetch(first + kKeyBlock);
      ask_scales();
      ask(first + 2 * kKeyBlock);
      __syncthreads();
      int buf = 0;
      for (int base = first; base < mine.hi; base += kKeyBlock, buf ^= 1) {
        // The next block into LDS, and the one behind it on its way: its bytes have
        // the whole of this block to arrive (loaded after the scores and placed behind the
        // values' product, 672 us where this took 660, when small pages' form served all).
        const float ks_now = ks_next, vs_now = vs_next;
        const bool ok_now = p_near >= 0;
        if (base + kKeyBlock < mine.hi) place(base + kKeyBlock, buf ^ 1);
        fetch(base + 2 * kKeyBlock);
        const bool busy = on && base < some.hi && base + kKeyBlock > some.lo;
        if (!busy) {
          ask_scales();
          ask(base + 3 * kKeyBlock);
        }
        if (busy) {
          // LDS bytes of this lane's first operands; the chunks of a row differ in an
          // exclusive or (hidden from the compiler, which would keep every sum)
          uint32_t at_k = uint32_t(buf) * (KB + VB) + k_at(n, h), at_v = uint32_t(buf) * (KB + VB) + v_at(n, 2 * h);
          asm volatile("" : "+v"(at_k), "+v"(at_v));
          // this lane half's two runs of keys: 16 h of either tile
          float4 in[2];
          if constexpr (ONE) {
            const float lv = ok_now ? fmaxf(__builtin_amdgcn_logf(vs_now), -126.f) : -126.f;
            in[0] = in[1] = make_float4(ks_now, lv, ok_now ? 1.f : 0.f, 0.f);
          } else {
            in[0] = info[buf][h];
            in[1] = info[buf][2 + h];
          }
          f32x16 s[2];
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) s[t][j] = 0.f;
          // Operands are read two steps ahead of their products (left alone, the
          // compiler reads one, waits, multiplies).
          f16x8 kf[3][2];
          auto read_keys = [&](int c) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
              kf[c % 3][t] = *reinterpret_cast<const f16x8 *>(lds[0] + (at_k ^ (32 * c)) + 32 * t * KROW);
          };
          read_keys(0);
          read_keys(1);
#pragma unroll
          for (int c = 0; c < KS; ++c) {
            if (c + 2 < KS) read_keys(c + 2);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int p = NP - 1; p >= 0; --p)
                s[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[c % 3][t], qf[p][c], s[t], 0, 0, 0);
          }
          // (scalar loads, where no LDS read is on its way: the two share a counter and
          // come back in any order)
          ask_scales();
          ask(base + 3 * kKeyBlock);
          const float lv[2] = {in[0].y, in[1].y};
          const bool ok0 = in[0].z != 0.f, ok1 = in[1].z != 0.f;
          auto seen = [&](int t) -> uint32_t {  // bit i: this row sees key 32 t + 16 h + i
            const int k0 = base + 32 * t + 16 * h, lo = min(max(row_lo - k0, 0), 16), hi = min(max(row_hi - k0, 0), 16);
            return (t ? ok1 : ok0) ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
          };
          const bool masked = base < every_lo || base + kKeyBlock > every_hi || __any(!ok0 || !ok1);
          if (masked) {
            const uint32_t ok[2] = {seen(0), seen(1)};
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int j = 0; j < 16; ++j) s[t][j] = (ok[t] >> j) & 1u ? s[t][j] : -__builtin_inff();
            // a page of which the row sees nothing may have anything as scales
#pragma unroll
            for (int t = 0; t < 2; ++t) in[t].x = ok[t] ? in[t].x : 1.f;
          }
          // (c_row and a page's scale are positive: the largest raw score is its largest score)
          float f[2] = {in[0].x * c_row, in[1].x * c_row}, top = -__builtin_inff(), both = -__builtin_inff();
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            f[t] = f[t] == 0.f ? 1e-37f : f[t];  // (so that a masked score stays -inf)
            float m = s[t][0];
#pragma unroll
            for (int j = 1; j < 16; ++j) m = fmaxf(m, s[t][j]);
            m = m > -__builtin_inff() ? m * f[t] : -__builtin_inff();
            top = fmaxf(top, m);
            if constexpr (!ONE) both = fmaxf(both, m > -__builtin_inff() ? m + lv[t] : m);
          }
          top = xor32_max(top);
          both = ONE ? top + lv[0] : xor32_max(both);
          float down, down_both;
          if (__any(passes(top, both, mx, lref, down, down_both))) {
            l *= down;
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] *= down_both;
          }
          float ref = mx > -__builtin_inff() ? mx : 0.f;
          const bool far = __builtin_fabsf(ref) > 65536.f;
          if (__any(far)) {
#pragma clang fp contract(off)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
              for (int j = 0; j < 16; ++j) s[t][j] = far ? s[t][j] * f[t] - ref : s[t][j];
              f[t] = far ? 1.f : f[t];
            }
            ref = far ? 0.f : ref;
          }
          // probabilities of 32 keys, and their values; the next values on their way
          // (heads up to 128: above, the registers do not hold two tiles' values)
          constexpr bool AHEAD = HDP <= 128;
          f16x8 vf[2][AHEAD ? MT : 1];
          auto value_at = [&](int k, int i) {  // step k: keys 8 (k & 1) .. + 7 of tile k / 2's runs
            return *reinterpret_cast<const f16x8 *>(lds[0] + (at_v ^ (16 * (4 * (k >> 1) + (k & 1)))) + 32 * i * 128);
          };
          auto read_values = [&](int k) {
            if constexpr (AHEAD) {
#pragma unroll
              for (int i = 0; i < MT; ++i) vf[k & 1][i] = value_at(k, i);
              __builtin_amdgcn_sched_barrier(0);
            }
          };
          read_values(0);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const float lf = apart<NP>(lv[t], lref), unscale = __builtin_amdgcn_exp2f(-lf), lift = __builtin_amdgcn_exp2f(lf + kLift),
                        shift = lf + kLift - ref;
            float sum = 0.f;
            f16x8 pf[NP][2];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
              for (int e = 0; e < 8; ++e) {
                const float raw_s = s[t][8 * u + e];
                float p = __builtin_amdgcn_exp2f(NP == 2 ? fmaf(raw_s, f[t], -ref) : fmaf(raw_s, f[t], shift));
                if constexpr (NP == 2) p *= lift;
                sum += p;  // (not of the rounded values: see above)
                const _Float16 h0 = _Float16(p);
                pf[0][u][e] = h0;
                if constexpr (NP == 2) pf[1][u][e] = _Float16(p - float(h0));
              }
            l = fmaf(sum, unscale, l);
#pragma unroll
            for (int u = 0; u < 2; ++u) {
              if (2 * t + u < 3) read_values(2 * t + u + 1);
#pragma unroll
              for (int i = 0; i < MT; ++i) {
                f16x8 v;
                if constexpr (AHEAD) v = vf[u][i];
                else v = value_at(2 * t + u, i);
#pragma unroll
                for (int p = NP - 1; p >= 0; --p) acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pf[p][u], acc[i], 0, 0, 0);
              }
            }
          }
          // (NaN values are cleared for the whole workgroup: where some row of another
          // wave does not see the block, too)
          uint32_t nans = 0;
          if (base < all_lo || base + kKeyBlock > all_hi || __any(!ok0 || !ok1))
#pragma unroll
            for (int v = 0; v < NW; ++v) nans |= dirty[buf][v];
          nans = __builtin_amdgcn_readfirstlane(nans);
          if (nans) {
            // outputs of rows that see a NaN value (a zero probability alone would
            // not keep it from the others)
            uint64_t sees = uint64_t(seen(0)) << (16 * h) | uint64_t(seen(1)) << (32 + 16 * h);
            sees |= uint64_t(uint32_t(__shfl_xor(int(uint32_t(sees)), 32, 64))) |
                    uint64_t(uint32_t(__shfl_xor(int(uint32_t(sees >> 32)), 32, 64))) << 32;
            // (bit r of nans: the 16 keys of run r)
            sees &= uint64_t((nans & 1u) * 0xffffu | (nans >> 1 & 1u) * 0xffff0000u) |
                    uint64_t((nans >> 2 & 1u) * 0xffffu | (nans >> 3 & 1u) * 0xffff0000u) << 32;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
              for (int j = 0; j < 16; ++j)
                if (nan_at[buf][32 * i + 8 * (j >> 2) + 4 * h + (j & 3)] & sees) acc[i][j] = __builtin_nanf("");
          }
        }
        __syncthreads();
      }
    }
    l = xor32_add(l);
    if (r_first + n < w.rows) {
      const RowOut<DT> to(a, w.row0, w.kvh, w.split, row, mx, l, h == 0);
      const float inv = over(l), up = __builtin_amdgcn_exp2f(lref);  // (in this order: see above)
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = 32 * i + 8 * j + 4 * h;
          if (d < a.hd) to.put(d, f32x4{acc[i][4 * j], acc[i][4 * j + 1], acc[i][4 * j + 2], acc[i][4 * j + 3]} * inv * up);
        }
    }
  }
}

// The shares of a row joined: M the largest maximum, o = sum_s o_s l_s 2^(m_s - M) /
// sum_s l_s 2^(m_s - M), divided at each step (the products may pass a float).  The
// cut of a workgroup is JoinShape's; a row's groups are added in group order.
template <int DT>
__global__ void __launch_bounds__(kJoinThreads)
paged_join_kernel(const float *__restrict__ part_o, const float2 *__restrict__ part_ml, const int32_t *__restrict__ cu, void *out,
                  long ldo, int B, int Hq, int hd, int splits, JoinShape cut, int n_rows) {
  typedef typename Store<DT>::T T;
  __shared__ f32x4 so[kJoinThreads];
  __shared__ float2 sm[kJoinThreads];
  const int tid = threadIdx.x, per = cut.per, groups = cut.groups;
  const JoinUnit unit = join_unit(tid, per, groups, cut.rows);
  const int grp = unit.group, d = unit.d;
  const long row = long(blockIdx.x) * cut.rows + unit.row, t = row / Hq;
  const bool live = unit.on && t >= cu[0] && t < min(cu[B], n_rows);  // rows of no request are left as they are
  float top = -__builtin_inff(), sum = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
  auto add = [&](float m, float l, f32x4 v) {  // one more share
    if (l == 0.f) return;                      // (of no key)
    const float up = fmaxf(top, m);
    float s0 = top == up ? sum : sum * __builtin_amdgcn_exp2f(top - up), s1 = m == up ? l : l * __builtin_amdgcn_exp2f(m - up);
    top = up;
    sum = s0 + s1;
    s0 /= sum;
    s1 /= sum;
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = fmaf(v[c], s1, o[c] * s0);
  };
  if (live) {
    const float2 *ml = part_ml + row * splits;
    const float *po = part_o + row * splits * hd + d;
#pragma unroll 4
    for (int s = grp; s < splits; s += groups) {
      const float2 m = ml[s];
      // (nothing was written where there was no key)
      const f32x4 v = *reinterpret_cast<const f32x4 *>(po + long(s) * hd);
      add(m.x, m.y, v);
    }
  }
  if (groups > 1) {
    so[tid] = o;
    sm[tid] = make_float2(top, sum);
    __syncthreads();
    if (grp != 0 || !live) return;
    for (int k = 1; k < groups; ++k) add(sm[tid + k * per].x, sm[tid + k * per].y, so[tid + k * per]);
  }
  if (!live) return;
  const float v[4] = {o[0], o[1], o[2], o[3]};
  st4<DT>(static_cast<T *>(out) + t * ldo + long(row - t * Hq) * hd + d, v);
}

template <int DT, int HDP>
hipError_t launch(const PagedArgs &a, const PagedShape &s, hipStream_t st) {
  const dim3 grid{unsigned(long(s.tiles) * s.splits * a.Hkv * a.B)};
  if (s.wide)
    if (a.plog >= 6)
      hipLaunchKernelGGL((attn_paged_wide_kernel<DT, HDP, true>), grid, dim3(256), 0, st, a);
    else
      hipLaunchKernelGGL((attn_paged_wide_kernel<DT, HDP, false>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_paged_kernel<DT, HDP>), grid, dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || s.splits == 1) return e;
  const JoinShape cut = join_shape(a.hd, s.splits);
  const long rows = long(a.n_rows) * a.Hq, jb = (rows + cut.rows - 1) / cut.rows;
  hipLaunchKernelGGL(paged_join_kernel<DT>, dim3(unsigned(jb)), dim3(kJoinThreads), 0, st, a.part_o, a.part_ml, a.cu, a.out, a.ldo,
                     a.B, a.Hq, a.hd, a.splits, cut, a.n_rows);
  return hipGetLastError();
}

template <int DT> hipError_t launch_hd(const PagedArgs &a, const PagedShape &s, hipStream_t st) {
  if (a.hd <= 64) return launch<DT, 64>(a, s, st);
  if (a.hd <= 128) return launch<DT, 128>(a, s, st);
  return launch<DT, 256>(a, s, st);
}

}  // namespace

hipError_t attention_paged(int dt, const PagedAttention &p, const PagedShape &s, hipStream_t st) {
  PagedArgs a;
  a.q = p.q;
  a.out = p.out;
  a.kc = static_cast<const uint8_t *>(p.k_cache);
  a.vc = static_cast<const uint8_t *>(p.v_cache);
  a.ks = p.k_scale;
  a.vs = p.v_scale;
  a.tables = p.tables;
  a.lens = p.lens;
  a.cu = p.cu;
  a.part_o = static_cast<float *>(p.workspace);
  a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(p.workspace) + paged_part_bytes(p.n_rows, p.Hq, p.hd, s.splits));
  a.err = p.err;
  a.ldq = p.ldq;
  a.ldo = p.ldo;
  a.B = p.B;
  a.Hq = p.Hq;
  a.Hkv = p.Hkv;
  a.G = p.Hq / p.Hkv;
  a.hd = p.hd;
  a.plog = __builtin_ctz(unsigned(p.page));
  a.n_pages = p.n_pages;
  a.n_rows = p.n_rows;
  a.width = p.width;
  a.causal = p.causal;
  a.window = p.window;
  a.splits = s.splits;
  a.chunk = s.chunk;
  a.tiles = s.tiles;
  a.c = float(double(p.scale) * 1.4426950408889634);
  switch (dt) {
  case F32: return launch_hd<F32>(a, s, st);
  case F16: return launch_hd<F16>(a, s, st);
  case BF16: return launch_hd<BF16>(a, s, st);
  default: return hipErrorInvalidValue;
  }
}

}  // namespace mh
