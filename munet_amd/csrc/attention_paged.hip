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
// two to below 2^14 and is then exact in fp16 for bf16 and fp16 inputs (down to
// 2^-38 of the row's largest value); fp32 inputs are the sum of two fp16 parts
// (22 bits and a sign).  Scores, the running maximum, the sum and the outputs are
// fp32.  A probability enters the second product as 2^14 w times its page's
// value scale over the largest one that the row has seen, rounded to fp16 (half a unit of 11
// bits down to 2^-28 of the largest; outputs of 16 bits are rounded as much
// once more), or as two such parts for fp32 inputs.
#include "mh_common.hpp"
#include "mh_kernels.hpp"
#include "paged_index.hpp"

namespace mh {
namespace {

typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

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

// NQ 16-row tiles of one (sequence, key/value head).  WIDE: the four waves take
// different rows and the same keys (many rows); else the same rows, and every
// fourth block of the keys each (few rows).
template <int DT, int HDP, int NQ, bool WIDE>
__global__ void __launch_bounds__(256) attn_paged_kernel(PagedArgs a) {
  typedef Store<DT> S;
  typedef typename S::T T;
  constexpr int NP = DT == F32 ? 2 : 1;  // fp16 parts of q and of the probabilities
  constexpr int J = HDP / 64, MT = HDP / 16;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
  int id = blockIdx.x;
  const int tile0 = id % a.tiles;
  id /= a.tiles;
  const int split = id % a.splits;
  id /= a.splits;
  const int kvh = id % a.Hkv, b = id / a.Hkv;

  const int P = 1 << a.plog;
  // (lengths past the block table's pages, and rows past the buffer, are cut)
  const int most = a.width << a.plog, len = min(max(a.lens[b], 0), most);
  const int row0 = a.cu[b], nq = min(a.cu[b + 1], a.n_rows) - row0;
  if (row0 < 0 || nq <= 0) return;
  if (a.lens[b] > most && tid == 0) atomicOr(a.err, kErrPage);
  const int rows = nq * a.G;
  const int32_t *table = a.tables + long(b) * a.width;
  constexpr int RW = 16 * NQ;               // rows per wave
  constexpr int RB = WIDE ? 4 * RW : RW;    // rows per workgroup

  // The merge of the four waves' shares (narrow form): 128 head values at a time.
  constexpr int MW = HDP < 128 ? HDP : 128, LD = MW + 4;
  __shared__ __align__(16) float wo[WIDE ? 1 : 4][WIDE ? 1 : RW][WIDE ? 4 : LD];
  __shared__ float2 wml[WIDE ? 1 : 4][WIDE ? 1 : RW];

  // (more tiles than the launch was sized for are walked)
  for (int tile = tile0; long(tile) * RB < rows; tile += a.tiles) {
    const int r_first = tile * RB + (WIDE ? wave * RW : 0);
    if (WIDE && r_first >= rows) break;  // (no barrier in this form)
    const int i0 = r_first / a.G, i1 = (min(r_first + RW, rows) - 1) / a.G;
    const KeyRange all = seen_keys(len, nq, i0, i1, a.causal, a.window);
    const KeyRange mine = key_share(all, split, a.splits, a.chunk);
    // keys that every row of the wave sees: [every_lo, every_hi)
    const int every_lo = seen_keys(len, nq, i1, i1, a.causal, a.window).lo;
    const int every_hi = seen_keys(len, nq, i0, i0, a.causal, a.window).hi;

    // the wave's queries: column n of tile x is row r_first + 16 x + n (past the
    // end: the last row again, not stored)
    f16x8 qf[NP][NQ][2 * J];
    float c_row[NQ], mx[NQ], l[NQ];
    float lref[NQ];  // log2 of the largest value scale that the row has seen
    int hi_row[NQ], lo_row[NQ];
    f32x4 acc[MT][NQ];
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      const int r = min(r_first + 16 * x + n, rows - 1), i = r / a.G, h = kvh * a.G + r - i * a.G;
      const T *qp = static_cast<const T *>(a.q) + long(row0 + i) * a.ldq + long(h) * a.hd;
      float v[2 * J][8], big = 0.f;
#pragma unroll
      for (int s = 0; s < 2 * J; ++s) {
        const int d = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
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
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float m = __builtin_fabsf(v[s][e]);
          big = m < __builtin_inff() ? fmaxf(big, m) : big;
        }
      }
      big = xor32_max(xor16_max(big));
      // 2^k times the row lies below 2^14
      const int ex = int(__float_as_uint(big) >> 23);  // biased exponent, 0 for zero and subnormal rows
      const int k = ex == 0 ? 0 : min(13 - (ex - 127), 120);
      const float up = __uint_as_float(uint32_t(k + 127) << 23);
      c_row[x] = a.c * __uint_as_float(uint32_t(127 - k) << 23);
#pragma unroll
      for (int s = 0; s < 2 * J; ++s) {
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

    const int step = WIDE ? kKeyBlock : 4 * kKeyBlock;
    for (int base = (mine.lo & ~(kKeyBlock - 1)) + (WIDE ? 0 : wave * kKeyBlock); base < mine.hi; base += step) {
      // the pages of this lane's key rows (group n >> 2) and of its scores and
      // values (group g); a page outside the pool holds no keys (page 0 is read
      // in its place and masked)
      const int tk = base + 16 * (n >> 2), tv = base + 16 * g;
      int pk = tk < mine.hi && (tk >> a.plog) < a.width ? table[tk >> a.plog] : -1;
      int pv = tv < mine.hi && (tv >> a.plog) < a.width ? table[tv >> a.plog] : -1;
      const bool page_ok = page_in_pool(pv, a.n_pages);
      if (!page_ok && tv < mine.hi && n == 0) atomicOr(a.err, kErrPage);
      pk = page_in_pool(pk, a.n_pages) ? pk : 0;
      pv = page_ok ? pv : 0;
      const uint8_t *kp = a.kc + page_base(pk, a.Hkv, kvh, P, a.hd) + long(tk & (P - 1)) * a.hd;
      const uint8_t *vp = a.vc + page_base(pv, a.Hkv, kvh, P, a.hd) + (tv & (P - 1));
      uint4 kr[4][J], vr[MT];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int d = 64 * j + 16 * g;
          kr[t][j] = d < a.hd ? *reinterpret_cast<const uint4 *>(kp + (4 * t + (n & 3)) * a.hd + d) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
      for (int i = 0; i < MT; ++i)
        vr[i] = 16 * i < a.hd ? *reinterpret_cast<const uint4 *>(vp + (16 * i + n) * P) : make_uint4(0, 0, 0, 0);
      const float ksc = a.ks[long(pv) * a.Hkv + kvh], vsc = a.vs[long(pv) * a.Hkv + kvh];

      // scores
      f32x4 s[4][NQ];
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int x = 0; x < NQ; ++x) s[t][x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const f16x8 k0 = cvt8(kr[t][j].x, kr[t][j].y), k1 = cvt8(kr[t][j].z, kr[t][j].w);
#pragma unroll
          for (int x = 0; x < NQ; ++x) {
#pragma unroll
            for (int p = NP - 1; p >= 0; --p) {
              s[t][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[p][x][2 * j], s[t][x], 0, 0, 0);
              s[t][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[p][x][2 * j + 1], s[t][x], 0, 0, 0);
            }
          }
        }
      }

      const float lv = page_ok ? fmaxf(__builtin_amdgcn_logf(vsc), -126.f) : -126.f;

      // some row does not see every key of the block
      const bool masked = base < max(every_lo, mine.lo) || base + kKeyBlock > min(every_hi, mine.hi) || __any(!page_ok);
      f16x8 pf[NP][NQ][2];
      uint32_t ok[NQ];
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        ok[x] = 0xffffu;
        if (masked) {
          // keys tv + e, lo <= tv + e < hi
          const int lo = min(max(lo_row[x] - tv, 0), 16), hi = min(max(hi_row[x] - tv, 0), 16);
          ok[x] = page_ok ? ((1u << hi) - 1u) & ~((1u << lo) - 1u) : 0u;
#pragma unroll
          for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[t][x][r] = (ok[x] >> (4 * t + r)) & 1u ? s[t][x][r] : -__builtin_inff();
        }
        // the value scales: this lane group's over the largest that the row has seen
        const float lnew = fmaxf(xor32_max(xor16_max(ok[x] ? lv : -126.f)), lref[x]), lf = ok[x] ? lv - lnew : 0.f;
        const float rescale = lnew == lref[x] ? 1.f : __builtin_amdgcn_exp2f(lref[x] - lnew);
        const float unscale = __builtin_amdgcn_exp2f(-lf), scale14 = __builtin_amdgcn_exp2f(lf + 14.f);
        lref[x] = lnew;
        // (a page's scale is positive: the largest raw score is the largest score)
        float f = ksc * c_row[x];
        float top = s[0][x][0];
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
          for (int r = 0; r < 4; ++r) top = fmaxf(top, s[t][x][r]);
        top = top > -__builtin_inff() ? top * f : -__builtin_inff();
        top = fmaxf(xor32_max(xor16_max(top)), mx[x]);
        float ref = top > -__builtin_inff() ? top : 0.f;
        const float down = mx[x] == top ? 1.f : __builtin_amdgcn_exp2f(mx[x] - ref);
        mx[x] = top;
        if (__any(down * rescale != 1.f)) {
          l[x] *= down;
#pragma unroll
          for (int i = 0; i < MT; ++i) acc[i][x] *= down * rescale;
        }
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
              float t = NP == 2 ? fmaf(raw, f, -ref) : fmaf(raw, f, lf + 14.f - ref);
              if (masked) t = raw == -__builtin_inff() ? raw : t;
              p[y] = __builtin_amdgcn_exp2f(t);
              if constexpr (NP == 2) p[y] *= scale14;
              sum += p[y];
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const _Float16 h0 = _Float16(p[y]);
              pf[0][x][u][e + y] = h0;
              if constexpr (NP == 2) pf[1][x][u][e + y] = _Float16(p[y] - float(h0));
            }
          }
        l[x] = fmaf(sum, unscale, l[x]);  // (2^14 w)
      }

      // values.  Keys that no row sees may hold anything, NaN among it: their
      // bytes are cleared.  A NaN value that only some rows see must reach
      // these alone, which a zero probability does not give: such a block (one
      // at the edge of the mask with a NaN byte) clears the NaN bytes and marks
      // the outputs of the rows that see them.
      bool nans = false;
      if (masked) {
        const int lo = min(max(max(all.lo, mine.lo) - tv, 0), 16), hi = page_ok ? min(max(min(all.hi, mine.hi) - tv, 0), 16) : 0;
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
          uint32_t w[4] = {vr[i].x, vr[i].y, vr[i].z, vr[i].w}, mark[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t nb = nan_bytes(w[c]);
            w[c] &= ~(nb * 0xffu);
            mark[c] = nb * 0x38u;  // e4m3 1.0
          }
          vr[i] = make_uint4(w[0], w[1], w[2], w[3]);
          const f16x8 m0 = cvt8(mark[0], mark[1]), m1 = cvt8(mark[2], mark[3]);
#pragma unroll
          for (int x = 0; x < NQ; ++x) {
            f16x8 s0, s1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              s0[e] = (ok[x] >> e) & 1u ? _Float16(1.f) : _Float16(0.f);
              s1[e] = (ok[x] >> (8 + e)) & 1u ? _Float16(1.f) : _Float16(0.f);
            }
            f32x4 hit = f32x4{0.f, 0.f, 0.f, 0.f};
            hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(m0, s0, hit, 0, 0, 0);
            hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(m1, s1, hit, 0, 0, 0);
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (hit[r] > 0.f) acc[i][x][r] = __builtin_nanf("");
          }
        }
      }
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const f16x8 v0 = cvt8(vr[i].x, vr[i].y), v1 = cvt8(vr[i].z, vr[i].w);
#pragma unroll
        for (int x = 0; x < NQ; ++x)
#pragma unroll
          for (int p = NP - 1; p >= 0; --p) {
            acc[i][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[p][x][0], acc[i][x], 0, 0, 0);
            acc[i][x] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[p][x][1], acc[i][x], 0, 0, 0);
          }
      }
    }

    // the values' scale, and the rows' sums over the lane groups
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      l[x] = xor32_add(xor16_add(l[x]));
#pragma unroll
      for (int i = 0; i < MT; ++i) acc[i][x] *= __builtin_amdgcn_exp2f(lref[x]);
    }

    // rows out: o = acc / l, or this share's (acc, maximum, l)
    auto put = [&](int r, int d, f32x4 o, float m, float sum) {
      const int i = r / a.G, h = kvh * a.G + r - i * a.G;
      if (a.splits == 1) {
        const float inv = sum == 0.f ? 0.f : 1.f / sum;  // (a row that sees no key is zero)
        const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
        st4<DT>(static_cast<T *>(a.out) + long(row0 + i) * a.ldo + long(h) * a.hd + d, v);
      } else {
        const long at = ((long(row0) + i) * a.Hq + h) * a.splits + split;
        if (!(sum == 0.f)) *reinterpret_cast<f32x4 *>(a.part_o + at * a.hd + d) = o;  // (the join skips empty shares)
        if (d == 0) a.part_ml[at] = make_float2(m, sum);
      }
    };
    if constexpr (WIDE) {
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        const int r = r_first + 16 * x + n;
        if (r < rows) {
#pragma unroll
          for (int i = 0; i < MT; ++i)
            if (16 * i < a.hd) put(r, 16 * i + 4 * g, acc[i][x], mx[x], l[x]);
        }
      }
    } else {
      // the four waves' shares of the keys, in wave order
      if (g == 0) {
#pragma unroll
        for (int x = 0; x < NQ; ++x) wml[wave][16 * x + n] = make_float2(mx[x], l[x]);
      }
#pragma unroll
      for (int part = 0; part < HDP / MW; ++part) {
#pragma unroll
        for (int x = 0; x < NQ; ++x)
#pragma unroll
          for (int i = 0; i < MW / 16; ++i)
            *reinterpret_cast<f32x4 *>(&wo[wave][16 * x + n][16 * i + 4 * g]) = acc[part * (MW / 16) + i][x];
        __syncthreads();
        for (int e = tid; e < RW * (MW / 4); e += 256) {
          const int rr = e / (MW / 4), d = 4 * (e % (MW / 4));
          const int r = r_first + rr;
          if (r < rows && part * MW + d < a.hd) {
            float top = wml[0][rr].x;
#pragma unroll
            for (int w = 1; w < 4; ++w) top = fmaxf(top, wml[w][rr].x);
            float sum = 0.f;
            f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const float2 ml = wml[w][rr];
              if (ml.y == 0.f) continue;  // (this wave saw no key)
              const float f = ml.x == top ? 1.f : __builtin_amdgcn_exp2f(ml.x - top);
              sum = fmaf(ml.y, f, sum);
              const f32x4 v = *reinterpret_cast<const f32x4 *>(&wo[w][rr][d]);
#pragma unroll
              for (int c = 0; c < 4; ++c) o[c] = fmaf(v[c], f, o[c]);
            }
            put(r, part * MW + d, o, top, sum);
          }
        }
        __syncthreads();
      }
    }
  }
}

// The shares of a row joined: M the largest maximum, o = sum_s o_s 2^(m_s - M) /
// sum_s l_s 2^(m_s - M), in share order.  hd / 4 threads per row.
template <int DT>
__global__ void __launch_bounds__(256)
paged_join_kernel(const float *__restrict__ part_o, const float2 *__restrict__ part_ml, const int32_t *__restrict__ cu, void *out,
                  long ldo, int B, int Hq, int hd, int splits, int n_rows) {
  typedef typename Store<DT>::T T;
  const int per = hd / 4, rpb = 256 / per, rr = threadIdx.x / per;
  const long row = long(blockIdx.x) * rpb + rr;
  if (rr >= rpb) return;
  const int d = 4 * (threadIdx.x - rr * per);
  const long t = row / Hq;
  if (t < cu[0] || t >= min(cu[B], n_rows)) return;  // rows of no sequence are left as they are
  const int h = int(row - t * Hq);
  const float2 *ml = part_ml + row * splits;
  const float *po = part_o + row * splits * hd + d;
  float top = -__builtin_inff();
  for (int s = 0; s < splits; ++s) top = fmaxf(top, ml[s].x);
  float sum = 0.f;
  f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    const float2 m = ml[s];
    if (m.y == 0.f) continue;  // (no key in this share)
    const float f = m.x == top ? 1.f : __builtin_amdgcn_exp2f(m.x - top);
    sum = fmaf(m.y, f, sum);
    const f32x4 v = *reinterpret_cast<const f32x4 *>(po + long(s) * hd);
#pragma unroll
    for (int c = 0; c < 4; ++c) o[c] = fmaf(v[c], f, o[c]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const float v[4] = {o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv};
  st4<DT>(static_cast<T *>(out) + t * ldo + long(h) * hd + d, v);
}

template <int DT, int HDP>
hipError_t launch(const PagedArgs &a, const PagedShape &s, hipStream_t st) {
  const long blocks = long(s.tiles) * s.splits * a.Hkv * a.B;
  if (blocks * 256 > 0xffffffffL) return hipErrorInvalidValue;
  const dim3 grid{unsigned(blocks)};
  constexpr int NQ = DT == F32 || HDP > 128 ? 1 : 2;
  if (s.wide)
    hipLaunchKernelGGL((attn_paged_kernel<DT, HDP, NQ, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attn_paged_kernel<DT, HDP, 1, false>), grid, dim3(256), 0, st, a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || s.splits == 1) return e;
  const int rpb = 256 / (a.hd / 4);
  const long rows = long(a.n_rows) * a.Hq, jb = (rows + rpb - 1) / rpb;
  if (jb * 256 > 0xffffffffL) return hipErrorInvalidValue;
  hipLaunchKernelGGL(paged_join_kernel<DT>, dim3(unsigned(jb)), dim3(256), 0, st, a.part_o, a.part_ml, a.cu, a.out, a.ldo, a.B, a.Hq,
                     a.hd, a.splits, a.n_rows);
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
