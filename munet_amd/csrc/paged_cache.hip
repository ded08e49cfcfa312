// The paged 8-bit KV cache's bookkeeping and its writes (paged_index.hpp has the
// layouts).
#include "mh_common.hpp"
#include "mh_kernels.hpp"
#include "paged_index.hpp"
#include "rotary.hpp"

namespace mh {
namespace {

// ---- page_plan ---------------------------------------------------------------

// Sums over the requests before its own: every workgroup adds them up itself
// instead of waiting for another (8 bytes a request, from the caches; one launch:
// 4096 requests 24 us a call, 16384 222, 65536 3050).
struct Need {
  int64_t tokens, pages;
};
__device__ __forceinline__ int64_t wave_sum64(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

__device__ __forceinline__ Need need_of(const PagePlan &p, int b) {
  const PlanNeed n = plan_need(p.lens[b], p.fresh[b], p.page, p.width);
  return Need{n.fresh, n.need - n.have};
}

// blockIdx.x is the request; its workgroups (blockIdx.y) go round its tokens, the
// last request's also round the slots behind the last token.  The first one
// writes the rest.
__global__ void __launch_bounds__(256) page_plan_kernel(PagePlan p, int *err) {
  __shared__ int64_t part[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x, turn = 256 * gridDim.y, at0 = 256 * blockIdx.y + tid;
  Need before{0, 0};
  for (int o = tid; o < b; o += 256) {
    const Need n = need_of(p, o);
    before.tokens += n.tokens;
    before.pages += n.pages;
  }
  const int64_t t = wave_sum64(before.tokens), g = wave_sum64(before.pages);
  if (lane == 0) {
    part[0][wave] = t;
    part[1][wave] = g;
  }
  __syncthreads();
  const int64_t tok = part[0][0] + part[0][1] + part[0][2] + part[0][3];
  const int64_t first = part[1][0] + part[1][1] + part[1][2] + part[1][3];
  const PlanNeed n = plan_need(p.lens[b], p.fresh[b], p.page, p.width);
  int32_t *table = p.tables + int64_t(b) * p.width;
  // a page of this request's list: held before, or the next free one
  auto page_at = [&](int i) -> int {
    int page = -1;
    if (i < n.have) page = i < p.width ? table[i] : -1;
    else if (i < n.need) page = first + i - n.have < p.n_free ? p.free_pages[first + i - n.have] : -1;
    return page_in_pool(page, p.n_pages) ? page : -1;
  };
  int bad = 0;
  for (int64_t i = at0; i < n.fresh; i += turn) {
    const int64_t at = tok + i, pos = int64_t(n.len) + i;
    if (at >= p.cap) {
      bad = 1;
      break;
    }
    const int nth = int(pos) / p.page, page = nth < p.width ? page_at(nth) : -1;  // (pos is below 2^31)
    if (page < 0) bad = 1;
    p.slots[at] = page < 0 ? -1 : page * p.page + int(pos) % p.page;
    if (p.positions) p.positions[at] = int(pos);
  }
  if (bad) atomicOr(err, kErrPlan);
  const int64_t end = tok + n.fresh;
  if (blockIdx.y == 0) {
    for (int i = n.have + tid; i < n.need; i += 256) table[i] = page_at(i);
    if (tid == 0) {
      p.total[b] = int(int64_t(n.len) + n.fresh);
      if (b == 0) p.cu[0] = 0;
      p.cu[b + 1] = int(end < p.cap ? end : p.cap);
      if (b + 1 == p.B) p.used[0] = int(first + n.need - n.have);
    }
  }
  // the slots behind the last token (a batch padded to a captured graph's size)
  if (b + 1 == p.B)
    for (int64_t i = end + at0; i < p.cap; i += turn) {
      p.slots[i] = -1;
      if (p.positions) p.positions[i] = 0;
    }
}

// ---- kv_store_paged -----------------------------------------------------------

// The least power of two whose 448-fold holds amax (e4m3's largest value is
// 1.75 * 2^8), between 2^-100 and 2^120.  A power of two costs no precision (the
// values are floating point) and moves a page to a larger scale without a
// second rounding but of the smallest values.
__device__ __forceinline__ float e4m3_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  const int e = int(b >> 23) - 127 - ((b & 0x7fffffu) > 0x600000u ? 7 : 8);
  return __uint_as_float(uint32_t(min(max(e, -100), 120) + 127) << 23);
}

// four values to e4m3, to nearest even; what is not finite becomes NaN
__device__ __forceinline__ uint32_t e4m3x4(const float v[4]) {
  float w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __builtin_fabsf(v[i]) < __builtin_inff() ? v[i] : __builtin_nanf("");
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], r, true));
}
__device__ __forceinline__ void e4m3x4_dec(uint32_t w, float v[4]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), false), b = __builtin_amdgcn_cvt_pk_f32_fp8(int(w), true);
  v[0] = a[0]; v[1] = a[1]; v[2] = b[0]; v[3] = b[1];
}
// (of ratios below 1: nothing becomes infinite, and NaN stays)
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  float v[4];
  e4m3x4_dec(w, v);
  const int r = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * ratio, v[1] * ratio, 0, false);
  return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(v[2] * ratio, v[3] * ratio, r, true));
}

// eight consecutive values
template <int DT> __device__ __forceinline__ void ld8(const typename Store<DT>::T *p, float v[8]) {
  if constexpr (DT == F32) {
    ld4<F32>(p, v);
    ld4<F32>(p + 4, v + 4);
  } else {
    dec8<DT>(*reinterpret_cast<const uint4 *>(p), v);
  }
}
__device__ __forceinline__ float amax8(const float v[8], float big) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float m = __builtin_fabsf(v[e]);
    big = m < __builtin_inff() ? fmaxf(big, m) : big;
  }
  return big;
}

// eight consecutive values as they lie
template <int DT> struct Raw {
  uint4 a, b;
  __device__ __forceinline__ void load(const typename Store<DT>::T *p) {
    a = reinterpret_cast<const uint4 *>(p)[0];
    if constexpr (DT == F32) b = reinterpret_cast<const uint4 *>(p)[1];
  }
  __device__ __forceinline__ void get(float v[8]) const {
    if constexpr (DT == F32) {
      v[0] = __uint_as_float(a.x); v[1] = __uint_as_float(a.y); v[2] = __uint_as_float(a.z); v[3] = __uint_as_float(a.w);
      v[4] = __uint_as_float(b.x); v[5] = __uint_as_float(b.y); v[6] = __uint_as_float(b.z); v[7] = __uint_as_float(b.w);
    } else {
      dec8<DT>(a, v);
    }
  }
};

// Piece c of a key: eight of its values.  Where pairs lie half the rotated part apart
// (ROT 1) these are both values of pairs 4 c .. 4 c + 3, two fours at `lo` and `hi`,
// so that a thread turns what it has; with ROT 2 (neighbours paired) eight consecutive
// values are those pairs (with eight values of a half, their partners loaded too and
// the queries in a launch of their own, 17k tokens of 8 heads of 128 and 32 query heads
// took 132 us, so and in one launch 104).  Behind the pairs values go as they lie.  The
// piece at the pairs' end may be mixed: `few` whole pairs, then (ROT 1) the values
// behind all pairs, first in the places of the missing first halves, then of the second.
// Rotated keys are floats, so that the cache's 8 bits are their only rounding.
template <int DT, int ROT> struct KeyPiece {
  int lo, hi, pair, few;  // few: pairs of this piece (0 to 4)
  bool mixed;
  __device__ __forceinline__ KeyPiece(int c, int half) {
    pair = 4 * c;
    few = ROT ? min(max(half - pair, 0), 4) : 0;
    mixed = few > 0 && few < 4;
    lo = ROT == 1 && few == 4 ? pair : 8 * c;
    hi = ROT == 1 && few == 4 ? pair + half : 8 * c + 4;
  }
  // where value e of a mixed piece lies
  __device__ __forceinline__ int at(int e, int half) const {
    if (e < 4) return e < few ? pair + e : 2 * half + e - few;
    return e - 4 < few ? half + pair + e - 4 : 2 * half + (4 - few) + e - 4 - few;
  }
  __device__ __forceinline__ void load(const typename Store<DT>::T *head, const float2 *tab, int half, float v[8]) const {
    if constexpr (ROT == 0) {
      ld8<DT>(head + lo, v);
    } else if (ROT == 1 && mixed) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = Store<DT>::dec(head[at(e, half)]);
#pragma unroll
      for (int i = 0; i < 3; ++i)
        if (i < few) turn(v[i], v[4 + i], tab[pair + i].x, tab[pair + i].y);
    } else {
      ldu4<DT>(head + lo, v);
      ldu4<DT>(head + hi, v + 4);
      if (few == 0) return;
      float4 a, b;
      if (ROT == 2 && mixed) {
        const float2 x = tab[pair], y = few > 1 ? tab[pair + 1] : make_float2(1.f, 0.f), z = few > 2 ? tab[pair + 2] : make_float2(1.f, 0.f);
        a = make_float4(x.x, x.y, y.x, y.y);
        b = make_float4(z.x, z.y, 1.f, 0.f);
      } else {
        a = angles2(tab + pair);
        b = angles2(tab + pair + 2);
      }
      if constexpr (ROT == 1) {
        turn(v[0], v[4], a.x, a.y);
        turn(v[1], v[5], a.z, a.w);
        turn(v[2], v[6], b.x, b.y);
        turn(v[3], v[7], b.z, b.w);
      } else {
        turn(v[0], v[1], a.x, a.y);
        if (few > 1) turn(v[2], v[3], a.z, a.w);
        if (few > 2) turn(v[4], v[5], b.x, b.y);
        if (few > 3) turn(v[6], v[7], b.z, b.w);
      }
    }
  }
  __device__ __forceinline__ void store(uint8_t *row, int half, const float v[8], float inv) const {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = v[e] * inv;
    const uint32_t first = e4m3x4(w), second = e4m3x4(w + 4);
    if constexpr (ROT == 1) {
      struct __attribute__((packed)) Any { uint32_t v; };
      if (mixed) {
#pragma unroll
        for (int e = 0; e < 8; ++e) row[at(e, half)] = uint8_t((e < 4 ? first : second) >> (8 * (e & 3)));
      } else {
        *reinterpret_cast<uint32_t *>(row + lo) = first;
        reinterpret_cast<Any *>(row + hi)->v = second;
      }
    } else {
      *reinterpret_cast<uint2 *>(row + lo) = make_uint2(first, second);
    }
  }
};
// A token's key piece as it is held: its bits, or rotated floats.
template <int DT, int ROT> struct Key {
  float f[8];
  __device__ __forceinline__ void load(const KeyPiece<DT, ROT> &k, const typename Store<DT>::T *head, const float2 *tab, int half) {
    k.load(head, tab, half, f);
  }
  __device__ __forceinline__ void get(float v[8]) const {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = f[e];
  }
};
template <int DT> struct Key<DT, 0> {
  Raw<DT> r;
  __device__ __forceinline__ void load(const KeyPiece<DT, 0> &k, const typename Store<DT>::T *head, const float2 *, int) { r.load(head + k.lo); }
  __device__ __forceinline__ void get(float v[8]) const { r.get(v); }
};

// The scale of a page (and head) that gets values of largest magnitude `top` from
// `place` on, and what its earlier tokens are multiplied by.
struct PageScale {
  float now, inv, ratio;
  __device__ __forceinline__ PageScale(float top, float held, int place) {
    const float want = e4m3_scale(top);
    const bool keep = place > 0 && held > want && held < __builtin_inff();
    now = keep ? held : want;
    inv = 1.0f / now;
    ratio = place > 0 && held > 0.f && held < now ? held * inv : 1.f;
  }
};
// The page's earlier tokens in a larger scale, by NT threads with U pieces of 16
// bytes each in flight (places past the last piece read that one again, and store
// nothing).
template <int NT, int U> __device__ __forceinline__ void rescale_keys(uint8_t *kd, int place, int hd, float ratio, int tid) {
  uint4 *p = reinterpret_cast<uint4 *>(kd);
  const int all = place * hd / 16;
  for (int c0 = tid; c0 < all; c0 += NT * U) {
    uint4 w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = p[min(c0 + NT * u, all - 1)];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + NT * u >= all) break;
      p[c0 + NT * u] = make_uint4(rescale4(w[u].x, ratio), rescale4(w[u].y, ratio), rescale4(w[u].z, ratio), rescale4(w[u].w, ratio));
    }
  }
}
template <int NT, int U> __device__ __forceinline__ void rescale_values(uint8_t *vd, int place, int hd, int P, float ratio, int tid) {
  // (whole 16-byte pieces of a row: what lies behind the earlier tokens is kept, or
  // written afterwards)
  const int pieces = (place + 15) / 16, all = hd * pieces;
  for (int c0 = tid; c0 < all; c0 += NT * U) {
    uint4 *p[U], w[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = min(c0 + NT * u, all - 1), d = c / pieces, i = c - d * pieces;
      p[u] = reinterpret_cast<uint4 *>(vd + int64_t(d) * P + 16 * i);
      w[u] = *p[u];
      at[u] = 16 * i;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (c0 + NT * u >= all) break;
      const uint32_t o[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
      uint32_t r[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int left = place - at[u] - 4 * q;  // earlier tokens from this word on
        const uint32_t m = left >= 4 ? 0xffffffffu : left <= 0 ? 0u : (1u << (8 * left)) - 1u;
        r[q] = (rescale4(o[q], ratio) & m) | (o[q] & ~m);
      }
      *p[u] = make_uint4(r[0], r[1], r[2], r[3]);
    }
  }
}

struct StoreArgs {
  const void *k, *v;
  const int32_t *slots;
  uint8_t *kc, *vc;
  float *ks, *vs;
  int *err;
  long ldk, ldv;
  int n, Hkv, hd, page, n_pages, per;
  const float2 *table;  // rotated keys: their angles
  int half;
  Rotary q;       // queries to rotate beside them (workgroups behind the heads'), 0 heads: none
  int q_unit;
  unsigned q_groups;
};

// A run is a stretch of tokens with consecutive slots inside one page.  The
// workgroup that holds a run's first token writes all of it for one head, and
// so owns the page's two scales.  Tokens at `per` consecutive places per
// workgroup.
template <int DT, int NT, int ROT, bool ONE>
__global__ void __launch_bounds__(NT) kv_store_paged_kernel(StoreArgs a) {
  typedef typename Store<DT>::T T;
  constexpr int VT = 64;  // tokens of a value tile
  constexpr int NW = NT / 64;
  __shared__ float red[2][NW];
  // (rows of VT + 4 bytes; of the run's quads in the short form)
  __shared__ __align__(16) uint8_t vt[ONE ? kPagedHeadMax * (VT + 4) : 32 * NT + 4 * kPagedHeadMax];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, head = blockIdx.y;
  const int t0 = blockIdx.x * a.per, hd = a.hd, P = a.page, h8 = hd / 8;
  const int64_t limit = int64_t(a.n_pages) * P;
  if constexpr (ROT != 0) {
    if (head >= a.Hkv) {
      const unsigned step = (gridDim.y - a.Hkv) * gridDim.x;
      for (unsigned i = (head - a.Hkv) * gridDim.x + blockIdx.x; i < a.q_groups; i += step) {
        const int64_t first = int64_t(i) * a.q.tokens;
        if constexpr (ONE)
          rotary_unit_as<DT, ROT == 2>(a.q_unit, [&](auto u, auto inter) {
            rotate_tokens<DT, decltype(u)::value, decltype(inter)::value, NT, 2>(a.q, first, a.slots, limit);
          });
        else rotate_tokens<DT, rotary_most(DT, ROT == 2), ROT == 2, NT, 2>(a.q, first, a.slots, limit);
      }
      return;
    }
  }
  uint64_t starts;
  if constexpr (ONE) {
    // One token for the workgroup (a decode step).  Where it is a run of its own, the
    // first wave stores it without LDS or barriers, a key piece or a value piece to
    // a lane (64 tokens, 8 heads of 128: 4.2 us, through LDS 7.1; rotated, with 32 query
    // heads 4.7, 12).  Its row, the slots and the scale are waited for one after
    // another.  A page that moves to a larger scale keeps eight pieces a lane in flight
    // (64 tokens whose pages all move, in pages of 64, 128 and 256: 7.4, 11.5 and 19 us; a piece
    // at a time 11.9, 19.5 and 34.6).  All four waves at it took 6.3, 9.8 and 15.5, but they
    // stay until the first one knows: 256 tokens whose pages stay as they are 8.4 us, so 7.5.
    const int vh = lane >> 5, c = lane & 31;
    const bool on = wave == 0 && c < h8;
    const KeyPiece<DT, ROT> piece(c, a.half);
    float v[8] = {};
    if (on) {
      const int64_t hv = int64_t(head) * hd;
      if (vh) ld8<DT>(static_cast<const T *>(a.v) + int64_t(t0) * a.ldv + hv + 8 * c, v);
      else piece.load(static_cast<const T *>(a.k) + int64_t(t0) * a.ldk + hv, ROT ? a.table + int64_t(t0) * a.half : nullptr, a.half, v);
    }
    const int s = a.slots[t0], before = a.slots[max(t0 - 1, 0)], behind = a.slots[min(t0 + 1, a.n - 1)];
    if ((s < -1 || s >= limit) && head == 0 && tid == 0) atomicOr(a.err, kErrPage);
    if (s < 0 || s >= limit) return;
    const int page = s / P, place = s - page * P;
    if (place != 0 && t0 != 0 && before == s - 1) return;  // (a run that starts before)
    if (place + 1 == P || t0 + 1 == a.n || behind != s + 1) {
      if (wave != 0) return;
      const int64_t sc = int64_t(page) * a.Hkv + head;
      float *scale = vh ? a.vs + sc : a.ks + sc;
      const float held = *scale;
      float big = on ? amax8(v, 0.f) : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor(big, o, 64));
      const PageScale ps(big, held, place);
      uint8_t *kd = a.kc + page_base(page, a.Hkv, head, P, hd), *vd = a.vc + page_base(page, a.Hkv, head, P, hd);
      const float kratio = __shfl(ps.ratio, 0, 64), vratio = __shfl(ps.ratio, 32, 64);
      if (kratio != 1.f) rescale_keys<64, 8>(kd, place, hd, kratio, lane);
      if (vratio != 1.f) {
        rescale_values<64, 8>(vd, place, hd, P, vratio, lane);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the new place lies in a piece that was rewritten
      }
      if (on && vh) {
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = v[e] * ps.inv;
        const uint32_t b[2] = {e4m3x4(w), e4m3x4(w + 4)};
#pragma unroll
        for (int e = 0; e < 8; ++e) vd[int64_t(8 * c + e) * P + place] = uint8_t(b[e >> 2] >> (8 * (e & 3)));
      } else if (on) {
        piece.store(kd + int64_t(place) * hd, a.half, v, ps.inv);
      }
      if (c == 0) *scale = ps.now;
      return;
    }
    starts = 1;
  } else {
    // the run starts among this workgroup's tokens (every wave finds the same)
    const int t = t0 + lane;
    bool first = false;
    if (lane < a.per && t < a.n) {
      const int s = a.slots[t];
      if ((s < -1 || s >= limit) && head == 0 && wave == 0) atomicOr(a.err, kErrPage);
      first = s >= 0 && s < limit && (s % P == 0 || t == 0 || a.slots[t - 1] != s - 1);
    }
    starts = __ballot(first);
  }
  while (starts) {
    const int t = t0 + __builtin_ctzll(starts);
    starts &= starts - 1;
    const int slot = a.slots[t], page = slot / P, place = slot - page * P;
    const int64_t sc = int64_t(page) * a.Hkv + head;
    const float held[2] = {a.ks[sc], a.vs[sc]};
    int n = 0;  // tokens of the run
    for (;;) {
      const int i = n + lane;
      const bool in = place + i < P && t + i < a.n && a.slots[min(t + i, a.n - 1)] == slot + i;
      const uint64_t out = ~__ballot(in);
      if (out) {
        n += __builtin_ctzll(out);
        break;
      }
      n += 64;
    }
    const T *kp = static_cast<const T *>(a.k) + int64_t(t) * a.ldk + int64_t(head) * hd;
    const T *vp = static_cast<const T *>(a.v) + int64_t(t) * a.ldv + int64_t(head) * hd;
    const float2 *tab = ROT ? a.table + int64_t(t) * a.half : nullptr;
    uint8_t *kd = a.kc + page_base(page, a.Hkv, head, P, hd), *vd = a.vc + page_base(page, a.Hkv, head, P, hd);

    // A run of at most NT pieces of 4 places and 8 head values (NT 256: 64 tokens of
    // heads of 128) is held in registers, a piece to a thread: loaded once, its values
    // transposed four places at a time (17k tokens, 8 heads of 128: 39 us, against 44
    // with two passes over memory and single bytes).
    const int q0 = place / 4, nq = (place + n - 1) / 4 - q0 + 1;
    const bool held_run = nq * h8 <= NT;
    const int pq = tid / h8, pd = 8 * (tid - pq * h8), pi = 4 * (q0 + pq) - place;  // this thread's piece: first token
    const KeyPiece<DT, ROT> kpiece(pd / 8, a.half);
    const bool mine = held_run && pq < nq;
    Key<DT, ROT> kr[4];
    Raw<DT> vr[4];
    float big[2] = {0.f, 0.f};
    if (mine) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int64_t i = min(max(pi + j, 0), n - 1);  // (places beside the run repeat its tokens, not stored)
        kr[j].load(kpiece, kp + i * a.ldk, tab + (ROT ? i * a.half : 0), a.half);
        vr[j].load(vp + i * a.ldv + pd);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float v[8];
        kr[j].get(v);
        big[0] = amax8(v, big[0]);
        vr[j].get(v);
        big[1] = amax8(v, big[1]);
      }
    }
    for (int c = held_run ? n * h8 : tid; c < n * h8; c += NT) {
      const int i = c / h8, d = 8 * (c - i * h8);
      float v[8];
      KeyPiece<DT, ROT>(d / 8, a.half).load(kp + int64_t(i) * a.ldk, tab + (ROT ? int64_t(i) * a.half : 0), a.half, v);
      big[0] = amax8(v, big[0]);
      ld8<DT>(vp + int64_t(i) * a.ldv + d, v);
      big[1] = amax8(v, big[1]);
    }
    float now[2], inv[2], ratio[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const float m = wave_max(big[x]);
      if (lane == 0) red[x][wave] = m;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      float top = red[x][0];
#pragma unroll
      for (int v = 1; v < NW; ++v) top = fmaxf(top, red[x][v]);
      const PageScale ps(top, held[x], place);
      now[x] = ps.now;
      inv[x] = ps.inv;
      ratio[x] = ps.ratio;
    }
    // the page's earlier tokens in the larger scale
    if (ratio[0] != 1.f) rescale_keys<NT, 1>(kd, place, hd, ratio[0], tid);
    if (ratio[1] != 1.f) rescale_values<NT, 1>(vd, place, hd, P, ratio[1], tid);
    __syncthreads();

    if (held_run) {
      const int rs = 4 * nq + 4;  // LDS bytes of a head value's places
      if (mine) {
        uint32_t w[4][2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float v[8];
          kr[j].get(v);
          if (pi + j >= 0 && pi + j < n) kpiece.store(kd + int64_t(place + pi + j) * hd, a.half, v, inv[0]);
          vr[j].get(v);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= inv[1];
          w[j][0] = e4m3x4(v);
          w[j][1] = e4m3x4(v + 4);
        }
        // four places of each head value to a word
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          uint32_t x = 0;
#pragma unroll
          for (int j = 0; j < 4; ++j) x |= ((w[j][e >> 2] >> (8 * (e & 3))) & 0xffu) << (8 * j);
          *reinterpret_cast<uint32_t *>(&vt[(pd + e) * rs + 4 * pq]) = x;
        }
      }
      __syncthreads();
      const int lo = place, hi = place + n, first = lo & ~15, pieces = (hi + 15) / 16 - lo / 16;
      for (int c = tid; c < hd * pieces; c += NT) {
        const int d = c / pieces, at = first + 16 * (c - d * pieces);
        const uint8_t *src = &vt[d * rs] + (at - 4 * q0);  // (before the row where the run starts inside the piece)
        uint8_t *dst = vd + int64_t(d) * P + at;
        if (at >= lo && at + 16 <= hi) {
          const uint32_t *s4 = reinterpret_cast<const uint32_t *>(src);
          *reinterpret_cast<uint4 *>(dst) = make_uint4(s4[0], s4[1], s4[2], s4[3]);
        } else {
          for (int e = max(lo - at, 0); e < min(hi - at, 16); ++e) dst[e] = src[e];
        }
      }
      __syncthreads();
      if (tid == 0) {
        a.ks[sc] = now[0];
        a.vs[sc] = now[1];
      }
      continue;
    }
    // keys, in their rows
    for (int c = tid; c < n * h8; c += NT) {
      const int i = c / h8, d = 8 * (c - i * h8);
      float v[8];
      const KeyPiece<DT, ROT> piece(d / 8, a.half);
      piece.load(kp + int64_t(i) * a.ldk, tab + (ROT ? int64_t(i) * a.half : 0), a.half, v);
      piece.store(kd + int64_t(place + i) * hd, a.half, v, inv[0]);
    }
    // values, transposed through LDS in tiles of VT places
    for (int c0 = place & ~(VT - 1); c0 < place + n; c0 += VT) {
      const int lo = max(c0, place), hi = min(c0 + VT, place + n);
      for (int c = tid; c < (hi - lo) * h8; c += NT) {
        const int i = c / h8, d = 8 * (c - i * h8);
        float v[8];
        ld8<DT>(vp + int64_t(lo - place + i) * a.ldv + d, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= inv[1];
        const uint32_t w[2] = {e4m3x4(v), e4m3x4(v + 4)};
#pragma unroll
        for (int e = 0; e < 8; ++e) vt[(d + e) * (VT + 4) + lo - c0 + i] = uint8_t(w[e >> 2] >> (8 * (e & 3)));
      }
      __syncthreads();
      const int first = lo & ~15, pieces = ((hi + 15) / 16) - lo / 16;
      for (int c = tid; c < hd * pieces; c += NT) {
        const int d = c / pieces, at = first + 16 * (c - d * pieces);
        const uint32_t *src = reinterpret_cast<const uint32_t *>(&vt[d * (VT + 4) + at - c0]);
        uint8_t *dst = vd + int64_t(d) * P + at;
        if (at >= lo && at + 16 <= hi) {
          *reinterpret_cast<uint4 *>(dst) = make_uint4(src[0], src[1], src[2], src[3]);
        } else {
          for (int e = max(lo - at, 0); e < min(hi - at, 16); ++e) dst[e] = vt[d * (VT + 4) + at - c0 + e];
        }
      }
      __syncthreads();
    }
    if (tid == 0) {
      a.ks[sc] = now[0];
      a.vs[sc] = now[1];
    }
  }
}

}  // namespace

hipError_t page_plan(const PagePlan &p, int *err, hipStream_t st) {
  if (p.B < 1 || p.B > kPlanMaxRequests) return hipErrorInvalidValue;
  const dim3 grid(unsigned(p.B), unsigned(plan_groups(p.B, p.cap)));
  hipLaunchKernelGGL(page_plan_kernel, grid, dim3(256), 0, st, p, err);
  return hipGetLastError();
}

hipError_t kv_store_paged(int dt, const void *k, const void *v, long ldk, long ldv, const int32_t *slots, void *k_cache,
                          void *v_cache, float *k_scale, float *v_scale, int n, int Hkv, int hd, int page, int n_pages, int *err,
                          hipStream_t st, const Rotary *rot) {
  if (n < 1 || n > 1 << 27 || Hkv < 1 || Hkv > 65535) return hipErrorInvalidValue;
  StoreArgs a{k, v, slots, static_cast<uint8_t *>(k_cache), static_cast<uint8_t *>(v_cache), k_scale, v_scale, err, ldk, ldv,
              n, Hkv, hd, page, n_pages, store_tokens(n, Hkv), rot ? reinterpret_cast<const float2 *>(rot->table) : nullptr, rot ? rot->half : 0,
              Rotary{}, 0, 0};
  // Threads for a page's pieces at once where workgroups take many tokens (17k
  // tokens, 8 heads of 128: pages of 128 42 us, 56 with 256 threads; of 256 56, 60);
  // where they take one, most would be idle.
  const int pieces = page / 4 * (hd / 8), nt = a.per == 1 ? 256 : pieces <= 64 ? 64 : pieces <= 128 ? 128 : pieces <= 256 ? 256 : pieces <= 512 ? 512 : 1024;
  dim3 grid(unsigned((n + a.per - 1) / a.per), unsigned(Hkv));
  if (rot && rot->heads) {
    // the queries behind the heads' workgroups: no more rows of them than a grid has left
    a.q = *rot;
    a.q_unit = rotary_unit(dt, a.q);
    // Of many tokens only in 16 bytes a thread: narrower ones need the registers of a
    // launch of their own (17.4k tokens, 32 heads of 128, rotated parts of 120, 100 and
    // 42 by halves: 169, 194 and 253 us, here 205, 246 and 420; 128: here 109).
    if (a.per > 1 && a.q_unit < rotary_most(dt, rot->interleaved)) {
      if (const hipError_t e = rotary(dt, *rot, slots, int64_t(n_pages) * page, st); e != hipSuccess) return e;
      a.q.heads = 0;
    }
  }
  if (a.q.heads) {
    rotary_cut(dt, a.q_unit, nt, a.q);
    a.q_groups = unsigned((n + a.q.tokens - 1) / a.q.tokens);
    grid.y += std::min((a.q_groups + grid.x - 1) / grid.x, std::max(1u, 65535u - grid.y));
  }
#define MH_STORE(DTV, ROT)                                                                                \
  if (a.per == 1)                                                                                         \
    hipLaunchKernelGGL((kv_store_paged_kernel<DTV, 256, ROT, true>), grid, dim3(256), 0, st, a);          \
  else if (nt == 64)                                                                                      \
    hipLaunchKernelGGL((kv_store_paged_kernel<DTV, 64, ROT, false>), grid, dim3(64), 0, st, a);           \
  else if (nt == 128)                                                                                     \
    hipLaunchKernelGGL((kv_store_paged_kernel<DTV, 128, ROT, false>), grid, dim3(128), 0, st, a);         \
  else if (nt == 256)                                                                                     \
    hipLaunchKernelGGL((kv_store_paged_kernel<DTV, 256, ROT, false>), grid, dim3(256), 0, st, a);         \
  else if (nt == 512)                                                                                     \
    hipLaunchKernelGGL((kv_store_paged_kernel<DTV, 512, ROT, false>), grid, dim3(512), 0, st, a);         \
  else                                                                                                    \
    hipLaunchKernelGGL((kv_store_paged_kernel<DTV, 1024, ROT, false>), grid, dim3(1024), 0, st, a);
#define MH_STORE_ROT(DTV)                                                                                 \
  if (!rot) {                                                                                             \
    MH_STORE(DTV, 0)                                                                                      \
  } else if (rot->interleaved) {                                                                          \
    MH_STORE(DTV, 2)                                                                                      \
  } else {                                                                                                \
    MH_STORE(DTV, 1)                                                                                      \
  }
  switch (dt) {
  case F32: MH_STORE_ROT(F32) break;
  case F16: MH_STORE_ROT(F16) break;
  case BF16: MH_STORE_ROT(BF16) break;
  default: return hipErrorInvalidValue;
  }
#undef MH_STORE_ROT
#undef MH_STORE
  return hipGetLastError();
}

}  // namespace mh
