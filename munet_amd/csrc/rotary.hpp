// Rotation of a head's pairs by a table's angles, shared by rotary.hip and the
// rotated form of the paged cache's store (paged_cache.hip).
//
// Pair j of a head (j < half) is (x_j, x_{j + half}), or (x_{2j}, x_{2j + 1}) where
// neighbours are paired; table row t holds (c, s) of each pair, and the pair
// becomes (a c - b s, a s + b c).  The rest of the head stays.
#pragma once

#include <type_traits>

#include "gemm_common.hpp"
#include "mh_common.hpp"
#include "mh_kernels.hpp"

namespace mh {
namespace {

// (one product fused, the other not: the same bits wherever this is inlined, so
// that a key rotated on its way into the cache is the key that rotary() gives)
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
#pragma clang fp contract(off)
  const float p = b * s, q = b * c, x = __builtin_fmaf(a, c, -p), y = __builtin_fmaf(a, s, q);
  a = x;
  b = y;
}

// N consecutive values.  N of 16 bytes: one load or store aligned to it; fewer: aligned
// to the type alone (a rotated part of 100 puts partners 100 bytes apart).
template <int DT, int N> __device__ __forceinline__ void ldv(const typename Store<DT>::T *p, float v[N]) {
  typedef typename Store<DT>::T T;
  if constexpr (DT == F32 && N == 4) ld4<F32>(p, v);
  else if constexpr (N == 8) dec8<DT>(*reinterpret_cast<const uint4 *>(p), v);
  else {
    struct __attribute__((packed, aligned(sizeof(T)))) Few { T v[N]; };
    const Few x = *reinterpret_cast<const Few *>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Store<DT>::dec(x.v[i]);
  }
}
template <int DT, int N> __device__ __forceinline__ void stv(typename Store<DT>::T *p, float v[N]) {
  typedef typename Store<DT>::T T;
  if constexpr (DT == F32 && N == 4) st4<F32>(p, v);
  else if constexpr (N == 8) {
    if constexpr (DT == F16) {
      round4_f16(v);
      round4_f16(v + 4);
    }
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = DT == F16 ? pack_f16x2_exact(v[2 * i], v[2 * i + 1]) : pack_bf16x2(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  } else {
    struct __attribute__((packed, aligned(sizeof(T)))) Few { T v[N]; };
    Few x;
#pragma unroll
    for (int i = 0; i < N; ++i) x.v[i] = Store<DT>::enc(v[i]);
    *reinterpret_cast<Few *>(p) = x;
  }
}

// Two pairs' angles (rows of an odd number of pairs start at 8 bytes).
__device__ __forceinline__ float4 angles2(const float2 *t) {
  struct __attribute__((packed, aligned(8))) Two { float4 v; };
  return reinterpret_cast<const Two *>(t)->v;
}

// Pairs a thread: 16 bytes of each load at most; and values of a piece behind the pairs.
constexpr int rotary_most(int dt, bool interleaved) { return (dt == F32 ? 4 : 8) / (interleaved ? 2 : 1); }
constexpr int rotary_tail(int dt, int unit, bool interleaved) { return unit == rotary_most(dt, interleaved) ? (dt == F32 ? 4 : 8) : unit; }

// One workgroup of NT threads at tokens first .. first + p.tokens - 1.  A thread
// takes U pairs (or, behind the pairs, as many values) of every p.lanes-th head:
// their angles are loaded once, and HB heads' values are in flight at a time.
// Where `slots` is given, tokens without one in 0 .. limit - 1 are left alone.
template <int DT, int U, bool INTERLEAVED, int NT, int HB = 4>
__device__ __forceinline__ void rotate_tokens(const Rotary &p, int64_t first, const int32_t *slots, int64_t limit) {
  typedef typename Store<DT>::T T;
  const int pairs = p.half / U, units = p.units, cols = min(units, NT);
  const int lt = threadIdx.x / (cols * p.lanes), r = threadIdx.x - lt * (cols * p.lanes);
  const int64_t t = first + lt;
  if (lt >= p.tokens || t >= p.n) return;
  if (slots) {
    const int s = slots[t];
    if (s < 0 || s >= limit) return;
  }
  const int lane = r / cols;
  const T *x = static_cast<const T *>(p.x) + t * p.ldx;
  T *out = static_cast<T *>(p.out) + t * p.ldo;
  for (int u = r - lane * cols; u < units; u += cols) {
    if (u < pairs) {
      const float2 *tab = reinterpret_cast<const float2 *>(p.table) + t * p.half + u * U;
      float c[U], s[U];
      if constexpr (U % 2 == 0) {
#pragma unroll
        for (int i = 0; i < U; i += 2) {
          const float4 cs = angles2(tab + i);
          c[i] = cs.x;
          s[i] = p.inverse ? -cs.y : cs.y;
          c[i + 1] = cs.z;
          s[i + 1] = p.inverse ? -cs.w : cs.w;
        }
      } else {
        c[0] = tab->x;
        s[0] = p.inverse ? -tab->y : tab->y;
      }
      const int ia = INTERLEAVED ? 2 * U * u : U * u, ib = INTERLEAVED ? ia + U : ia + p.half;
      for (int h = lane; h < p.heads; h += HB * p.lanes) {
        float a[HB][U], b[HB][U];
#pragma unroll
        for (int k = 0; k < HB; ++k) {
          const int hk = h + k * p.lanes;
          if (hk < p.heads) {
            const T *xh = x + hk * p.hd;
            if constexpr (INTERLEAVED) {
              float v[2 * U];
              ldv<DT, 2 * U>(xh + ia, v);
#pragma unroll
              for (int i = 0; i < U; ++i) {
                a[k][i] = v[2 * i];
                b[k][i] = v[2 * i + 1];
              }
            } else {
              ldv<DT, U>(xh + ia, a[k]);
              ldv<DT, U>(xh + ib, b[k]);
            }
          }
        }
#pragma unroll
        for (int k = 0; k < HB; ++k) {
          const int hk = h + k * p.lanes;
          if (hk < p.heads) {
            T *o = out + hk * p.hd;
#pragma unroll
            for (int i = 0; i < U; ++i) turn(a[k][i], b[k][i], c[i], s[i]);
            if constexpr (INTERLEAVED) {
              float v[2 * U];
#pragma unroll
              for (int i = 0; i < U; ++i) {
                v[2 * i] = a[k][i];
                v[2 * i + 1] = b[k][i];
              }
              stv<DT, 2 * U>(o + ia, v);
            } else {
              stv<DT, U>(o + ia, a[k]);
              stv<DT, U>(o + ib, b[k]);
            }
          }
        }
      }
    } else {
      // behind the pairs: as they are (units counts these where out is not x), as many values as a thread's pairs
      constexpr int W = rotary_tail(DT, U, INTERLEAVED);
      struct __attribute__((packed, aligned(sizeof(T)))) Piece { T v[W]; };
      const int at = 2 * p.half + (u - pairs) * W;
      for (int h = lane; h < p.heads; h += p.lanes)
        *reinterpret_cast<Piece *>(out + h * p.hd + at) = *reinterpret_cast<const Piece *>(x + h * p.hd + at);
    }
  }
}

// Four consecutive values, aligned to the type alone (a rotated part of 100 puts
// partners 100 bytes apart).
template <int DT> __device__ __forceinline__ void ldu4(const typename Store<DT>::T *p, float v[4]) {
  struct __attribute__((packed, aligned(4))) F4 { f32x4 v; };
  struct __attribute__((packed, aligned(2))) H4 { uint2 v; };
  if constexpr (DT == F32) {
    const f32x4 x = reinterpret_cast<const F4 *>(p)->v;
    v[0] = x[0]; v[1] = x[1]; v[2] = x[2]; v[3] = x[3];
  } else {
    const uint2 x = reinterpret_cast<const H4 *>(p)->v;
    v[0] = Store<DT>::dec(uint16_t(x.x)); v[1] = Store<DT>::dec(uint16_t(x.x >> 16));
    v[2] = Store<DT>::dec(uint16_t(x.y)); v[3] = Store<DT>::dec(uint16_t(x.y >> 16));
  }
}

// How many pairs a thread takes: 16 bytes of each load, where sizes, spacing and
// addresses allow it, else the largest power of two below that divides a head's parts.
// 16500 tokens, 40 heads of 128 bf16 values, rotated parts of 128, 120, 100 and 42 by
// halves: 69, 107, 115 and 185 us (one pair a thread wherever 16 bytes do not fit:
// 175 and more).
inline int rotary_unit(int dt, const Rotary &p) {
  const int64_t es = int64_t(dt_size(dt)), e = 16 / es;
  const int most = rotary_most(dt, p.interleaved), tail = p.x == p.out ? 0 : p.hd - 2 * p.half;
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out);
  if (p.half % most == 0 && (2 * p.half) % e == 0 && p.hd % e == 0 && at % 16 == 0 && (p.n == 1 || (p.ldx % e == 0 && p.ldo % e == 0))) return most;
  int u = most / 2;
  while (u > 1 && (p.half % u || tail % u)) u /= 2;
  return u;
}

// f with the unit and the layout as types.
template <int DT, bool INTERLEAVED, int U = rotary_most(DT, INTERLEAVED), typename F>
__host__ __device__ __forceinline__ void rotary_unit_as(int unit, F &&f) {
  if constexpr (U == 1) f(std::integral_constant<int, 1>(), std::integral_constant<bool, INTERLEAVED>());
  else if (unit == U) f(std::integral_constant<int, U>(), std::integral_constant<bool, INTERLEAVED>());
  else rotary_unit_as<DT, INTERLEAVED, U / 2>(unit, f);
}
template <int DT, typename F> inline void rotary_units(bool interleaved, int unit, F &&f) {
  if (interleaved) rotary_unit_as<DT, true>(unit, f);
  else rotary_unit_as<DT, false>(unit, f);
}

// The cut for workgroups of NT threads: units a head, threads that share a unit's
// heads (so that each takes several heads where there are tokens enough), tokens.
inline void rotary_cut(int dt, int unit, int threads, Rotary &p) {
  const int w = rotary_tail(dt, unit, p.interleaved);
  p.units = p.half / unit + (p.x == p.out ? 0 : (p.hd - 2 * p.half) / w);
  const int cols = p.units < threads ? p.units : threads, most = threads / cols;
  const int64_t all = int64_t(p.n) * cols * p.heads;
  const int per = all >= (int64_t(1) << 20) ? 4 : 1;  // heads a thread
  int lanes = (p.heads + per - 1) / per;
  p.lanes = lanes < most ? lanes : most;
  p.tokens = threads / (cols * p.lanes);
}

}  // namespace
}  // namespace mh
