// Rotation of a head's pairs by a table's angles, shared by rotary.hip and the
// rotated form of the paged cache's store (paged_cache.hip).
//
// Pair j of a head (j < half) is (x_j, x_{j + half}), or (x_{2j}, x_{2j + 1}) where
// neighbours are paired; table row t holds (c, s) of each pair, and the pair
// becomes (a c - b s, a s + b c).  The rest of the head stays.
#pragma once

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

// N consecutive values (one load or store of up to 16 bytes, aligned to its size).
template <int DT, int N> __device__ __forceinline__ void ldv(const typename Store<DT>::T *p, float v[N]) {
  if constexpr (N == 1) v[0] = Store<DT>::dec(*p);
  else if constexpr (DT == F32 && N == 2) {
    const float2 x = *reinterpret_cast<const float2 *>(p);
    v[0] = x.x;
    v[1] = x.y;
  } else if constexpr (N == 4) ld4<DT>(p, v);
  else {
    static_assert(DT != F32 && N == 8, "16 bytes at most");
    dec8<DT>(*reinterpret_cast<const uint4 *>(p), v);
  }
}
template <int DT, int N> __device__ __forceinline__ void stv(typename Store<DT>::T *p, float v[N]) {
  if constexpr (N == 1) *p = Store<DT>::enc(v[0]);
  else if constexpr (DT == F32 && N == 2) *reinterpret_cast<float2 *>(p) = make_float2(v[0], v[1]);
  else if constexpr (DT == F32) st4<DT>(p, v);
  else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      if constexpr (DT == F16) round4_f16(v + i);
    }
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i)
      w[i] = DT == F16 ? pack_f16x2_exact(v[2 * i], v[2 * i + 1]) : pack_bf16x2(v[2 * i], v[2 * i + 1]);
    if constexpr (N == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
  }
}

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
          const float4 cs = reinterpret_cast<const float4 *>(tab)[i / 2];
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
            if constexpr (INTERLEAVED && U > 1) {
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
            if constexpr (INTERLEAVED && U > 1) {
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
      // behind the pairs: as they are (units counts these where out is not x)
      constexpr int W = U == 1 ? 1 : 16 / int(sizeof(T));
      struct __attribute__((aligned(W * sizeof(T)))) Piece { T v[W]; };
      const int at = 2 * p.half + (u - pairs) * W;
      for (int h = lane; h < p.heads; h += p.lanes)
        *reinterpret_cast<Piece *>(out + h * p.hd + at) = *reinterpret_cast<const Piece *>(x + h * p.hd + at);
    }
  }
}

// Eight rotated values of a head from d on (a multiple of 8; the head 16-byte
// aligned).
template <int DT, bool INTERLEAVED>
__device__ __forceinline__ void turned8(const typename Store<DT>::T *head, const float2 *tab, int half, int d, float v[8]) {
  constexpr int N = DT == F32 ? 4 : 8;
#pragma unroll
  for (int e = 0; e < 8; e += N) ldv<DT, N>(head + d + e, v + e);
  if (d >= 2 * half) return;
  if constexpr (INTERLEAVED) {
    if (half % 4 == 0) {
      const float4 *t = reinterpret_cast<const float4 *>(tab + d / 2);
      const float4 x = t[0], y = t[1];
      turn(v[0], v[1], x.x, x.y);
      turn(v[2], v[3], x.z, x.w);
      turn(v[4], v[5], y.x, y.y);
      turn(v[6], v[7], y.z, y.w);
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int j = (d + e) >> 1;
      if (j < half) turn(v[e], v[e + 1], tab[j].x, tab[j].y);
    }
  } else {
    if (half % 8 == 0) {  // the partners are eight values half a rotated part away
      float w[8];
      const bool low = d < half;
#pragma unroll
      for (int e = 0; e < 8; e += N) ldv<DT, N>(head + (low ? d + half : d - half) + e, w + e);
      const float4 *t = reinterpret_cast<const float4 *>(tab + (low ? d : d - half));
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const float4 cs = t[e / 2];
        float a0 = low ? v[e] : w[e], b0 = low ? w[e] : v[e], a1 = low ? v[e + 1] : w[e + 1], b1 = low ? w[e + 1] : v[e + 1];
        turn(a0, b0, cs.x, cs.y);
        turn(a1, b1, cs.z, cs.w);
        v[e] = low ? a0 : b0;
        v[e + 1] = low ? a1 : b1;
      }
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int i = d + e;
      if (i < half) {
        float b = Store<DT>::dec(head[i + half]);
        turn(v[e], b, tab[i].x, tab[i].y);
      } else if (i < 2 * half) {
        float a = Store<DT>::dec(head[i - half]);
        turn(a, v[e], tab[i - half].x, tab[i - half].y);
      }
    }
  }
}

// How many pairs a thread takes: 16 bytes of each load, where sizes, spacing and
// addresses allow it, else one.
inline int rotary_unit(int dt, const Rotary &p) {
  const int64_t es = int64_t(dt_size(dt)), e = 16 / es;
  const int u = int(p.interleaved ? e / 2 : e);
  const uintptr_t at = reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.out);
  const bool whole = p.half % u == 0 && (2 * p.half) % e == 0 && p.hd % e == 0 && at % 16 == 0 && (p.n == 1 || (p.ldx % e == 0 && p.ldo % e == 0));
  return whole ? u : 1;
}
// The cut for workgroups of NT threads: units a head, threads that share a unit's
// heads (so that each takes several heads where there are tokens enough), tokens.
inline void rotary_cut(int dt, int unit, int threads, Rotary &p) {
  const int w = unit == 1 ? 1 : int(16 / dt_size(dt));
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
