// Rotation of a head's pairs by a table's angles, shared by rotary.hip and the
// rotated form of the paged cache's store (paged_cache.hip).
//
// Pair j of a head (j < half) is (x_j, x_{j + half}), or (x_{2j}, x_{2j + 1}) where
// neighbours are paired; table row t holds (c, s) of each pair, and the pair
// becomes (a c - b s, a s + b c).  The rest of the head stays.
#pragma once

#include "mh_common.hpp"
#include "mh_kernels.hpp"

namespace mh {

// (explicit fma and mul: the same bits wherever this is inlined, so that a key
// rotated on its way into the cache is the key that rotary() gives)
__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
  const float x = __fmaf_rn(a, c, -__fmul_rn(b, s)), y = __fmaf_rn(a, s, __fmul_rn(b, c));
  a = x;
  b = y;
}

// Token t's heads by one workgroup of NT threads: a thread a pair, or a value
// behind the pairs.
template <int DT, int NT> __device__ __forceinline__ void rotate_token(const Rotary &p, int64_t t) {
  typedef typename Store<DT>::T T;
  const T *x = static_cast<const T *>(p.x) + t * p.ldx;
  T *out = static_cast<T *>(p.out) + t * p.ldo;
  const float2 *tab = reinterpret_cast<const float2 *>(p.table) + t * p.half;
  const int units = p.hd - p.half, per = units * p.heads;
  for (int i = threadIdx.x; i < per; i += NT) {
    const int h = i / units, u = i - h * units, at = h * p.hd;
    if (u < p.half) {
      const float2 cs = tab[u];
      const int ia = at + (p.interleaved ? 2 * u : u), ib = at + (p.interleaved ? 2 * u + 1 : u + p.half);
      float a = Store<DT>::dec(x[ia]), b = Store<DT>::dec(x[ib]);
      turn(a, b, cs.x, p.inverse ? -cs.y : cs.y);
      out[ia] = Store<DT>::enc(a);
      out[ib] = Store<DT>::enc(b);
    } else if (p.out != p.x) {
      out[at + u + p.half] = x[at + u + p.half];
    }
  }
}

// Eight rotated values of a head from d on (a multiple of 8).
template <int DT, bool INTERLEAVED>
__device__ __forceinline__ void turned8(const typename Store<DT>::T *head, const float2 *tab, int half, int d, float v[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = Store<DT>::dec(head[d + e]);
  if constexpr (INTERLEAVED) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const int j = (d + e) >> 1;
      if (j < half) turn(v[e], v[e + 1], tab[j].x, tab[j].y);
    }
  } else {
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

}  // namespace mh
