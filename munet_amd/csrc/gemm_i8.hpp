// The epilogue of the 8-bit integer products (gemm_i8*.hip): sums in int32, which
// hold K < 2^17 products of magnitude 2^14 exactly; everything after in 32-bit
// floats, rounded once.
#pragma once

#include "gemm_pipe.hpp"

namespace mh {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// A scale as a fraction and a power of two.  The product of two scales may lie
// outside the floats where the result does not (and below the normal ones, where
// it loses digits): fractions multiply, powers add.
struct Scale {
  float f;
  int e;
  __device__ __forceinline__ Scale() {}
  __device__ __forceinline__ explicit Scale(float s) : f(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};

// Four values of a bias or residual, zeros past the row.
template <int DT>
__device__ __forceinline__ void i8_load4(const typename Store<DT>::T *p, int left, bool quads, float v[4]) {
  if (quads && left >= 4) {
    ld4<DT>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? Store<DT>::dec(p[i]) : 0.f;
  }
}

// Columns n .. n + 3 of row m from their scaled sums, with the bias and the residual.
template <int DT>
__device__ __forceinline__ void i8_store4(const LinearI8 &p, int m, int n, float (&v)[4], const float (&bias)[4], const float (&resid)[4]) {
  typedef typename Store<DT>::T T;
  T *out = static_cast<T *>(p.out) + int64_t(m) * p.ldo + n;
  if (p.bias) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(v[i], bias[i]);
  }
  if (p.act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // (NaN stays)
  } else if (p.act == ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __fmul_rn(v[i], sigmoidf_ref(1.702f * v[i]));
  }
  if (p.resid) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __fadd_rn(v[i], resid[i]);
  }
  if (p.quads && n + 4 <= p.N) {
    if constexpr (DT == BF16) {
      *reinterpret_cast<uint2 *>(out) = pack4_bf16(v);
    } else if constexpr (DT == F16) {
      round4_f16(v);
      *reinterpret_cast<uint2 *>(out) = make_uint2(pack_f16x2_exact(v[0], v[1]), pack_f16x2_exact(v[2], v[3]));
    } else {
      st4<DT>(out, v);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) out[i] = Store<DT>::enc(v[i]);
  }
}

// Whether sums times any two scales of this size, one after the other, stay normal floats or
// overflow where the result does.
__device__ __forceinline__ bool plain_scale(float s) { return s == 0.f || (s >= 0x1p-60f && s <= 0x1p60f); }

// A wave's tile: lane (li, lg) of fragment (i, j) has row 16 i + li, columns
// 16 j + 4 lg .. + 3.  What is the same for several fragments is loaded before
// the first store (a load behind a store waits for it: out might be what is read), a
// row's residual before its stores.  (Whole rows through LDS were slower: 4096 x
// 4096 x 1024 on 256 x 128 tiles 38 us, 34 so.)
template <int DT, typename G, bool PLAIN>
__device__ __forceinline__ void i8_store_as(const LinearI8 &p, int mw, int n0, const i32x4 (&acc)[G::FM][G::FN], const float (&fx)[G::FM],
                                            const float (&fw)[G::FN][4]) {
  typedef typename Store<DT>::T T;
  float bias[G::FN][4], resid[G::FN][4];
  if (p.bias) {
#pragma unroll
    for (int j = 0; j < G::FN; ++j)
      i8_load4<DT>(static_cast<const T *>(p.bias) + n0 + j * 16, p.N - (n0 + j * 16), p.quads, bias[j]);
  }
#pragma unroll
  for (int i = 0; i < G::FM; ++i) {
    const int m = mw + i * 16;
    if (p.resid && m < p.M) {
#pragma unroll
      for (int j = 0; j < G::FN; ++j)
        i8_load4<DT>(static_cast<const T *>(p.resid) + int64_t(m) * p.ldr + n0 + j * 16, p.N - (n0 + j * 16), p.quads, resid[j]);
    }
#pragma unroll
    for (int j = 0; j < G::FN; ++j) {
      const int n = n0 + j * 16;
      float v[4];
      if constexpr (PLAIN) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = __fmul_rn(__fmul_rn(float(acc[i][j][e]), fx[i]), fw[j][e]);
      } else {
        const Scale sx(fx[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const Scale sw(fw[j][e]);
          v[e] = __builtin_amdgcn_ldexpf(__fmul_rn(__fmul_rn(float(acc[i][j][e]), sx.f), sw.f), sx.e + sw.e);
        }
      }
      if (m < p.M && n < p.N) i8_store4<DT>(p, m, n, v, bias[j], resid[j]);
    }
  }
}
// Scales of ordinary size multiply as they are, others as fractions and powers of two: the
// same bits where both can.  Roundings are explicit: a row's results do not
// depend on the kernel.
template <int DT, typename G>
__device__ __forceinline__ void i8_store(const LinearI8 &p, const G &g, int m0, int n0, const i32x4 (&acc)[G::FM][G::FN]) {
  const int mw = m0 + g.wm * G::WTM + g.li, nw = n0 + g.wn * G::WTN + 4 * g.lg;
  float fx[G::FM], fw[G::FN][4];
  bool plain = true;
#pragma unroll
  for (int i = 0; i < G::FM; ++i) fx[i] = p.sx[min(mw + i * 16, p.M - 1)];
#pragma unroll
  for (int j = 0; j < G::FN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) fw[j][e] = p.sw[min(nw + j * 16 + e, p.N - 1)];
#pragma unroll
  for (int i = 0; i < G::FM; ++i) plain &= plain_scale(fx[i]);
#pragma unroll
  for (int j = 0; j < G::FN; ++j)
#pragma unroll
    for (int e = 0; e < 4; ++e) plain &= plain_scale(fw[j][e]);
  if (__all(plain)) i8_store_as<DT, G, true>(p, mw, nw, acc, fx, fw);
  else i8_store_as<DT, G, false>(p, mw, nw, acc, fx, fw);
}

}  // namespace
}  // namespace mh
