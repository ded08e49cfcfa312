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

// Output columns n .. n + 3 of row m from their sums.
template <int DT>
__device__ __forceinline__ void i8_store4(const LinearI8 &p, int m, int n, i32x4 acc, Scale sx, const Scale (&sw)[4]) {
  typedef typename Store<DT>::T T;
  const T *bias = static_cast<const T *>(p.bias);
  const T *resid = p.resid ? static_cast<const T *>(p.resid) + int64_t(m) * p.ldr + n : nullptr;
  T *out = static_cast<T *>(p.out) + int64_t(m) * p.ldo + n;
  float v[4], r[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_amdgcn_ldexpf(float(acc[i]) * sx.f * sw[i].f, sx.e + sw[i].e);
  const bool quad = p.quads && n + 4 <= p.N;
  if (bias) {
    if (quad) ld4<DT>(bias + n, r);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = n + i < p.N ? Store<DT>::dec(bias[n + i]) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += r[i];
  }
  if (p.act == ACT_RELU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];  // (NaN stays)
  } else if (p.act == ACT_GELU) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] *= sigmoidf_ref(1.702f * v[i]);
  }
  if (resid) {
    if (quad) ld4<DT>(resid, r);
    else
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = n + i < p.N ? Store<DT>::dec(resid[i]) : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += r[i];
  }
  if (quad) {
    if constexpr (DT == BF16) *reinterpret_cast<uint2 *>(out) = pack4_bf16(v);
    else if constexpr (DT == F16) {
      round4_f16(v);
      *reinterpret_cast<uint2 *>(out) = make_uint2(pack_f16x2_exact(v[0], v[1]), pack_f16x2_exact(v[2], v[3]));
    } else st4<DT>(out, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < p.N) out[i] = Store<DT>::enc(v[i]);
  }
}

}  // namespace
}  // namespace mh
