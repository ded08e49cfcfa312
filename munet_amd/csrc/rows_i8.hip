// Rows of floating-point values as 8-bit integers with a scale each, and back.
#include <algorithm>

#include "mh_common.hpp"
#include "mh_kernels.hpp"

namespace mh {
namespace {

// The least magnitude that a row is measured by: its 127th part is a normal float.
constexpr float kLeastMax = 0x1.fcp-120f;  // 127 * 2^-126

// Bits of a row's largest magnitude -> what the row is measured by; NaN where the
// row has a value that is not finite.
__device__ __forceinline__ float row_measure(uint32_t top) {
  return top >= 0x7f800000u ? __builtin_nanf("") : fmaxf(__uint_as_float(top), kLeastMax);
}

// The whole number nearest to 127 x / a, ties to even, for |x| <= a.  inv is
// 127 / a, rounded: t is within 127 * 2^-23 of the quotient, so that only
// quotients that near to a half are looked at again, where 254 |x| and
// (2 h + 1) a, products of 24 and 8 bits, are exact in 64.
__device__ __forceinline__ int nearest_i8(float x, float a, float inv) {
  const float t = __fmul_rn(__builtin_fabsf(x), inv), h = __builtin_floorf(t);
  float q = __builtin_rintf(t);
  if (__builtin_fabsf(t - h - 0.5f) < 3e-5f) {
    const double d = 254.0 * double(__builtin_fabsf(x)) - (2.0 * double(h) + 1.0) * double(a);
    q = d > 0 ? h + 1.f : d < 0 ? h : 2.f * __builtin_rintf(0.5f * h + 0.25f);
  }
  return int(__builtin_copysignf(q, x));
}

template <int DT>
__global__ void __launch_bounds__(256) quantize_rows_kernel(QuantRows p) {
  typedef typename Store<DT>::T T;
  __shared__ uint32_t red[4];
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const T *x = static_cast<const T *>(p.x) + r * p.ldx;
    uint32_t top = 0;
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) top = max(top, __float_as_uint(Store<DT>::dec(x[c])) & 0x7fffffffu);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, uint32_t(__shfl_xor(int(top), o, 64)));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
    __syncthreads();
    const float a = row_measure(max(max(red[0], red[1]), max(red[2], red[3]))), inv = 127.f / a;
    __syncthreads();
    int8_t *q = p.q + r * p.ldq;
    for (int64_t c = threadIdx.x; c < p.cols; c += 256) q[c] = a != a ? 0 : int8_t(nearest_i8(Store<DT>::dec(x[c]), a, inv));
    if (threadIdx.x == 0) p.scale[r] = a / 127.f;
  }
}

template <int DT>
__global__ void __launch_bounds__(256) dequantize_rows_kernel(QuantRows p) {
  typedef typename Store<DT>::T T;
  for (int64_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
    const float s = p.scale[r];
    for (int64_t c = threadIdx.x; c < p.cols; c += 256)
      (static_cast<T *>(p.out) + r * p.ldx)[c] = Store<DT>::enc(float(p.q[r * p.ldq + c]) * s);
  }
}

}  // namespace

hipError_t quantize_rows(int dt, const QuantRows &p, hipStream_t st) {
  const unsigned grid = unsigned(std::min(p.rows, 1 << 20));
  switch (dt) {
  case F32: hipLaunchKernelGGL(quantize_rows_kernel<F32>, dim3(grid), dim3(256), 0, st, p); break;
  case F16: hipLaunchKernelGGL(quantize_rows_kernel<F16>, dim3(grid), dim3(256), 0, st, p); break;
  case BF16: hipLaunchKernelGGL(quantize_rows_kernel<BF16>, dim3(grid), dim3(256), 0, st, p); break;
  default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t dequantize_rows(int dt, const QuantRows &p, hipStream_t st) {
  const unsigned grid = unsigned(std::min(p.rows, 1 << 20));
  switch (dt) {
  case F32: hipLaunchKernelGGL(dequantize_rows_kernel<F32>, dim3(grid), dim3(256), 0, st, p); break;
  case F16: hipLaunchKernelGGL(dequantize_rows_kernel<F16>, dim3(grid), dim3(256), 0, st, p); break;
  case BF16: hipLaunchKernelGGL(dequantize_rows_kernel<BF16>, dim3(grid), dim3(256), 0, st, p); break;
  default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mh
