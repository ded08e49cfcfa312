// Rows of floating-point values as 8-bit integers with a scale each, and back.
//
// Both are bound by memory: a row is read once and held in registers while its
// largest magnitude is found.  8192 rows of 8192 bf16 values: 40 us, 5.0 TB/s, which is
// what a large copy reaches; back 30 us (read from the last-level cache).  Rows past
// 32768 values are read twice: 2048 of 40000 values 69 us, 3.6 TB/s of what is read once.
#include <algorithm>

#include "gemm_common.hpp"
#include "mh_common.hpp"
#include "mh_kernels.hpp"

namespace mh {
namespace {

// The least magnitude that a row is measured by: its 127th part is a normal float.
constexpr float kLeastMax = 0x1.fcp-120f;  // 127 * 2^-126

// Eight values of a row as they lie.  Rows start anywhere: loads and stores of
// 16 bytes are not aligned; the values of a row's last piece go one by one, and
// those behind the row are zeros.
template <typename T> struct Eight {
  struct __attribute__((packed)) Any { T v[8]; };
  T v[8];
  __device__ __forceinline__ void load(const T *p, int64_t left) {
    if (left >= 8) {
      const Any a = *reinterpret_cast<const Any *>(p);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = a.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = i < left ? p[i] : T(0);
    }
  }
  __device__ __forceinline__ void store(T *p, int64_t left) const {
    if (left >= 8) {
      Any a;
#pragma unroll
      for (int i = 0; i < 8; ++i) a.v[i] = v[i];
      *reinterpret_cast<Any *>(p) = a;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = v[i];
    }
  }
};
struct __attribute__((packed)) Bytes8 { uint32_t a, b; };

// The whole number nearest to 127 x / a, ties to even, where the quotient lies next
// to a half: 254 |x| and (2 h + 1) a, products of 24 and 8 bits, are exact in 64.
__device__ __noinline__ float nearest_exact(float x, float a, float inv) {
  const float h = __builtin_floorf(__builtin_fabsf(x * inv));
  const double d = 254.0 * double(__builtin_fabsf(x)) - (2.0 * double(h) + 1.0) * double(a);
  const float q = d > 0 ? h + 1.f : d < 0 ? h : 2.f * __builtin_rintf(0.5f * h + 0.25f);
  return __builtin_copysignf(q, x);
}

// Eight values as bytes.  x inv + 1.5 2^23 is rounded to a whole number by the sum,
// whose low byte is the result.  inv = 127 / a is rounded, so that the quotient is
// off by up to 127 2^-24: one that near to a half is looked at again.
template <int DT> __device__ __forceinline__ Bytes8 to_bytes(const Eight<typename Store<DT>::T> &e, float a, float inv) {
  constexpr float kWhole = 12582912.f;
  uint32_t w[8];
  float far = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float x = Store<DT>::dec(e.v[i]), r = __builtin_fmaf(x, inv, kWhole);
    far = fmaxf(far, __builtin_fabsf(__builtin_fmaf(x, inv, kWhole - r)));
    w[i] = __float_as_uint(r);
  }
  if (far > 0.49997f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = Store<DT>::dec(e.v[i]);
      if (__builtin_fabsf(__builtin_fmaf(x, inv, kWhole - __uint_as_float(w[i]))) > 0.49997f)
        w[i] = __float_as_uint(nearest_exact(x, a, inv) + kWhole);
    }
  }
  auto four = [](uint32_t a, uint32_t b, uint32_t c, uint32_t d) {  // their low bytes
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400u), __builtin_amdgcn_perm(b, a, 0x0c0c0400u), 0x05040100u);
  };
  return Bytes8{four(w[0], w[1], w[2], w[3]), four(w[4], w[5], w[6], w[7])};
}
__device__ __forceinline__ void put_bytes(int8_t *p, Bytes8 b, int64_t left) {
  if (left >= 8) {
    *reinterpret_cast<Bytes8 *>(p) = b;
  } else {
    for (int i = 0; i < left; ++i) p[i] = int8_t((i < 4 ? b.a : b.b) >> (8 * (i & 3)));
  }
}

// NT threads a row, CH pieces a thread where the row is held (HELD; else it is
// read twice); a workgroup of at least 256 threads takes several short rows.
template <int DT, int NT, int CH, bool HELD>
__global__ void __launch_bounds__(NT < 256 ? 256 : NT) quantize_rows_kernel(QuantRows p) {
  typedef typename Store<DT>::T T;
  constexpr int ROWS = NT < 256 ? 256 / NT : 1, NW = NT / 64;
  static_assert(NT % 64 == 0, "whole waves");
  __shared__ uint32_t red[NT < 256 ? 1 : NW];
  const int tid = threadIdx.x % NT;
  for (int64_t r = int64_t(blockIdx.x) * ROWS + threadIdx.x / NT; r < p.rows; r += int64_t(gridDim.x) * ROWS) {
    const T *x = static_cast<const T *>(p.x) + r * p.ldx;
    Eight<T> e[CH];
    // the largest magnitude, by its bits
    typedef T Pair __attribute__((ext_vector_type(2)));
    Pair big = {0, 0};
    uint32_t top = 0;
    auto look = [&](const Eight<T> &v) {
      if constexpr (DT == F32) {
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v.v[i]) & 0x7fffffffu);
      } else {
#pragma unroll
        for (int i = 0; i < 8; i += 2) big = __builtin_elementwise_max(big, Pair{v.v[i], v.v[i + 1]} & Pair{0x7fff, 0x7fff});
      }
    };
    if constexpr (HELD) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int c = 8 * (tid + NT * k);
        e[k].load(x + c, p.cols - c);
      }
#pragma unroll
      for (int k = 0; k < CH; ++k) look(e[k]);
    } else {
      for (int64_t c = 8 * tid; c < p.cols; c += 8 * NT) {
        e[0].load(x + c, p.cols - c);
        look(e[0]);
      }
    }
    if constexpr (DT != F32) top = __float_as_uint(Store<DT>::dec(max(big[0], big[1])));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, uint32_t(__shfl_xor(int(top), o, 64)));
    if constexpr (NW > 1) {
      if ((tid & 63) == 0) red[tid >> 6] = top;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < NW; ++w) top = max(top, red[w]);
      __syncthreads();
    }
    // a value that is not finite: the row's scale is NaN, its whole numbers 0
    const bool fine = top < 0x7f800000u;
    const float a = fine ? fmaxf(__uint_as_float(top), kLeastMax) : __builtin_nanf(""), inv = 127.f / a;
    int8_t *q = p.q + r * p.ldq;
    if constexpr (HELD) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int c = 8 * (tid + NT * k);
        if (c < p.cols) put_bytes(q + c, fine ? to_bytes<DT>(e[k], a, inv) : Bytes8{0, 0}, p.cols - c);
      }
    } else {
      for (int64_t c = 8 * tid; c < p.cols; c += 8 * NT) {
        e[0].load(x + c, p.cols - c);
        put_bytes(q + c, fine ? to_bytes<DT>(e[0], a, inv) : Bytes8{0, 0}, p.cols - c);
      }
    }
    if (tid == 0) p.scale[r] = a / 127.f;
  }
}

template <int DT> __global__ void __launch_bounds__(256) dequantize_rows_kernel(QuantRows p, int threads) {
  typedef typename Store<DT>::T T;
  // `threads` a row: short rows share a workgroup
  const int rows = 256 / threads, lr = threadIdx.x / threads, tid = threadIdx.x - lr * threads;
  if (lr >= rows) return;
  for (int64_t r = int64_t(blockIdx.x) * rows + lr; r < p.rows; r += int64_t(gridDim.x) * rows) {
    const float s = p.scale[r];
    const int8_t *q = p.q + r * p.ldq;
    T *out = static_cast<T *>(p.out) + r * p.ldx;
    for (int64_t c = 8 * tid; c < p.cols; c += 8 * threads) {
      Eight<int8_t> b;
      b.load(q + c, p.cols - c);
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = float(b.v[i]) * s;
      Eight<T> e;
      if constexpr (DT == BF16) {
#pragma unroll
        for (int i = 0; i < 8; i += 2) {
          const uint32_t w = pack_bf16x2(v[i], v[i + 1]);
          e.v[i] = uint16_t(w);
          e.v[i + 1] = uint16_t(w >> 16);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) e.v[i] = Store<DT>::enc(v[i]);
      }
      e.store(out + c, p.cols - c);
    }
  }
}

template <int DT, int NT, int CH, bool HELD = true> hipError_t launch(const QuantRows &p, hipStream_t st) {
  constexpr int ROWS = NT < 256 ? 256 / NT : 1;
  const unsigned grid = unsigned(std::min((int64_t(p.rows) + ROWS - 1) / ROWS, int64_t(1) << 21));
  hipLaunchKernelGGL((quantize_rows_kernel<DT, NT, CH, HELD>), dim3(grid), dim3(NT < 256 ? 256 : NT), 0, st, p);
  return hipGetLastError();
}

// Threads a row: one piece of eight values each (up to 2048 values: 2048 rows 6.0 us,
// 8192 15.1; a wave with four pieces 9.2 and 17.4), longer rows only while there are
// few of them (one piece | four: 64 x 4096 3.8 | 5.0 us, 512 x 4096 6.0 | 6.5, 1024 x
// 4096 9.1 | 7.4, 8192 x 4096 52 | 28).
template <int DT> hipError_t quantize(const QuantRows &p, hipStream_t st) {
  const int pieces = (p.cols - 1) / 8 + 1;
  if (pieces <= 64) return launch<DT, 64, 1>(p, st);
  if (pieces <= 256) return launch<DT, 256, 1>(p, st);
  if (pieces <= 1024 && p.rows <= 512) return launch<DT, 1024, 1>(p, st);
  if (pieces <= 1024) return launch<DT, 256, 4>(p, st);
  if (pieces <= 4096) return launch<DT, 1024, 4>(p, st);
  return launch<DT, 1024, 1, false>(p, st);
}

template <int DT> hipError_t dequantize(const QuantRows &p, hipStream_t st) {
  const int threads = std::min(256, (p.cols - 1) / 8 + 1), rows = 256 / threads;
  const unsigned grid = unsigned(std::min((int64_t(p.rows) + rows - 1) / rows, int64_t(1) << 22));
  hipLaunchKernelGGL(dequantize_rows_kernel<DT>, dim3(grid), dim3(256), 0, st, p, threads);
  return hipGetLastError();
}

}  // namespace

hipError_t quantize_rows(int dt, const QuantRows &p, hipStream_t st) {
  switch (dt) {
  case F32: return quantize<F32>(p, st);
  case F16: return quantize<F16>(p, st);
  case BF16: return quantize<BF16>(p, st);
  default: return hipErrorInvalidValue;
  }
}

hipError_t dequantize_rows(int dt, const QuantRows &p, hipStream_t st) {
  switch (dt) {
  case F32: return dequantize<F32>(p, st);
  case F16: return dequantize<F16>(p, st);
  case BF16: return dequantize<BF16>(p, st);
  default: return hipErrorInvalidValue;
  }
}

}  // namespace mh
