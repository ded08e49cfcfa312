// Rotary positions: the angles of a step's tokens, worked out once for all
// layers, and the rotation of token rows by them (rotary.hpp has the pairs).
#include <algorithm>

#include "mh_common.hpp"
#include "mh_kernels.hpp"
#include "rotary.hpp"

namespace mh {
namespace {

// ---- rotary_table --------------------------------------------------------------

// (m cos a, m sin a) of a = position * frequency, in 64 bits: a document's
// position is a million turns of the fastest pair, of which 32 bits would leave
// four digits of the last one.  The angle is taken in turns, less the whole ones and
// then the quarters.  A pair's turns a position are frequency / 2 pi to twice 64
// bits, hi + lo (their rounding alone is 2^-25 of a turn at 2^31 positions), and
// pos hi = p + its remainder exactly: no sum of these may be fused with a product, which
// would hold the remainder already.  What is left, of at most an eighth, goes
// through the Taylor series to x^17 and x^16 (the next terms are below 2^-58), and the
// quarters say which is which.  A thread keeps its pair's turns for all tokens.
// 17000 tokens of 64 pairs: 5.8 us (1.5 TB/s written; 5.7 with the turns in 64 bits), 7.7 with a library sincos and a
// division for each value.
struct Turns {
  double hi, lo;
  __device__ __forceinline__ explicit Turns(double freq) {
#pragma clang fp contract(off)
    constexpr double kTurn = 0.15915494309189535, kRest = -9.839338337591243e-18;  // 1 / 2 pi = kTurn + kRest
    hi = freq * kTurn;
    lo = fma(freq, kTurn, -hi) + freq * kRest;
  }
};
__device__ __forceinline__ float2 angle(double pos, Turns turns, double m) {
#pragma clang fp contract(off)
  const double p = pos * turns.hi, lo = fma(pos, turns.lo, fma(pos, turns.hi, -p)), t = (p - rint(p)) + lo;
  const double quarters = rint(4.0 * t), x = (t - 0.25 * quarters) * 6.283185307179586476925, y = x * x;
  double s = 1.0 / 355687428096000.0, c = 1.0 / 20922789888000.0;
  s = fma(s, y, -1.0 / 1307674368000.0);
  c = fma(c, y, -1.0 / 87178291200.0);
  s = fma(s, y, 1.0 / 6227020800.0);
  c = fma(c, y, 1.0 / 479001600.0);
  s = fma(s, y, -1.0 / 39916800.0);
  c = fma(c, y, -1.0 / 3628800.0);
  s = fma(s, y, 1.0 / 362880.0);
  c = fma(c, y, 1.0 / 40320.0);
  s = fma(s, y, -1.0 / 5040.0);
  c = fma(c, y, -1.0 / 720.0);
  s = fma(s, y, 1.0 / 120.0);
  c = fma(c, y, 1.0 / 24.0);
  s = fma(s, y, -1.0 / 6.0);
  c = fma(c, y, -0.5);
  s = m * fma(s * y, x, x);
  c = m * fma(c, y, 1.0);
  const int q = int(quarters) & 3;
  const double u = q & 1 ? -s : c, v = q & 1 ? c : s;  // a quarter on: (-sin, cos)
  return q & 2 ? make_float2(float(-u), float(-v)) : make_float2(float(u), float(v));
}

__global__ void __launch_bounds__(256) rotary_table_kernel(const int32_t *__restrict__ pos, const double *__restrict__ freq,
                                                           float2 *__restrict__ table, int n, int half, int cols, int rows, double m) {
  const int lr = threadIdx.x / cols, lc = threadIdx.x - lr * cols;
  if (lr >= rows) return;
  for (int j = lc; j < half; j += cols) {
    const Turns turns(freq[j]);
    for (int64_t t = int64_t(blockIdx.x) * rows + lr; t < n; t += int64_t(gridDim.x) * rows) table[t * half + j] = angle(pos[t], turns, m);
  }
}

// ---- rotary --------------------------------------------------------------------

template <int DT, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(Rotary p, const int32_t *slots, int64_t limit) {
  for (int64_t t = int64_t(blockIdx.x) * p.tokens; t < p.n; t += int64_t(gridDim.x) * p.tokens)
    rotate_tokens<DT, U, INTERLEAVED, 256>(p, t, slots, limit);
}

template <int DT> void launch(const Rotary &p, int unit, const int32_t *slots, int64_t limit, unsigned grid, hipStream_t st) {
  rotary_units<DT>(p.interleaved, unit, [&](auto u, auto inter) {
    hipLaunchKernelGGL((rotary_kernel<DT, decltype(u)::value, decltype(inter)::value>), dim3(grid), dim3(256), 0, st, p, slots, limit);
  });
}

}  // namespace

hipError_t rotary_table(const int32_t *positions, const double *freq, float *table, int n, int half, double magnitude,
                        hipStream_t st) {
  const int cols = std::min(half, 256), rows = 256 / cols;
  const int64_t groups = (int64_t(n) + rows - 1) / rows;
  // (eight workgroups to a CU, then several tokens to a thread)
  hipLaunchKernelGGL(rotary_table_kernel, dim3(unsigned(std::min<int64_t>(groups, 2048))), dim3(256), 0, st, positions, freq,
                     reinterpret_cast<float2 *>(table), n, half, cols, rows, magnitude);
  return hipGetLastError();
}

hipError_t rotary(int dt, Rotary p, const int32_t *slots, int64_t limit, hipStream_t st) {
  const int unit = rotary_unit(dt, p);
  rotary_cut(dt, unit, 256, p);
  const unsigned grid = unsigned(std::min<int64_t>((int64_t(p.n) + p.tokens - 1) / p.tokens, 1 << 22));
  switch (dt) {
  case F32: launch<F32>(p, unit, slots, limit, grid, st); break;
  case F16: launch<F16>(p, unit, slots, limit, grid, st); break;
  case BF16: launch<BF16>(p, unit, slots, limit, grid, st); break;
  default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mh
