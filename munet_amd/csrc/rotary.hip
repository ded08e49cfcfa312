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
// four digits of the last one.
__global__ void __launch_bounds__(256) rotary_table_kernel(const int32_t *__restrict__ pos, const double *__restrict__ freq,
                                                           float2 *__restrict__ table, int64_t total, int half, double m) {
  for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < total; i += int64_t(gridDim.x) * 256) {
    const int64_t t = i / half;
    const int j = int(i - t * half);
    double s, c;
    sincos(double(pos[t]) * freq[j], &s, &c);
    table[i] = make_float2(float(m * c), float(m * s));
  }
}

// ---- rotary --------------------------------------------------------------------

template <int DT, int U, bool INTERLEAVED>
__global__ void __launch_bounds__(256) rotary_kernel(Rotary p, const int32_t *slots, int64_t limit) {
  for (int64_t t = int64_t(blockIdx.x) * p.tokens; t < p.n; t += int64_t(gridDim.x) * p.tokens)
    rotate_tokens<DT, U, INTERLEAVED, 256>(p, t, slots, limit);
}

template <int DT, int U>
void launch(const Rotary &p, const int32_t *slots, int64_t limit, unsigned grid, hipStream_t st) {
  constexpr int V = U == 1 ? 1 : U / 2;  // (interleaved pairs lie in one load)
  if (p.interleaved) hipLaunchKernelGGL((rotary_kernel<DT, V, true>), dim3(grid), dim3(256), 0, st, p, slots, limit);
  else hipLaunchKernelGGL((rotary_kernel<DT, U, false>), dim3(grid), dim3(256), 0, st, p, slots, limit);
}

}  // namespace

hipError_t rotary_table(const int32_t *positions, const double *freq, float *table, int n, int half, double magnitude,
                        hipStream_t st) {
  const int64_t total = int64_t(n) * half;
  const unsigned grid = unsigned(std::min<int64_t>((total + 255) / 256, 1 << 20));
  hipLaunchKernelGGL(rotary_table_kernel, dim3(grid), dim3(256), 0, st, positions, freq, reinterpret_cast<float2 *>(table), total,
                     half, magnitude);
  return hipGetLastError();
}

hipError_t rotary(int dt, Rotary p, const int32_t *slots, int64_t limit, hipStream_t st) {
  const int unit = rotary_unit(dt, p);
  rotary_cut(dt, unit, 256, p);
  const unsigned grid = unsigned(std::min<int64_t>((int64_t(p.n) + p.tokens - 1) / p.tokens, 1 << 22));
  switch (dt) {
  case F32: unit == 1 ? launch<F32, 1>(p, slots, limit, grid, st) : launch<F32, 4>(p, slots, limit, grid, st); break;
  case F16: unit == 1 ? launch<F16, 1>(p, slots, limit, grid, st) : launch<F16, 8>(p, slots, limit, grid, st); break;
  case BF16: unit == 1 ? launch<BF16, 1>(p, slots, limit, grid, st) : launch<BF16, 8>(p, slots, limit, grid, st); break;
  default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

}  // namespace mh
