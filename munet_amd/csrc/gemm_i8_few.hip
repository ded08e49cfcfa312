// Products of 8-bit integers with few rows (a decode step's tokens): bound by the
// weights' bytes and, before them, by the latency of a load.
//
// A workgroup has up to 16 MF rows and 16 NF columns; its W waves share K out in
// pieces of CH steps of 64, one after another, and each loads its operands
// straight into registers (lane (li, lg) holds 16 bytes of row li from 16 lg on, which
// is the MFMA's operand): no LDS, no barrier and no wait for another wave until the
// sums are added at the end, in int32, so in any order.  1 x 4096 x 4096, weights not
// in L2: 6.2 us (2.7 TB/s; 32 x 32 tiles through LDS 7.1, 64 x 64 10.6), 1 x 2304 x 768
// 2.9 us, of which an empty kernel takes 2.3.
#include "gemm_i8.hpp"
#include "gemm_i8_tiles.hpp"

namespace mh {
namespace {

template <int DT, int MF, int NF, int W, int CH, bool ODD>
__global__ void __launch_bounds__(64 * W) gemm_i8_few_kernel(LinearI8 p) {
  __shared__ i32x4 red[W][MF * NF][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int li = lane & 15, lg = lane >> 4;
  const int n0 = blockIdx.x * (16 * NF), m0 = blockIdx.y * (16 * MF);
  const int8_t *xr[MF], *wr[NF];
#pragma unroll
  for (int i = 0; i < MF; ++i) xr[i] = p.x + int64_t(min(m0 + 16 * i + li, p.M - 1)) * p.ldx + 16 * lg;
#pragma unroll
  for (int j = 0; j < NF; ++j) wr[j] = p.w + int64_t(min(n0 + 16 * j + li, p.N - 1)) * p.ldw + 16 * lg;
  int xs[MF], ws[NF];
#pragma unroll
  for (int i = 0; i < MF; ++i) xs[i] = row_shift(xr[i]);
#pragma unroll
  for (int j = 0; j < NF; ++j) ws[j] = row_shift(wr[j]);
  i32x4 acc[MF][NF] = {};
  const int whole = p.K / 64, pieces = whole / CH;  // steps and pieces that every lane has
  struct Piece { RowBlock<ODD> x[CH][MF], w[CH][NF]; } a, b;
  auto load = [&](Piece &q, int piece) {
#pragma unroll
    for (int s = 0; s < CH; ++s) {
      const int k = (piece * CH + s) * 64;
#pragma unroll
      for (int j = 0; j < NF; ++j) q.w[s][j].load(wr[j] + k, ws[j]);
#pragma unroll
      for (int i = 0; i < MF; ++i) q.x[s][i].load(xr[i] + k, xs[i]);
    }
  };
  auto add = [&](const Piece &q) {
#pragma unroll
    for (int s = 0; s < CH; ++s)
#pragma unroll
      for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.w[s][j].get(ws[j]), q.x[s][i].get(xs[i]), acc[i][j], 0, 0, 0);
  };
  int c = wave;
  if (c < pieces) load(a, c);
  for (; c < pieces; c += 2 * W) {
    if (c + W < pieces) load(b, c + W);
    add(a);
    if (c + W >= pieces) break;
    if (c + 2 * W < pieces) load(a, c + 2 * W);
    add(b);
  }
  // the steps behind the last whole piece, the last one of them not whole
  for (int s = pieces * CH + wave; s * 64 < p.K; s += W) {
    RowBlock<ODD> x[MF], w[NF];
    const int k = s * 64, left = p.K - k - 16 * lg;
#pragma unroll
    for (int j = 0; j < NF; ++j) w[j].load_end(wr[j] + k, ws[j], left);
#pragma unroll
    for (int i = 0; i < MF; ++i) x[i].load_end(xr[i] + k, xs[i], left);
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
      for (int j = 0; j < NF; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[j].get(ws[j]), x[i].get(xs[i]), acc[i][j], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < MF; ++i)
#pragma unroll
    for (int j = 0; j < NF; ++j) red[wave][i * NF + j][lane] = acc[i][j];
  __syncthreads();
  typedef I8Geom<16, 16, 1, 1> G;
  const G g(0, lane);
#pragma unroll 1
  for (int f = wave; f < MF * NF; f += W) {
    i32x4 sum[1][1] = {{red[0][f][lane]}};
#pragma unroll
    for (int v = 1; v < W; ++v) sum[0][0] += red[v][f][lane];
    const int m = m0 + 16 * (f / NF), n = n0 + 16 * (f % NF);
    if (m < p.M && n < p.N) i8_store<DT, G>(p, g, m, n, sum);
  }
}

template <int DT, int MF, int NF, int W, int CH> hipError_t launch(const LinearI8 &p, hipStream_t st) {
  const dim3 grid(unsigned((p.N + 16 * NF - 1) / (16 * NF)), unsigned((p.M + 16 * MF - 1) / (16 * MF)));
  if (p.M > kI8FewRows || int64_t(grid.x) * grid.y > kI8MaxTiles) return hipErrorInvalidValue;
  if (odd_rows(p)) hipLaunchKernelGGL((gemm_i8_few_kernel<DT, MF, NF, W, CH, true>), grid, dim3(64 * W), 0, st, p);
  else hipLaunchKernelGGL((gemm_i8_few_kernel<DT, MF, NF, W, CH, false>), grid, dim3(64 * W), 0, st, p);
  return hipGetLastError();
}

template <int DT> hipError_t run(const LinearI8 &p, int form, hipStream_t st) {
  return form == 0 ? launch<DT, 1, 1, 4, 4>(p, st) : launch<DT, 1, 2, 8, 4>(p, st);
}

}  // namespace

hipError_t linear_i8_few(int dt, const LinearI8 &p, int form, hipStream_t st) {
  switch (dt) {
  case F32: return run<F32>(p, form, st);
  case F16: return run<F16>(p, form, st);
  case BF16: return run<BF16>(p, form, st);
  default: return hipErrorInvalidValue;
  }
}

}  // namespace mh
