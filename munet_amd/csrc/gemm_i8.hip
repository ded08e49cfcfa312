// out[M, N] = act(sx_m sw_n sum_k x[m, k] w[n, k] + bias_n) + resid[m, n] with x and w
// in 8-bit integers (v_mfma_i32_16x16x64_i8: 64 products of K per instruction).
#include "gemm_i8.hpp"

namespace mh {
namespace {

// 16 bytes of a row from k on, zeros past K.  Rows start anywhere: the loads are
// not aligned.
__device__ __forceinline__ i32x4 row_chunk(const int8_t *row, int k, int K) {
  struct __attribute__((packed)) Any { i32x4 v; };
  if (k + 16 <= K) return reinterpret_cast<const Any *>(row + k)->v;
  i32x4 r = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (k + i < K) r[i >> 2] |= int(uint32_t(uint8_t(row[k + i])) << (8 * (i & 3)));
  return r;
}

// Any K, any row spacing: 64 x 64 tiles of four waves, slabs of 128 bytes of K
// staged through registers into two LDS buffers (gemm_pipe.hpp's layout).
template <int DT>
__global__ void __launch_bounds__(256) gemm_i8_any_kernel(LinearI8 p) {
  constexpr int BM = 64, BN = 64;
  typedef PipeGeom<BM, BN, 2, 2> G;
  __shared__ u32x4 lds[2][(BM + BN) * 8];
  int m0, n0;
  pipe_tile<BM, BN>(p.M, p.N, 0, m0, n0);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const G g(wave, lane);
  const int c0 = tid & 7, r0 = tid >> 3;
  const int8_t *xr[2], *wr[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    xr[i] = p.x + int64_t(min(m0 + r0 + 32 * i, p.M - 1)) * p.ldx;
    wr[i] = p.w + int64_t(min(n0 + r0 + 32 * i, p.N - 1)) * p.ldw;
  }
  i32x4 ra[2], rb[2];
  auto load = [&](int kt) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      ra[i] = row_chunk(xr[i], kt * 128 + c0 * 16, p.K);
      rb[i] = row_chunk(wr[i], kt * 128 + c0 * 16, p.K);
    }
  };
  auto put = [&](int b) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = r0 + 32 * i;
      lds[b][r * 8 + (c0 ^ (r & 7))] = __builtin_bit_cast(u32x4, ra[i]);
      lds[b][BM * 8 + r * 8 + (c0 ^ (r & 7))] = __builtin_bit_cast(u32x4, rb[i]);
    }
  };
  i32x4 acc[G::FM][G::FN] = {};
  const int KT = (p.K + 127) / 128;
  load(0);
  put(0);
  __syncthreads();
  for (int kt = 0; kt < KT; ++kt) {
    if (kt + 1 < KT) load(kt + 1);
    u32x4 af[G::FM], bf[G::FN];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks == 0) g.template frags<0>(lds[kt & 1], af, bf);
      else g.template frags<1>(lds[kt & 1], af, bf);
#pragma unroll
      for (int i = 0; i < G::FM; ++i)
#pragma unroll
        for (int j = 0; j < G::FN; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, bf[j]), __builtin_bit_cast(i32x4, af[i]),
                                                            acc[i][j], 0, 0, 0);
    }
    if (kt + 1 < KT) put((kt + 1) & 1);
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < G::FN; ++j) {
    const int n = n0 + g.wn * G::WTN + j * 16 + 4 * g.lg;
    Scale sw[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) sw[i] = Scale(p.sw[min(n + i, p.N - 1)]);
#pragma unroll
    for (int i = 0; i < G::FM; ++i) {
      const int m = m0 + g.wm * G::WTM + i * 16 + g.li;
      if (m < p.M && n < p.N) i8_store4<DT>(p, m, n, acc[i][j], Scale(p.sx[m]), sw);
    }
  }
}

template <int DT> hipError_t launch_any(const LinearI8 &p, hipStream_t st) {
  const int64_t tiles = int64_t((p.M + 63) / 64) * ((p.N + 63) / 64);
  if (tiles > kI8MaxTiles) return hipErrorInvalidValue;
  hipLaunchKernelGGL(gemm_i8_any_kernel<DT>, dim3(unsigned(tiles)), dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace

hipError_t linear_i8(int dt, const LinearI8 &p, hipStream_t st) {
  switch (dt) {
  case F32: return launch_any<F32>(p, st);
  case F16: return launch_any<F16>(p, st);
  case BF16: return launch_any<BF16>(p, st);
  default: return hipErrorInvalidValue;
  }
}

}  // namespace mh
