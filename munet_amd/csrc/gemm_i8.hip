// Products of 8-bit integers with a scale for each row of both operands:
// out[M, N] = act(sx_m sw_n sum_k x[m, k] w[n, k] + bias_n) + resid[m, n] with x and w
// in 8-bit integers (v_mfma_i32_16x16x64_i8: 64 products of K per instruction).
#include <cstdlib>

#include "gemm_i8.hpp"
#include "gemm_i8_tiles.hpp"

namespace mh {
namespace {

// Any K, any row spacing: four waves, slabs of 128 bytes of K staged through
// registers into two LDS buffers (gemm_pipe.hpp's layout).
template <int DT, int BM, int BN> __global__ void __launch_bounds__(256) gemm_i8_any_kernel(LinearI8 p, int gn) {
  constexpr int XCH = BM / 32, WCH = BN / 32;
  typedef I8Geom<BM, BN, 2, 2> G;
  __shared__ u32x4 lds[2][(BM + BN) * 8];
  int m0, n0;
  pipe_tile<BM, BN>(p.M, p.N, gn, m0, n0);
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const G g(wave, lane);
  // chunk c0 of rows r0 + 32 i; rows past the end read the last one
  const int c0 = tid & 7, r0 = tid >> 3;
  const int8_t *xr[XCH], *wr[WCH];
#pragma unroll
  for (int i = 0; i < XCH; ++i) xr[i] = p.x + int64_t(min(m0 + r0 + 32 * i, p.M - 1)) * p.ldx + c0 * 16;
#pragma unroll
  for (int i = 0; i < WCH; ++i) wr[i] = p.w + int64_t(min(n0 + r0 + 32 * i, p.N - 1)) * p.ldw + c0 * 16;
  i32x4 ra[XCH], rb[WCH];
  const int KT = (p.K + 127) / 128;
  auto end = [](const int8_t *at, int left) {
    RowBlock<true> r;
    const int shift = row_shift(at);
    r.load_end(at, shift, left);
    return r.get(shift);
  };
  auto load = [&](int kt) {
    const int k = kt * 128;
    if (k + 128 <= p.K) {
#pragma unroll
      for (int i = 0; i < XCH; ++i) ra[i] = row_bytes(xr[i] + k);
#pragma unroll
      for (int i = 0; i < WCH; ++i) rb[i] = row_bytes(wr[i] + k);
    } else {
      const int left = p.K - k - c0 * 16;
#pragma unroll
      for (int i = 0; i < XCH; ++i) ra[i] = end(xr[i] + k, left);
#pragma unroll
      for (int i = 0; i < WCH; ++i) rb[i] = end(wr[i] + k, left);
    }
  };
  auto put = [&](int b) {
#pragma unroll
    for (int i = 0; i < XCH; ++i) lds[b][(r0 + 32 * i) * 8 + (c0 ^ G::xswizzle(r0 + 32 * i))] = __builtin_bit_cast(u32x4, ra[i]);
#pragma unroll
    for (int i = 0; i < WCH; ++i) lds[b][(BM + r0 + 32 * i) * 8 + (c0 ^ G::wswizzle(r0 + 32 * i))] = __builtin_bit_cast(u32x4, rb[i]);
  };
  i32x4 acc[G::FM][G::FN] = {};
  load(0);
  put(0);
  __syncthreads();
  for (int kt = 0; kt < KT; ++kt) {
    if (kt + 1 < KT) load(kt + 1);
    u32x4 af[G::FM], bf[G::FN];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int i = 0; i < G::FM; ++i) af[i] = g.xfrag(lds[kt & 1], i, 4 * ks + g.lg);
#pragma unroll
      for (int j = 0; j < G::FN; ++j) bf[j] = g.wfrag(lds[kt & 1], j, 4 * ks + g.lg);
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
  i8_store<DT, G>(p, g, m0, n0, acc);
}

// 64 lanes x 16 bytes from a buffer resource into LDS bytes [m0, m0 + 1024); lanes past
// the resource's end write zeros.
__device__ __forceinline__ void dma16_at(__amdgpu_buffer_rsrc_t res, uint32_t voff, uint32_t soff, uint32_t ldsaddr) {
  asm volatile("s_mov_b32 m0, %3\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds" ::"v"(voff), "s"(res), "s"(soff), "s"(ldsaddr)
               : "memory", "m0");
}

// Rows and addresses in whole 16-byte blocks: slabs of 128 bytes of K go straight
// into S LDS stages, as in gemm_dma_kernel (gemm_pipe.hpp has the layout, the
// schedule of a step and why its loads are inline assembly).  A slab of 128 int8
// takes as many MFMA cycles as one of 64 16-bit values for twice the products.
// Where the last slab is not whole, its blocks past K are read from past the
// end of the resource, as zeros.
template <int DT, int BM, int BN, int WGM, int WGN, int S>
__global__ void __launch_bounds__(WGM * WGN * 64) gemm_i8_kernel(LinearI8 p, int gn) {
  typedef I8Geom<BM, BN, WGM, WGN> G;
  constexpr int NW = G::NW, FM = G::FM, FN = G::FN;
  constexpr int ABLK = BM / 8 / NW, BBLK = BN / 8 / NW, NDMA = ABLK + BBLK;
  static_assert(BM % (8 * NW) == 0 && BN % (8 * NW) == 0, "the waves share the loads evenly");
  static_assert(S >= 2 && NDMA * (S - 1) < 64, "stages");
  constexpr uint32_t STAGE = (BM + BN) * 128;
  __shared__ u32x4 lds[S][(BM + BN) * 8];
  int m0, n0;
  pipe_tile<BM, BN>(p.M, p.N, gn, m0, n0);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const G g(wave, lane);
  // lane l of a load fetches block row l / 8's chunk that lies at LDS slot l % 8
  const int lr = lane >> 3, lc = (lane & 7) ^ G::xswizzle(lr);
  auto wchunk = [&](int i) { return (lane & 7) ^ G::wswizzle((wave * BBLK + i) * 8 + lr); };
  const int KT = (p.K + 127) / 128;
  // (a tile's rows span less than 2^31 bytes: the host checks; rows past the end
  // read the last one, their results are not stored)
  const int rx = min(BM, p.M - m0), rw = min(BN, p.N - n0);
  const __amdgpu_buffer_rsrc_t xres = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p.x + int64_t(m0) * p.ldx), 0,
                                                                        int((rx - 1) * p.ldx) + p.K, 0x00020000);
  const __amdgpu_buffer_rsrc_t wres = __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t *>(p.w + int64_t(n0) * p.ldw), 0,
                                                                        int((rw - 1) * p.ldw) + p.K, 0x00020000);
  uint32_t aoff[ABLK], boff[BBLK];
#pragma unroll
  for (int i = 0; i < ABLK; ++i) aoff[i] = uint32_t(min((wave * ABLK + i) * 8 + lr, rx - 1)) * uint32_t(p.ldx) + lc * 16;
#pragma unroll
  for (int i = 0; i < BBLK; ++i) boff[i] = uint32_t(min((wave * BBLK + i) * 8 + lr, rw - 1)) * uint32_t(p.ldw) + wchunk(i) * 16;
  const uint32_t lds0 = uint32_t(reinterpret_cast<uintptr_t>((lds_void_t *)&lds[0][0]));
  const uint32_t wa = lds0 + wave * ABLK * 1024, wb = lds0 + BM * 128 + wave * BBLK * 1024;
  // this lane's blocks of the last slab that lie past K
  const int rest = p.K - (KT - 1) * 128;
  const uint32_t xpast = lc * 16 >= rest ? 0x80000000u : 0u;
  uint32_t wpast[2];  // (the chunk alternates at most between two of a wave's blocks)
#pragma unroll
  for (int i = 0; i < 2; ++i) wpast[i] = wchunk(i < BBLK ? i : 0) * 16 >= rest ? 0x80000000u : 0u;
  // load T of a slab into a stage; LAST: of the last slab
#define MH_DMA(T, KT_, LAST, ST)                                                                               \
  {                                                                                                           \
    if ((T) < ABLK)                                                                                           \
      dma16_at(xres, aoff[(T) % ABLK] | ((LAST) ? xpast : 0u), (KT_) * 128, wa + (ST) * STAGE + ((T) % ABLK) * 1024);  \
    else                                                                                                      \
      dma16_at(wres, boff[((T) - ABLK) % BBLK] | ((LAST) ? wpast[((T) - ABLK) % BBLK % 2] : 0u), (KT_) * 128,  \
               wb + (ST) * STAGE + (((T) - ABLK) % BBLK) * 1024);                                             \
  }
  i32x4 acc[FM][FN];
  u32x4 af0[FM], bf0[FN], af1[FM], bf1[FN];
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    const int kt = min(s, KT - 1);
#pragma unroll
    for (int t = 0; t < NDMA; ++t) MH_DMA(t, kt, kt == KT - 1, s);
  }
  dma_wait<NDMA *(S - 2)>();
  __syncthreads();
#pragma unroll
  for (int i = 0; i < FM; ++i) af0[i] = g.xfrag(lds[0], i, g.lg);
#pragma unroll
  for (int j = 0; j < FN; ++j) bf0[j] = g.wfrag(lds[0], j, g.lg);

  constexpr int NMM = FM * FN, NRD = FM + FN, RPM = 2;
  constexpr int LATE = S == 2 ? (NRD + RPM - 1) / RPM : 0;  // two stages: the wait comes late in the second half
  static_assert(LATE <= NMM, "late wait");
  constexpr int STAGE4 = (BM + BN) * 8;
  const int c1 = 4 + g.lg, c0f = g.lg;
  auto mma = [](i32x4 &c, u32x4 b, u32x4 a) {
    c = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4, b), __builtin_bit_cast(i32x4, a), c, 0, 0, 0);
  };
#define MH_FRAG(L, C, X, AF, BF)                                                                               \
  {                                                                                                           \
    if ((X) < FM) AF[(X) % FM] = g.xfrag(L, (X) % FM, C);                                                     \
    else BF[((X) - FM) % FN] = g.wfrag(L, ((X) - FM) % FN, C);                                                \
  }
  int stg = 0;
#define MH_STEP(KK, FIRST)                                                                                     \
  {                                                                                                           \
    const int s_ = stg, sn_ = s_ + 1 == S ? 0 : s_ + 1, sf_ = s_ == 0 ? S - 1 : s_ - 1;                        \
    const int kf_ = min((KK) + S - 1, KT - 1);                                                                \
    const bool last_ = kf_ == KT - 1;                                                                         \
    const u32x4 *Ls_ = &lds[0][0] + s_ * STAGE4, *Ln_ = &lds[0][0] + sn_ * STAGE4;                             \
    _Pragma("unroll") for (int t = 0; t < NMM; ++t) {                                                         \
      if (FIRST) acc[t / FN][t % FN] = i32x4{0, 0, 0, 0};                                                     \
      mma(acc[t / FN][t % FN], bf0[t % FN], af0[t / FN]);                                                     \
      if (t < NDMA) MH_DMA(t, kf_, last_, sf_)                                                                \
      else if (t < NDMA + NRD) MH_FRAG(Ls_, c1, t - NDMA, af1, bf1)                                           \
      __builtin_amdgcn_sched_barrier(0);                                                                      \
    }                                                                                                         \
    _Pragma("unroll") for (int t = NMM; t < NDMA + NRD; ++t) {                                                \
      if (t < NDMA) MH_DMA(t, kf_, last_, sf_)                                                                \
      else MH_FRAG(Ls_, c1, t - NDMA, af1, bf1)                                                               \
    }                                                                                                         \
    if constexpr (LATE == 0) {                                                                                \
      dma_wait<NDMA *(S - 2)>();                                                                              \
      __syncthreads();                                                                                        \
    }                                                                                                         \
    _Pragma("unroll") for (int t = 0; t < NMM; ++t) {                                                         \
      if (LATE > 0 && t == NMM - LATE) {                                                                      \
        dma_wait<0>();                                                                                        \
        __syncthreads();                                                                                      \
      }                                                                                                       \
      mma(acc[t / FN][t % FN], bf1[t % FN], af1[t / FN]);                                                     \
      if (LATE == 0) {                                                                                        \
        if (t < NRD) MH_FRAG(Ln_, c0f, t, af0, bf0)                                                           \
      } else if (t >= NMM - LATE) {                                                                           \
        _Pragma("unroll") for (int q_ = 0; q_ < RPM; ++q_)                                                    \
          if (RPM * (t - (NMM - LATE)) + q_ < NRD) MH_FRAG(Ln_, c0f, RPM * (t - (NMM - LATE)) + q_, af0, bf0)  \
      }                                                                                                       \
      __builtin_amdgcn_sched_barrier(0);                                                                      \
    }                                                                                                         \
    if constexpr (LATE == 0) {                                                                                \
      _Pragma("unroll") for (int t = NMM; t < NRD; ++t) MH_FRAG(Ln_, c0f, t, af0, bf0)                         \
    }                                                                                                         \
    stg = sn_;                                                                                                \
  }
  MH_STEP(0, true);
  for (int k = 1; k < KT; ++k) MH_STEP(k, false);
#undef MH_STEP
#undef MH_FRAG
#undef MH_DMA
  dma_wait<0>();  // no load is in flight when the workgroup ends
  i8_store<DT, G>(p, g, m0, n0, acc);
}

// Column groups of the tile enumeration, as in gemm_pipe.hip.
int column_groups(const LinearI8 &p) { return 2L * p.N >= p.M ? (p.N >= 4L * p.M ? 16 : 8) : 0; }

template <int DT, int BM, int BN> hipError_t launch_any(const LinearI8 &p, hipStream_t st) {
  const int64_t tiles = int64_t((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  if (tiles > kI8MaxTiles) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_i8_any_kernel<DT, BM, BN>), dim3(unsigned(tiles)), dim3(256), 0, st, p, column_groups(p));
  return hipGetLastError();
}

template <int DT, int BM, int BN, int WGM, int WGN, int S> hipError_t launch(const LinearI8 &p, hipStream_t st) {
  const int64_t tiles = int64_t((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  if (tiles > kI8MaxTiles) return hipErrorInvalidValue;
  hipLaunchKernelGGL((gemm_i8_kernel<DT, BM, BN, WGM, WGN, S>), dim3(unsigned(tiles)), dim3(WGM * WGN * 64), 0, st, p, column_groups(p));
  return hipGetLastError();
}

// Whether rows and addresses go in 16-byte blocks, tiles of up to 256 rows within the
// 31 bits of a buffer resource.
bool blocks(const LinearI8 &p) {
  return p.K % 16 == 0 && p.ldx % 16 == 0 && p.ldw % 16 == 0 && reinterpret_cast<uintptr_t>(p.x) % 16 == 0 &&
         reinterpret_cast<uintptr_t>(p.w) % 16 == 0 && p.ldx < (1 << 22) && p.ldw < (1 << 22);
}

template <int DT> hipError_t run(const LinearI8 &p, hipStream_t st) {
  const bool whole = blocks(p);
  int tile = i8_tile(whole, p.M, p.N, p.K);
  // MUNET_HIP_I8_TILE names a kernel for tests and tuning (read at every call; one that
  // the operands do not suit takes the automatic choice)
  if (const char *force = std::getenv("MUNET_HIP_I8_TILE")) {
    const int f = std::atoi(force);
    if (f == 0 || f == 10 || (f >= 1 && f <= 9 && whole) || ((f == 100 || f == 101) && p.M <= kI8FewRows)) tile = f;
  }
  switch (tile) {
  case 1: return launch<DT, 256, 256, 2, 4, 2>(p, st);
  case 2: return launch<DT, 256, 128, 4, 2, 3>(p, st);
  case 3: return launch<DT, 128, 128, 4, 2, 4>(p, st);
  case 4: return launch<DT, 128, 64, 4, 2, 6>(p, st);
  case 5: return launch<DT, 64, 64, 2, 2, 5>(p, st);
  case 6: return launch<DT, 64, 64, 2, 2, 3>(p, st);
  case 7: return launch<DT, 64, 32, 2, 2, 6>(p, st);
  case 8: return launch<DT, 32, 32, 2, 2, 9>(p, st);
  case 9: return launch<DT, 64, 128, 2, 4, 3>(p, st);
  case 10: return launch_any<DT, 128, 128>(p, st);
  case 100:
  case 101: return linear_i8_few(DT, p, tile - 100, st);
  default: return launch_any<DT, 64, 64>(p, st);
  }
}

}  // namespace

hipError_t linear_i8(int dt, const LinearI8 &p, hipStream_t st) {
  switch (dt) {
  case F32: return run<F32>(p, st);
  case F16: return run<F16>(p, st);
  case BF16: return run<BF16>(p, st);
  default: return hipErrorInvalidValue;
  }
}

}  // namespace mh
