// The epilogue of the 8-bit integer products (gemm_i8*.hip): sums in int32, which
// hold K < 2^17 products of magnitude 2^14 exactly; everything after in 32-bit
// floats, rounded once.
#pragma once

#include "gemm_pipe.hpp"

namespace mh {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// 16 bytes of a row from anywhere.
__device__ __forceinline__ i32x4 row_bytes(const int8_t *p) {
  struct __attribute__((packed)) Any { i32x4 v; };
  return reinterpret_cast<const Any *>(p)->v;
}
// 16 bytes of a row.  ODD: rows start anywhere, `shift` bytes behind a word; whole
// words are loaded, five of them, all of which hold some of the 16 bytes, and
// shifted when they are used (in the kernels of few rows: loads that are not aligned to
// words took 64 x 12801 x 4095 from 68 to 177 us; the tiles, which load further ahead,
// are slower with words, 8192 x 8191 x 8191 1.9 ms against 1.1).  Else the row's blocks start at words.
template <bool ODD> struct RowBlock {
  i32x4 v;
  int next;
  __device__ __forceinline__ void load(const int8_t *p, int shift) {
    struct __attribute__((packed, aligned(4))) Words { i32x4 v; };
    const int8_t *w = ODD ? p - shift : p;
    v = reinterpret_cast<const Words *>(w)->v;
    if constexpr (ODD) next = reinterpret_cast<const int *>(w)[shift ? 4 : 3];
  }
  // where `left` values are left of the row: zeros behind them, and no word without one
  __device__ __forceinline__ void load_end(const int8_t *p, int shift, int left) {
    if (left >= 16) {
      load(p, shift);
      return;
    }
    const int first = ODD ? shift : 0, end = left > 0 ? first + left : 0;
    const int *w = reinterpret_cast<const int *>(p - first);
    uint32_t r[5];
#pragma unroll
    for (int q = 0; q < 5; ++q) {
      const int n = end - 4 * q;
      const uint32_t x = n > 0 && (ODD || q < 4) ? uint32_t(w[q]) : 0u;
      r[q] = n >= 4 ? x : n > 0 ? x & ((1u << (8 * n)) - 1u) : 0u;
    }
    v = i32x4{int(r[0]), int(r[1]), int(r[2]), int(r[3])};
    if constexpr (ODD) next = int(r[4]);
  }
  __device__ __forceinline__ i32x4 get(int shift) const {
    if constexpr (!ODD) return v;
    const uint32_t s = uint32_t(shift);
    return i32x4{int(__builtin_amdgcn_alignbyte(uint32_t(v[1]), uint32_t(v[0]), s)), int(__builtin_amdgcn_alignbyte(uint32_t(v[2]), uint32_t(v[1]), s)),
                 int(__builtin_amdgcn_alignbyte(uint32_t(v[3]), uint32_t(v[2]), s)), int(__builtin_amdgcn_alignbyte(uint32_t(next), uint32_t(v[3]), s))};
  }
};
__device__ __forceinline__ int row_shift(const int8_t *p) { return int(reinterpret_cast<uintptr_t>(p) & 3); }
inline bool odd_rows(const LinearI8 &p) {
  return ((reinterpret_cast<uintptr_t>(p.x) | reinterpret_cast<uintptr_t>(p.w)) & 3) || (p.ldx & 3) || (p.ldw & 3);
}

// A scale as a fraction and a power of two.  The product of two scales may lie
// outside the floats where the result does not (and below the normal ones, where
// it loses digits): fractions multiply, powers add.
struct Scale {
  float f;
  int e;
  __device__ __forceinline__ Scale() {}
  __device__ __forceinline__ explicit Scale(float s) : f(__builtin_amdgcn_frexp_mantf(s)), e(__builtin_amdgcn_frexp_expf(s)) {}
};

// A wave's tile of BM x BN / (WGM x WGN) outputs.  The sums of fragment (i, j) lie in
// lane (li, lg) as four of row 16 i + li; which four columns they are is decided by
// the rows of w that the fragment is given: fragments 2 q and 2 q + 1 take
// alternate fours of 32 columns, so that a lane ends with eight consecutive
// columns, 32 q + 8 lg .. + 7, and four lanes with 64 consecutive bytes of 16-bit
// results (with a fragment to 16 consecutive columns, so stores of 8 bytes, 4096 x
// 2304 x 128 took 16.5 us on 256 x 256 tiles, 7.2 without its stores; so 12.5).
template <int BM, int BN, int WGM, int WGN> struct I8Geom : PipeGeom<BM, BN, WGM, WGN> {
  typedef PipeGeom<BM, BN, WGM, WGN> P;
  static constexpr int FM = P::FM, FN = P::FN;
  static constexpr int COLS = FN == 1 ? 4 : 8, GROUPS = FN * 4 / COLS;  // consecutive columns of a lane
  static_assert(FN == 1 || FN % 2 == 0, "fragments go in pairs");
  __device__ __forceinline__ I8Geom(int wave, int lane) : P(wave, lane) {}
  // LDS: row r's chunk c lies at c ^ swizzle(r), so that the eight rows that eight
  // consecutive lanes read spread over the banks
  static __device__ __forceinline__ int xswizzle(int r) { return r & 7; }
  static __device__ __forceinline__ int wswizzle(int r) { return FN == 1 ? r & 7 : (r & 3) | ((r >> 1) & 4); }
  __device__ __forceinline__ u32x4 xfrag(const u32x4 *L, int i, int c) const {
    const int r = this->wm * P::WTM + i * 16 + this->li;
    return L[r * 8 + (c ^ xswizzle(r))];
  }
  __device__ __forceinline__ u32x4 wfrag(const u32x4 *L, int j, int c) const {
    const int r = this->wn * P::WTN + (FN == 1 ? this->li : 32 * (j / 2) + 8 * (this->li >> 2) + 4 * (j & 1) + (this->li & 3));
    return L[BM * 8 + r * 8 + (c ^ wswizzle(r))];
  }
  __device__ __forceinline__ int row(int m0, int i) const { return m0 + this->wm * P::WTM + i * 16 + this->li; }
  __device__ __forceinline__ int col(int n0, int q) const { return n0 + this->wn * P::WTN + 32 * q + COLS * this->lg; }
};

// C consecutive values, aligned to their type alone, and their stores.
template <int DT, int C> __device__ __forceinline__ void i8_get(const typename Store<DT>::T *p, float (&v)[C]) {
  struct __attribute__((packed, aligned(4))) F4 { f32x4 v; };
  struct __attribute__((packed, aligned(2))) H8 { uint4 v; };
  struct __attribute__((packed, aligned(2))) H4 { uint2 v; };
  if constexpr (DT == F32) {
#pragma unroll
    for (int i = 0; i < C; i += 4) {
      const f32x4 x = reinterpret_cast<const F4 *>(p + i)->v;
      v[i] = x[0]; v[i + 1] = x[1]; v[i + 2] = x[2]; v[i + 3] = x[3];
    }
  } else if constexpr (C == 8) {
    dec8<DT>(reinterpret_cast<const H8 *>(p)->v, v);
  } else {
    const uint2 x = reinterpret_cast<const H4 *>(p)->v;
    v[0] = Store<DT>::dec(uint16_t(x.x)); v[1] = Store<DT>::dec(uint16_t(x.x >> 16));
    v[2] = Store<DT>::dec(uint16_t(x.y)); v[3] = Store<DT>::dec(uint16_t(x.y >> 16));
  }
}
template <int DT, int C> __device__ __forceinline__ void i8_put(typename Store<DT>::T *p, float (&v)[C]) {
  struct __attribute__((packed, aligned(4))) F4 { f32x4 v; };
  struct __attribute__((packed, aligned(2))) H8 { uint4 v; };
  struct __attribute__((packed, aligned(2))) H4 { uint2 v; };
  if constexpr (DT == F32) {
#pragma unroll
    for (int i = 0; i < C; i += 4) reinterpret_cast<F4 *>(p + i)->v = f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]};
  } else {
    uint32_t w[C / 2];
    if constexpr (DT == F16) {
#pragma unroll
      for (int i = 0; i < C; i += 4) round4_f16(v + i);
    }
#pragma unroll
    for (int i = 0; i < C / 2; ++i) w[i] = DT == F16 ? pack_f16x2_exact(v[2 * i], v[2 * i + 1]) : pack_bf16x2(v[2 * i], v[2 * i + 1]);
    if constexpr (C == 8) reinterpret_cast<H8 *>(p)->v = make_uint4(w[0], w[1], w[2], w[3]);
    else reinterpret_cast<H4 *>(p)->v = make_uint2(w[0], w[1]);
  }
}
// A product that no sum is fused with: which of them the compiler fuses differs from one
// kernel to the next, and so would the bits.
__device__ __forceinline__ float mul_alone(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}
template <int ACT> __device__ __forceinline__ float i8_act(float v) {
  if constexpr (ACT == ACT_RELU) return v < 0.f ? 0.f : v;  // (NaN stays)
  if constexpr (ACT == ACT_GELU) return mul_alone(v, sigmoidf_ref(mul_alone(1.702f, v)));
  return v;
}

// Whether sums times any two scales of this size, one after the other, stay normal floats or
// overflow where the result does.
__device__ __forceinline__ bool plain_scale(float s) { return s == 0.f || (s >= 0x1p-60f && s <= 0x1p60f); }

// A wave's results.  What is the same for several fragments is loaded before the
// first store (a load behind a store waits for it: out might be what is read), a
// row's residual before its stores.  The code is straight and runs once a tile, so
// that it is fetched while it runs: what every fragment might need, inline in
// each, was 100 KB of it.  Hence one path for whole tiles with scales of ordinary
// size, which multiply as they are, for each activation, and one for all else,
// where scales are fractions and powers of two: the same bits where both can.
// No sum is fused with a product, a missing bias or residual is a zero: a row's
// results do not depend on the kernel.  (Whole rows through LDS were slower: 4096 x 4096 x
// 1024 on 256 x 128 tiles 38 us, 34 from registers.)
template <int DT, typename G, int ACT>
__device__ __forceinline__ void i8_store_whole(const LinearI8 &p, const G &g, int m0, int n0, const i32x4 (&acc)[G::FM][G::FN],
                                               const float (&fx)[G::FM], const float (&fw)[G::GROUPS][G::COLS],
                                               const float (&bias)[G::GROUPS][G::COLS]) {
  typedef typename Store<DT>::T T;
#pragma unroll
  for (int i = 0; i < G::FM; ++i) {
    const int m = g.row(m0, i);
    if (m < p.M) {
      float resid[G::GROUPS][G::COLS] = {};
      if (p.resid) {
        const T *r = static_cast<const T *>(p.resid) + int64_t(m) * p.ldr + g.col(n0, 0);
#pragma unroll
        for (int q = 0; q < G::GROUPS; ++q) i8_get<DT>(r + q * 32, resid[q]);
      }
      T *out = static_cast<T *>(p.out) + int64_t(m) * p.ldo + g.col(n0, 0);
#pragma unroll
      for (int q = 0; q < G::GROUPS; ++q) {
        float v[G::COLS];
#pragma unroll
        for (int e = 0; e < G::COLS; ++e)
          v[e] = i8_act<ACT>(mul_alone(mul_alone(float(acc[i][q * (G::COLS / 4) + e / 4][e % 4]), fx[i]), fw[q][e]) + bias[q][e]) + resid[q][e];
        i8_put<DT>(out + q * 32, v);
      }
    }
  }
}
template <int DT, typename G>
__device__ __forceinline__ void i8_store_any(const LinearI8 &p, const G &g, int m0, int n0, const i32x4 (&acc)[G::FM][G::FN],
                                             const float (&fx)[G::FM], const float (&fw)[G::GROUPS][G::COLS],
                                             const float (&bias)[G::GROUPS][G::COLS]) {
  typedef typename Store<DT>::T T;
#pragma unroll
  for (int i = 0; i < G::FM; ++i) {
    const int m = g.row(m0, i);
    const Scale sx(fx[i]);
#pragma unroll
    for (int q = 0; q < G::GROUPS; ++q) {
      const int n = g.col(n0, q), left = p.N - n;
      if (m < p.M && left > 0) {
        float v[G::COLS], resid[G::COLS] = {};
        if (p.resid) {
          const T *r = static_cast<const T *>(p.resid) + int64_t(m) * p.ldr + n;
#pragma unroll
          for (int e = 0; e < G::COLS; ++e)
            if (e < left) resid[e] = Store<DT>::dec(r[e]);
        }
#pragma unroll
        for (int e = 0; e < G::COLS; ++e) {
          const Scale sw(fw[q][e]);
          v[e] = __builtin_amdgcn_ldexpf(mul_alone(mul_alone(float(acc[i][q * (G::COLS / 4) + e / 4][e % 4]), sx.f), sw.f), sx.e + sw.e) + bias[q][e];
          v[e] = (p.act == ACT_RELU ? i8_act<ACT_RELU>(v[e]) : p.act == ACT_GELU ? i8_act<ACT_GELU>(v[e]) : v[e]) + resid[e];
        }
        T *out = static_cast<T *>(p.out) + int64_t(m) * p.ldo + n;
        if (left >= G::COLS) {
          i8_put<DT>(out, v);
        } else {
#pragma unroll
          for (int e = 0; e < G::COLS; ++e)
            if (e < left) out[e] = Store<DT>::enc(v[e]);
        }
      }
    }
  }
}
template <int DT, typename G>
__device__ __forceinline__ void i8_store(const LinearI8 &p, const G &g, int m0, int n0, const i32x4 (&acc)[G::FM][G::FN]) {
  typedef typename Store<DT>::T T;
  const bool whole = n0 + (g.wn + 1) * G::WTN <= p.N;
  float fx[G::FM], fw[G::GROUPS][G::COLS], bias[G::GROUPS][G::COLS] = {};
  bool plain = true;
#pragma unroll
  for (int i = 0; i < G::FM; ++i) fx[i] = p.sx[min(g.row(m0, i), p.M - 1)];
#pragma unroll
  for (int q = 0; q < G::GROUPS; ++q) {
    const int n = g.col(n0, q);
    if (whole) {
      i8_get<F32>(p.sw + n, fw[q]);
      if (p.bias) i8_get<DT>(static_cast<const T *>(p.bias) + n, bias[q]);
    } else {
#pragma unroll
      for (int e = 0; e < G::COLS; ++e) {
        fw[q][e] = p.sw[min(n + e, p.N - 1)];
        if (p.bias) bias[q][e] = Store<DT>::dec(static_cast<const T *>(p.bias)[min(n + e, p.N - 1)]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < G::FM; ++i) plain &= plain_scale(fx[i]);
#pragma unroll
  for (int q = 0; q < G::GROUPS; ++q)
#pragma unroll
    for (int e = 0; e < G::COLS; ++e) plain &= plain_scale(fw[q][e]);
  if (whole && __all(plain)) {
    if (p.act == ACT_NONE) i8_store_whole<DT, G, ACT_NONE>(p, g, m0, n0, acc, fx, fw, bias);
    else if (p.act == ACT_RELU) i8_store_whole<DT, G, ACT_RELU>(p, g, m0, n0, acc, fx, fw, bias);
    else i8_store_whole<DT, G, ACT_GELU>(p, g, m0, n0, acc, fx, fw, bias);
  } else {
    i8_store_any<DT, G>(p, g, m0, n0, acc, fx, fw, bias);
  }
}

}  // namespace
}  // namespace mh
