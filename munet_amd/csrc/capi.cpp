// C ABI of libmunet_hip.so (declared in include/munet_hip.h).
//
// Thin layer: validate arguments, translate MuNet's capability-call
// arguments into launcher arguments, enqueue, and turn HIP failures into a
// non-zero status with a thread-local message (the C++ side above maps that
// to std::runtime_error, as MuNet's backends throw, reference
// src/backend/cuda_backend.cu:15-31 for the error convention).
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <stdexcept>
#include <string>
#include <unordered_map>
#include <vector>

#include "../../include/munet_hip.h"
#include "gemm_i8_tiles.hpp"
#include "host_codec.hpp"
#include "mh_kernels.hpp"
#include "mh_runtime.hpp"
#include "paged_index.hpp"

namespace mh {

void hip_check(hipError_t e, const char *what);

namespace {
thread_local std::string g_last_error;

struct DeviceState {
  int *err_flag = nullptr;  // two device ints: embedding index errors, those of the paged cache
  void *workspace = nullptr;
  size_t workspace_bytes = 0;
};
std::mutex g_mu;
std::unordered_map<int, DeviceState> g_devices;

// Fixed scratch for mh_matmul_noalloc: the operand transposes that mh_matmul
// stages in its growable workspace go here instead, so that entry point
// never allocates.  Each GPU the library runs on holds its own copy, at its
// own address, until the process ends.  In host code `scratch` names only
// the host-side shadow of the symbol; device addresses come from
// hipGetSymbolAddress, once per device, and are kept in g_scratch.
constexpr size_t kScratchBytes = size_t(64) << 20;
constexpr int kMaxDevices = 64;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];
void *g_scratch[kMaxDevices] = {};
std::mutex g_scratch_mu;

// The device address of `scratch` on `device` (the current device),
// resolved on first use and kept.
void *scratch_ptr(int device) {
  if (device < 0 || device >= kMaxDevices) throw Error("device ordinal out of range for the scratch table");
  std::lock_guard<std::mutex> lk(g_scratch_mu);
  if (!g_scratch[device]) {
    void *ptr = nullptr;
    hip_check(hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch)), "hipGetSymbolAddress(scratch)");
    if (!ptr) throw Error("hipGetSymbolAddress(scratch) returned no address");
    g_scratch[device] = ptr;
  }
  return g_scratch[device];
}

void check_dt(int dt, bool allow_int = false) {
  if (dt < 0 || dt > 3 || (!allow_int && dt == 3)) throw Error("unsupported dtype code " + std::to_string(dt));
}
}  // namespace

void set_last_error(const std::string &msg) { g_last_error = msg; }

void hip_check(hipError_t e, const char *what) {
  if (e != hipSuccess) throw Error(std::string(what) + ": " + hipGetErrorString(e));
}

int current_device() {
  int d = 0;
  hip_check(hipGetDevice(&d), "hipGetDevice");
  return d;
}

static DeviceState &state() {
  const int d = current_device();
  std::lock_guard<std::mutex> lk(g_mu);
  DeviceState &s = g_devices[d];
  if (!s.err_flag) {
    hip_check(hipMalloc(&s.err_flag, 2 * sizeof(int)), "hipMalloc(error flag)");
    hip_check(hipMemset(s.err_flag, 0, 2 * sizeof(int)), "hipMemset(error flag)");
  }
  return s;
}

int *device_error_flag() { return state().err_flag; }
int *serving_error_flag() { return state().err_flag + 1; }

void *workspace(size_t bytes) {
  DeviceState &s = state();
  std::lock_guard<std::mutex> lk(g_mu);
  if (bytes > s.workspace_bytes) {
    if (s.workspace) {
      hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");
      hip_check(hipFree(s.workspace), "hipFree(workspace)");
      s.workspace = nullptr;
    }
    const size_t rounded = (bytes + (1u << 20) - 1) & ~size_t((1u << 20) - 1);
    hip_check(hipMalloc(&s.workspace, rounded), "hipMalloc(workspace)");
    s.workspace_bytes = rounded;
  }
  return s.workspace;
}

static double g_last_kernel_us = 0.0;
void set_last_kernel_time_us(double us) { g_last_kernel_us = us; }

}  // namespace mh

using namespace mh;

#define MH_TRY(...)                                    \
  try {                                                \
    __VA_ARGS__;                                       \
    return 0;                                          \
  } catch (const std::exception &e) {                  \
    mh::set_last_error(e.what());                      \
    return 1;                                          \
  }

#define S_(p) static_cast<hipStream_t>(p)

namespace {

void bin_call(int dt, int op, const void *a, const void *b, void *out, int ndim, const int *shape, const int64_t *sa,
              const int64_t *sb, void *stream) {
  check_dt(dt);
  if (ndim < 0 || ndim > kMaxDims) throw Error("broadcast rank must be <= 6");
  BcastArgs g;
  g.ndim = ndim;
  g.total = 1;
  for (int d = 0; d < ndim; ++d) {
    if (shape[d] < 0) throw Error("negative dimension");
    g.shape[d] = shape[d];
    g.sa[d] = long(sa[d]);
    g.sb[d] = long(sb[d]);
    g.total *= size_t(shape[d]);
  }
  hip_check(binary(dt, op, a, b, out, g, S_(stream)), "binary");
}

void un_call(int dt, int op, const void *in, void *out, size_t n, void *stream, float c = 0.f) {
  check_dt(dt);
  hip_check(unary(dt, op, in, out, n, c, S_(stream)), "unary");
}

// Bytes of transposed operands a matmul stages: A when transA, B when not
// transB (the NT GEMM reads A [M,K] and B as [N,K]), each slot 256-aligned.
size_t matmul_staging_bytes(int dt, int batch, int M, int K, int N, bool transA, bool transB, long sb) {
  const size_t es = dt_size(dt);
  const size_t nb_b = sb == 0 ? 1 : size_t(batch);
  size_t need = 0;
  if (transA) need += (size_t(batch) * M * K * es + 255) & ~size_t(255);
  if (!transB) need += (nb_b * K * N * es + 255) & ~size_t(255);
  return need;
}

void matmul_check(int dt, int batch, int M, int K, int N) {
  check_dt(dt);
  if (M < 0 || K < 0 || N < 0 || batch < 0) throw Error("matmul: negative size");
}

// A [M,K] (or [K,M] when transA) and B [K,N] (or [N,K] when transB) per
// batch slice -> the NT GEMM's operands, transposing into `ws` (at least
// matmul_staging_bytes, 256-byte aligned).
void matmul_staged(int dt, const void *a, const void *b, void *out, int batch, int M, int K, int N, bool transA,
                   bool transB, long sa, long sb, long sc, char *ws, void *stream) {
  const size_t es = dt_size(dt);
  const int nb_b = sb == 0 ? 1 : batch;
  const void *A = a, *Bt = b;
  long lsa = sa, lsb = sb;
  if (transA) {
    // per-slice [K,M] -> [M,K]; slices may be strided, so one launch each
    // unless they are packed back to back
    char *dst = ws;
    if (sa == long(M) * K || batch == 1) {
      hip_check(transpose2d(dt, a, dst, batch, K, M, S_(stream)), "transpose A");
    } else {
      for (int z = 0; z < batch; ++z)
        hip_check(transpose2d(dt, static_cast<const char *>(a) + size_t(z) * sa * es, dst + size_t(z) * M * K * es,
                              1, K, M, S_(stream)),
                  "transpose A");
    }
    A = dst;
    lsa = long(M) * K;
    ws += (size_t(batch) * M * K * es + 255) & ~size_t(255);
  }
  if (!transB) {
    char *dst = ws;
    if (sb == 0 || sb == long(K) * N || nb_b == 1) {
      hip_check(transpose2d(dt, b, dst, nb_b, K, N, S_(stream)), "transpose B");
    } else {
      for (int z = 0; z < nb_b; ++z)
        hip_check(transpose2d(dt, static_cast<const char *>(b) + size_t(z) * sb * es, dst + size_t(z) * K * N * es,
                              1, K, N, S_(stream)),
                  "transpose B");
    }
    Bt = dst;
    lsb = sb == 0 ? 0 : long(K) * N;
  }
  EpiArgs ep;
  ep.out = out;
  ep.ldc = N;
  hip_check(gemm_nt(dt, A, Bt, M, N, K, K, K, batch, lsa, lsb, sc, ep, -1, S_(stream)), "gemm");
}

void matmul_call(int dt, const void *a, const void *b, void *out, int batch, int M, int K, int N, bool transA,
                 bool transB, long sa, long sb, long sc, void *stream) {
  matmul_check(dt, batch, M, K, N);
  if (M == 0 || N == 0 || batch == 0) return;
  const size_t need = matmul_staging_bytes(dt, batch, M, K, N, transA, transB, sb);
  char *ws = need ? static_cast<char *>(workspace(need)) : nullptr;
  matmul_staged(dt, a, b, out, batch, M, K, N, transA, transB, sa, sb, sc, ws, stream);
}

}  // namespace

namespace {

void aligned16(const void *p, const char *what) {
  if (reinterpret_cast<uintptr_t>(p) % 16) throw Error(std::string(what) + " must be 16-byte aligned");
}
void check_page(const char *op, int page, int n_pages) {
  if (page < kPageMin || page > kPageMax || (page & (page - 1)))
    throw Error(std::string(op) + ": a page holds 16, 32, 64, 128 or 256 tokens");
  if (n_pages < 1 || int64_t(n_pages) * page > 0x7fffffff) throw Error(std::string(op) + ": the pool must hold 1 to 2^31 - 1 tokens");
}
void check_pool(const char *op, const void *kc, const void *vc, const void *ks, const void *vs, int Hkv, int hd, int page,
                int n_pages) {
  check_page(op, page, n_pages);
  if (Hkv < 1 || Hkv > 65535) throw Error(std::string(op) + ": bad key/value head count");
  if (hd < 16 || hd > kPagedHeadMax || hd % 16) throw Error(std::string(op) + ": head_dim must be a multiple of 16, at most 256");
  if (!kc || !vc || !ks || !vs) throw Error(std::string(op) + ": null cache");
  aligned16(kc, "k_cache");
  aligned16(vc, "v_cache");
}
void check_rows(const char *op, const char *what, int dt, const void *p, int64_t ld, int64_t cols) {
  if (!p) throw Error(std::string(op) + ": null " + what);
  aligned16(p, what);
  if (ld < cols || ld * int64_t(dt_size(dt)) % 16)
    throw Error(std::string(op) + ": rows of " + what + " must be whole, a multiple of 16 bytes apart");
}
// n rows of cols elements, ld apart, aligned to their type.
void check_whole_rows(const char *op, const char *what, size_t es, const void *p, int64_t n, int64_t ld, int64_t cols) {
  if (!p) throw Error(std::string(op) + ": null " + what);
  if (reinterpret_cast<uintptr_t>(p) % es) throw Error(std::string(op) + ": " + what + " must be aligned to its type");
  if (ld < cols) throw Error(std::string(op) + ": rows of " + what + " must be whole");
  if (ld > (int64_t(1) << 56) / n) throw Error(std::string(op) + ": rows of " + what + " too far apart");
}
// Whether two sets of rows share a byte; sets of the same spacing that lie beside
// each other (columns of one buffer) do not.
struct RowSet {
  const void *p;
  int64_t rows, ld, cols;  // (in bytes)
};
bool rows_meet(const RowSet &a, const RowSet &b) {
  if (!a.p || !b.p || a.rows < 1 || b.rows < 1 || a.cols < 1 || b.cols < 1) return false;
  const uintptr_t x = reinterpret_cast<uintptr_t>(a.p), y = reinterpret_cast<uintptr_t>(b.p);
  const uintptr_t xe = x + uintptr_t((a.rows - 1) * a.ld + a.cols), ye = y + uintptr_t((b.rows - 1) * b.ld + b.cols);
  if (xe <= y || ye <= x) return false;
  if (a.rows > 1 && b.rows > 1 && a.ld == b.ld) {
    const uintptr_t d = (y >= x ? (y - x) : uintptr_t(a.ld) - (x - y) % uintptr_t(a.ld)) % uintptr_t(a.ld);
    return d < uintptr_t(a.cols) || uintptr_t(a.ld) - d < uintptr_t(b.cols);
  }
  return true;
}
// n bytes from p, as one row
RowSet whole(const void *p, int64_t n) { return {p, 1, n, n}; }
void check_rotation(const char *op, const float *table, int hd, int half) {
  if (half < 1 || hd < 1 || half > hd / 2) throw Error(std::string(op) + ": the rotated part must be 2 values at least and fit the head");
  if (!table) throw Error(std::string(op) + ": null table");
  aligned16(table, "table");
}
void check_sample_size(int rows, int cols) {
  if (rows < 0 || cols < 1) throw Error("sample: bad row count or empty rows");
  if (rows >= 1 << 22) throw Error("sample: more rows than one launch takes (2^22 - 1)");
  if (cols > kSampleMaxCols) throw Error("sample: more tokens than indexes of 32 bits go round (2^31 - 2^21)");
}
// The cut of an attention_paged call, its sizes checked.
PagedShape paged_call_shape(int dt, int B, int n_rows, int Hq, int Hkv, int hd, int max_q, int max_len, int window) {
  check_dt(dt);
  if (B < 0 || n_rows < 0 || max_q < 0 || max_len < 0 || window < 0) throw Error("attention_paged: negative size");
  if (Hkv < 1 || Hq < 1 || Hq % Hkv) throw Error("attention_paged: query heads must be a multiple of key/value heads");
  if (hd < 16 || hd > kPagedHeadMax || hd % 16) throw Error("attention_paged: head_dim must be a multiple of 16, at most 256");
  if (int64_t(n_rows) * Hq > (1 << 30)) throw Error("attention_paged: more than 2^30 query rows");
  if (int64_t(B) * Hkv > kPagedMaxBlocks) throw Error("attention_paged: more requests times key/value heads than one launch takes (2^23 - 1)");
  PagedShape s = paged_shape(B, Hq, Hkv, std::min(max_q, n_rows), max_len, window);
  // (a batch padded with more rows than one launch joins: no shares)
  if (s.splits > 1 && int64_t(n_rows) * Hq > kJoinMaxBlocks * join_shape(hd, s.splits).rows) s.splits = 1;
  return s;
}

}  // namespace

extern "C" {

const char *mh_last_error(void) { return mh::g_last_error.c_str(); }
const char *mh_version(void) { return "munet-hip 0.1 (gfx950)"; }

int mh_query_support(int feature, int dtype, int *available, int *fallback_policy, int *accumulation_dtype) {
  MH_TRY({
    check_dt(dtype, true);
    if (!available || !fallback_policy || !accumulation_dtype) throw Error("query_support: null output");
    const bool fp = dtype != MH_I32;
    bool ok = false;
    switch (feature) {
    // the float products, elementwise, activation, normalisation and spatial
    // kernels: fp32, fp16 and bf16 storages
    case MH_FEATURE_ELEMENTWISE_BINARY:
    case MH_FEATURE_MATMUL:
    case MH_FEATURE_UNARY_ACTIVATION:
    case MH_FEATURE_SOFTMAX:
    case MH_FEATURE_CONVOLUTION:
    case MH_FEATURE_POOLING:
    case MH_FEATURE_LAYER_NORM:
    case MH_FEATURE_ATTENTION:
    case MH_FEATURE_EMBEDDING:
    case MH_FEATURE_MASKED_FILL:
      ok = fp;
      break;
    // data movement: any storage, int32 included (broadcast_row runs as a
    // strided gather with a zero row stride)
    case MH_FEATURE_BROADCAST_ROW:
    case MH_FEATURE_CONCAT:
    case MH_FEATURE_TO_CONTIGUOUS:
      ok = true;
      break;
    // training-only capabilities and the reductions are not part of the
    // inference path: unavailable, never silently sent to the CPU
    default:
      ok = false;
      break;
    }
    *available = ok ? 1 : 0;
    *fallback_policy = MH_POLICY_EXPLICIT_UNSUPPORTED;
    *accumulation_dtype = MH_F32;
  })
}

int mh_device_count(int *count) {
  MH_TRY({
    int n = 0;
    if (hipGetDeviceCount(&n) != hipSuccess) n = 0;
    *count = n;
  })
}

int mh_init(int device) {
  MH_TRY({
    hip_check(hipSetDevice(device), "hipSetDevice");
    (void)state();
    (void)scratch_ptr(device);
  })
}

int mh_check_device_errors(void) {
  MH_TRY({
    int *flag = device_error_flag();
    int both[2] = {0, 0};
    hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");
    hip_check(hipMemcpy(both, flag, sizeof both, hipMemcpyDeviceToHost), "hipMemcpy(error flag)");
    const int h = both[0] | both[1];
    if (h) {
      hip_check(hipMemset(flag, 0, sizeof both), "hipMemset(error flag)");
      // all that is set: one error often brings the next
      std::string told;
      auto tell = [&](int bit, const char *what) {
        if (h & bit) told += std::string(told.empty() ? "" : "; ") + what;
      };
      tell(kErrEmbedding, "Embedding index out of range");
      tell(kErrPlan, "page_plan: out of free pages, table width or slots");
      tell(kErrPage, "paged KV cache: page, slot or length out of range");
      throw Error(told.empty() ? "device error flag set" : told);
    }
  })
}

// ---- allocation / transfer -------------------------------------------------
int mh_allocate(void **ptr, size_t bytes) {
  MH_TRY({
    *ptr = nullptr;
    if (bytes) hip_check(hipMalloc(ptr, bytes), "hipMalloc");
  })
}
int mh_deallocate(void *ptr) { MH_TRY(if (ptr) hip_check(hipFree(ptr), "hipFree")) }
int mh_memset(void *ptr, int value, size_t bytes, void *stream) {
  MH_TRY(if (bytes) hip_check(hipMemsetAsync(ptr, value, bytes, S_(stream)), "hipMemsetAsync"))
}
int mh_copy(const void *src, void *dst, size_t bytes, int src_dev, int dst_dev, void *stream) {
  MH_TRY({
    if (bytes > 0 && (!src || !dst)) throw Error("hip copy: null pointer with non-zero byte count");
    if (!bytes) return 0;
    hipMemcpyKind kind;
    if (src_dev == MH_DEVICE_CPU && dst_dev == MH_DEVICE_CPU) kind = hipMemcpyHostToHost;
    else if (src_dev == MH_DEVICE_CPU) kind = hipMemcpyHostToDevice;
    else if (dst_dev == MH_DEVICE_CPU) kind = hipMemcpyDeviceToHost;
    else kind = hipMemcpyDeviceToDevice;
    hip_check(hipMemcpyAsync(dst, src, bytes, kind, S_(stream)), "hipMemcpyAsync");
    if (kind == hipMemcpyDeviceToHost || kind == hipMemcpyHostToDevice)
      hip_check(hipStreamSynchronize(S_(stream)), "hipStreamSynchronize");
  })
}
int mh_synchronize(void *stream) {
  MH_TRY({
    if (stream) hip_check(hipStreamSynchronize(S_(stream)), "hipStreamSynchronize");
    else hip_check(hipDeviceSynchronize(), "hipDeviceSynchronize");
  })
}
double mh_get_last_kernel_time_us(void) { return mh::g_last_kernel_us; }

int mh_to_contiguous(int dt, const void *src, void *dst, int ndim, const int *shape, const int64_t *strides,
                     int64_t offset, void *stream) {
  MH_TRY({
    check_dt(dt, true);
    if (ndim < 0 || ndim > kMaxDims) throw Error("to_contiguous: rank must be <= 6");
    StridedArgs g;
    g.ndim = ndim;
    g.offset = long(offset);
    g.total = 1;
    for (int d = 0; d < ndim; ++d) {
      g.shape[d] = shape[d];
      g.strides[d] = long(strides[d]);
      g.total *= size_t(shape[d]);
    }
    hip_check(to_contiguous(dt, src, dst, g, S_(stream)), "to_contiguous");
  })
}

// ---- elementwise -----------------------------------------------------------
int mh_add(int dt, const void *a, const void *b, void *out, int ndim, const int *shape, const int64_t *sa,
           const int64_t *sb, void *stream) {
  MH_TRY(bin_call(dt, BIN_ADD, a, b, out, ndim, shape, sa, sb, stream))
}
int mh_sub(int dt, const void *a, const void *b, void *out, int ndim, const int *shape, const int64_t *sa,
           const int64_t *sb, void *stream) {
  MH_TRY(bin_call(dt, BIN_SUB, a, b, out, ndim, shape, sa, sb, stream))
}
int mh_mul(int dt, const void *a, const void *b, void *out, int ndim, const int *shape, const int64_t *sa,
           const int64_t *sb, void *stream) {
  MH_TRY(bin_call(dt, BIN_MUL, a, b, out, ndim, shape, sa, sb, stream))
}
int mh_div(int dt, const void *a, const void *b, void *out, int ndim, const int *shape, const int64_t *sa,
           const int64_t *sb, void *stream) {
  MH_TRY(bin_call(dt, BIN_DIV, a, b, out, ndim, shape, sa, sb, stream))
}
int mh_relu(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_RELU, in, out, n, stream)) }
int mh_sigmoid(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_SIGMOID, in, out, n, stream)) }
int mh_exp(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_EXP, in, out, n, stream)) }
int mh_log(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_LOG, in, out, n, stream)) }
int mh_sqrt(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_SQRT, in, out, n, stream)) }
int mh_rsqrt(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_RSQRT, in, out, n, stream)) }
int mh_sin(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_SIN, in, out, n, stream)) }
int mh_cos(int dt, const void *in, void *out, size_t n, void *stream) { MH_TRY(un_call(dt, UN_COS, in, out, n, stream)) }
int mh_gelu(int dt, const void *in, void *out, size_t n, void *stream) {
  MH_TRY(un_call(dt, UN_GELU, in, out, n, stream, host_round(dt, 1.702f)))
}
int mh_softmax(int dt, const void *in, void *out, int batch, int classes, void *stream) {
  MH_TRY({
    check_dt(dt);
    hip_check(softmax_rows(dt, in, out, batch, classes, S_(stream)), "softmax");
  })
}
int mh_masked_fill(int dt, const void *x, const int32_t *mask, void *out, size_t n, double value, void *stream) {
  MH_TRY({
    check_dt(dt);
    // the fill value is written through the dtype codec (-1e9 -> -inf in fp16)
    hip_check(masked_fill(dt, x, mask, out, n, float(value), S_(stream)), "masked_fill");
  })
}
int mh_layer_norm(int dt, const void *x, const void *w, const void *b, void *out, int rows, int cols, float eps,
                  void *stream) {
  MH_TRY({
    check_dt(dt);
    hip_check(layernorm(dt, x, w, b, out, rows, cols, eps, S_(stream)), "layer_norm");
  })
}
int mh_embedding(int dt, const int32_t *ids, const void *w, void *out, int n, int V, int D, void *stream) {
  MH_TRY({
    check_dt(dt);
    hip_check(embedding(dt, ids, w, nullptr, out, n, V, D, 1, device_error_flag(), S_(stream)), "embedding");
  })
}
int mh_embedding_pos(int dt, const int32_t *ids, const void *tok_w, const void *pos_w, void *out, int n, int V, int D,
                     int T, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (T <= 0) throw Error("embedding_pos: T must be positive");
    hip_check(embedding(dt, ids, tok_w, pos_w, out, n, V, D, T, device_error_flag(), S_(stream)), "embedding");
  })
}
int mh_convert(int sdt, const void *in, int ddt, void *out, size_t n, void *stream) {
  MH_TRY({
    check_dt(sdt, true);
    check_dt(ddt, true);
    hip_check(convert(sdt, in, ddt, out, n, S_(stream)), "convert");
  })
}
int mh_check_f16_rounding(unsigned long long *mismatches, void *stream) {
  MH_TRY({
    if (!mismatches) throw Error("check_f16_rounding: mismatches must be set");
    hip_check(check_f16_rounding(mismatches, S_(stream)), "check_f16_rounding");
  })
}
int mh_argmax(int dt, const void *x, int32_t *out, int rows, int cols, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (cols <= 0) throw Error("argmax: empty rows");
    hip_check(argmax_rows(dt, x, out, rows, cols, S_(stream)), "argmax");
  })
}
int mh_measure_mfma_peak(int dt, int iters, double *flops_per_s, void *stream) {
  MH_TRY({
    if (dt != MH_BF16 && dt != MH_F16) throw Error("measure_mfma_peak: dtype must be bfloat16 or float16");
    if (iters <= 0 || !flops_per_s) throw Error("measure_mfma_peak: iters must be positive and flops_per_s set");
    hip_check(mfma_peak(dt, iters, flops_per_s, S_(stream)), "measure_mfma_peak");
  })
}
int mh_measure_hbm_read(const void *buf, size_t bytes, int reps, double *bytes_per_s, void *stream) {
  MH_TRY({
    if (!buf || bytes < (size_t(1) << 20) || reps <= 0 || !bytes_per_s || (uintptr_t)buf % 16)
      throw Error("measure_hbm_read: needs a 16-byte aligned buffer of at least 1 MiB, reps > 0 and bytes_per_s");
    hip_check(hbm_read_rate(buf, bytes, reps, bytes_per_s, S_(stream)), "measure_hbm_read");
  })
}

// ---- blas ------------------------------------------------------------------
int mh_matmul(int dt, const void *a, const void *b, void *out, int M, int K, int N, int transA, int transB,
              void *stream) {
  MH_TRY(matmul_call(dt, a, b, out, 1, M, K, N, transA != 0, transB != 0, 0, 0, 0, stream))
}
int mh_matmul_noalloc(int dt, const void *a, const void *b, void *out, int M, int K, int N, int transA, int transB,
                      void *stream) {
  MH_TRY({
    matmul_check(dt, 1, M, K, N);
    if (M == 0 || N == 0) return 0;
    const size_t need = matmul_staging_bytes(dt, 1, M, K, N, transA != 0, transB != 0, 0);
    if (need > kScratchBytes)
      throw Error("matmul_noalloc: the transposed operands need " + std::to_string(need) + " bytes of scratch, " +
                  "more than its fixed " + std::to_string(kScratchBytes) + " bytes");
    char *ws = nullptr;
    if (need) {
      int dev = 0;
      hip_check(hipGetDevice(&dev), "hipGetDevice");
      ws = static_cast<char *>(scratch_ptr(dev));
    }
    matmul_staged(dt, a, b, out, 1, M, K, N, transA != 0, transB != 0, 0, 0, 0, ws, stream);
  })
}
int mh_batched_matmul(int dt, const void *a, const void *b, void *out, int batch, int M, int K, int N, int transA,
                      int transB, int64_t sa, int64_t sb, int64_t sc, void *stream) {
  MH_TRY(matmul_call(dt, a, b, out, batch, M, K, N, transA != 0, transB != 0, long(sa), long(sb), long(sc), stream))
}
int mh_linear(int dt, const void *x, const void *w_t, const void *bias, void *out, int M, int K, int N, int act,
              const void *resid, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (act < 0 || act > 2) throw Error("linear: bad activation code");
    EpiArgs ep;
    ep.out = out;
    ep.ldc = N;
    ep.bias = bias;
    ep.act = act;
    ep.gelu_c = host_round(dt, 1.702f);
    ep.resid = resid;
    ep.ldr = N;
    hip_check(gemm_nt(dt, x, w_t, M, N, K, K, K, 1, 0, 0, 0, ep, -1, S_(stream)), "linear");
  })
}
int mh_pack_linear_weight(int dt, const void *w, void *w_t, int in_f, int out_f, void *stream) {
  MH_TRY({
    check_dt(dt);
    hip_check(transpose2d(dt, w, w_t, 1, in_f, out_f, S_(stream)), "pack_linear_weight");
  })
}
int mh_qkv_projection(int dt, const void *x, const void *wqkv_t, const void *bqkv, void *q, void *k, void *v, int B,
                      int T, int E, int H, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (H <= 0 || E % H != 0) throw Error("qkv_projection: embed_dim must be divisible by num_heads");
    const int hd = E / H;
    if (hd % 4 != 0) throw Error("qkv_projection: head_dim must be a multiple of 4");
    EpiArgs ep;
    ep.mode = EPI_HEADSPLIT;
    ep.outs[0] = q;
    ep.outs[1] = k;
    ep.outs[2] = v;
    ep.bias = bqkv;
    ep.T = T;
    ep.H = H;
    ep.hd = hd;
    ep.E = E;
    hip_check(gemm_nt(dt, x, wqkv_t, B * T, 3 * E, E, E, E, 1, 0, 0, 0, ep, -1, S_(stream)), "qkv_projection");
  })
}

// ---- attention ---------------------------------------------------------------
int mh_attention(int dt, const void *q, const void *k, const void *v, void *ctx, int B, int H, int T, int hd,
                 int causal, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (hd <= 0) throw Error("attention: head_dim must be positive");
    if (size_t(T) * 4 > 64 * 1024 && !(hd == 64 && dt != MH_F32))
      throw Error("attention: sequence too long for the generic kernel");
    const float scale = host_round(dt, 1.0f / std::sqrt(float(hd)));
    hip_check(attention(dt, q, k, v, ctx, B, H, T, hd, causal, scale, 0, S_(stream)), "attention");
  })
}

int mh_attention_textbook(int dt, const void *q, const void *k, const void *v, void *ctx, int B, int H, int T, int hd,
                          int causal, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (hd <= 0) throw Error("attention: head_dim must be positive");
    if (size_t(T) * 4 > 64 * 1024 && !(hd == 64 && dt != MH_F32))
      throw Error("attention: sequence too long for the generic kernel");
    const float scale = host_round(dt, 1.0f / std::sqrt(float(hd)));
    hip_check(attention(dt, q, k, v, ctx, B, H, T, hd, causal, scale, 0, S_(stream), 1), "attention_textbook");
  })
}

// ---- paged KV cache ----------------------------------------------------------
int mh_page_plan(const int32_t *lens, const int32_t *new_lens, const int32_t *free_pages, int32_t *tables,
                 int32_t *total_lens, int32_t *cu, int32_t *slots, int32_t *positions, int32_t *used, int B, int n_free,
                 int width, int page, int n_pages, int n_slots, void *stream) {
  MH_TRY({
    check_page("page_plan", page, n_pages);
    if (B < 0 || n_free < 0 || width < 0 || n_slots < 0) throw Error("page_plan: negative size");
    if (B > kPlanMaxRequests) throw Error("page_plan: more requests than one launch takes (2^20)");
    if (int64_t(width) * page > kPagedMaxKeys) throw Error("page_plan: a table row must hold at most 2^31 - 4096 tokens");
    if (B == 0) return 0;
    if (!lens || !new_lens || !total_lens || !cu || !used || (width && !tables) || (n_free && !free_pages) ||
        (n_slots && !slots))
      throw Error("page_plan: null argument");
    {  // (requests read those before them while others write)
      struct Range {
        const void *at;
        int64_t n;
      };
      const Range in[] = {{lens, B}, {new_lens, B}, {free_pages, n_free}},
                  out[] = {{tables, int64_t(B) * width}, {total_lens, B}, {cu, int64_t(B) + 1}, {slots, n_slots}, {positions, n_slots}, {used, 1}};
      auto meet = [](const Range &x, const Range &y) {
        const uintptr_t a = reinterpret_cast<uintptr_t>(x.at), b = reinterpret_cast<uintptr_t>(y.at);
        return a && b && a < b + 4 * uintptr_t(y.n) && b < a + 4 * uintptr_t(x.n);
      };
      for (const Range &o : out) {
        for (const Range &i : in)
          if (meet(o, i)) throw Error("page_plan: an output overlaps an input");
        for (const Range &other : out)
          if (&other != &o && meet(o, other)) throw Error("page_plan: two outputs overlap");
      }
    }
    PagePlan p;
    p.lens = lens;
    p.fresh = new_lens;
    p.free_pages = free_pages;
    p.tables = tables;
    p.total = total_lens;
    p.cu = cu;
    p.slots = slots;
    p.positions = positions;
    p.used = used;
    p.B = B;
    p.n_free = n_free;
    p.width = width;
    p.page = page;
    p.n_pages = n_pages;
    p.cap = n_slots;
    hip_check(page_plan(p, serving_error_flag(), S_(stream)), "page_plan");
  })
}
int mh_kv_store_paged(int dt, const void *k, const void *v, int64_t ldk, int64_t ldv, const int32_t *slots,
                      void *k_cache, void *v_cache, float *k_scale, float *v_scale, int n, int Hkv, int hd, int page,
                      int n_pages, void *stream) {
  MH_TRY({
    check_dt(dt);
    check_pool("kv_store_paged", k_cache, v_cache, k_scale, v_scale, Hkv, hd, page, n_pages);
    if (n < 0) throw Error("kv_store_paged: negative size");
    if (n > 1 << 27) throw Error("kv_store_paged: more tokens than one launch takes (2^27)");
    if (n == 0) return 0;
    if (!slots) throw Error("kv_store_paged: null slots");
    check_rows("kv_store_paged", "k", dt, k, ldk, int64_t(Hkv) * hd);
    check_rows("kv_store_paged", "v", dt, v, ldv, int64_t(Hkv) * hd);
    hip_check(kv_store_paged(dt, k, v, long(ldk), long(ldv), slots, k_cache, v_cache, k_scale, v_scale, n, Hkv, hd, page, n_pages,
                             serving_error_flag(), S_(stream)),
              "kv_store_paged");
  })
}
int mh_attention_paged_workspace(int dt, int B, int n_rows, int Hq, int Hkv, int hd, int max_q, int max_len, int window,
                                 size_t *bytes) {
  MH_TRY({
    if (!bytes) throw Error("attention_paged_workspace: null output");
    const PagedShape s = paged_call_shape(dt, B, n_rows, Hq, Hkv, hd, max_q, max_len, window);
    *bytes = B && n_rows ? paged_workspace_bytes(n_rows, Hq, hd, s.splits) : 0;
  })
}
int mh_attention_paged(int dt, const void *q, int64_t ldq, const void *k_cache, const void *v_cache, const float *k_scale,
                       const float *v_scale, const int32_t *tables, const int32_t *lens, const int32_t *cu, void *out,
                       int64_t ldo, int B, int n_rows, int Hq, int Hkv, int hd, int page, int n_pages, int width, int max_q,
                       int max_len, int causal, int window, float scale, void *workspace, size_t workspace_bytes,
                       void *stream) {
  MH_TRY({
    const PagedShape s = paged_call_shape(dt, B, n_rows, Hq, Hkv, hd, max_q, max_len, window);
    check_pool("attention_paged", k_cache, v_cache, k_scale, v_scale, Hkv, hd, page, n_pages);
    if (width < 0 || int64_t(width) * page > kPagedMaxKeys)
      throw Error("attention_paged: a table row must hold at most 2^31 - 4096 tokens");
    // (its product with log2(e) is a float)
    if (!(std::fabs(scale) <= 0x1p127f)) throw Error("attention_paged: the scale must be finite, of at most 2^127");
    if (B == 0 || n_rows == 0) return 0;
    if (!lens || !cu || (width && !tables)) throw Error("attention_paged: null argument");
    check_rows("attention_paged", "q", dt, q, ldq, int64_t(Hq) * hd);
    check_rows("attention_paged", "out", dt, out, ldo, int64_t(Hq) * hd);
    const size_t need = paged_workspace_bytes(n_rows, Hq, hd, s.splits);
    if (need > workspace_bytes || (need && !workspace))
      throw Error("attention_paged: needs a workspace of " + std::to_string(need) + " bytes, got " + std::to_string(workspace_bytes));
    if (need) aligned16(workspace, "workspace");
    PagedAttention p;
    p.q = q;
    p.out = out;
    p.k_cache = k_cache;
    p.v_cache = v_cache;
    p.k_scale = k_scale;
    p.v_scale = v_scale;
    p.tables = tables;
    p.lens = lens;
    p.cu = cu;
    p.workspace = workspace;
    p.err = serving_error_flag();
    p.ldq = long(ldq);
    p.ldo = long(ldo);
    p.B = B;
    p.Hq = Hq;
    p.Hkv = Hkv;
    p.hd = hd;
    p.page = page;
    p.n_pages = n_pages;
    p.n_rows = n_rows;
    p.width = width;
    p.causal = causal != 0;
    p.window = window;
    p.scale = scale == 0.f ? float(1.0 / std::sqrt(double(hd))) : scale;
    hip_check(attention_paged(dt, p, s, S_(stream)), "attention_paged");
  })
}

// ---- rotary positions ----------------------------------------------------------
int mh_rotary_frequencies(double *freq, double *magnitude, int rot, double base, int scaling, double factor, double original,
                          double low, double high) {
  MH_TRY({
    if (!freq) throw Error("rotary_frequencies: null freq");
    if (rot < 2 || rot % 2) throw Error("rotary_frequencies: the rotated part must be an even number of values");
    if (!(base > 0) || !std::isfinite(base)) throw Error("rotary_frequencies: the base must be positive");
    if (scaling < MH_ROTARY_PLAIN || scaling > MH_ROTARY_TURNS) throw Error("rotary_frequencies: unknown scaling");
    if (scaling != MH_ROTARY_PLAIN && (!(factor > 0) || !std::isfinite(factor)))
      throw Error("rotary_frequencies: the factor must be positive");
    if (scaling == MH_ROTARY_BASE && rot < 4) throw Error("rotary_frequencies: a changed base needs a rotated part of 4 at least");
    if (scaling == MH_ROTARY_TURNS && (!(original > 0) || !std::isfinite(original) || !(low >= 0) || !(high > low) || !std::isfinite(high)))
      throw Error("rotary_frequencies: needs original > 0 and 0 <= low < high");
    if (scaling == MH_ROTARY_BASE) base *= std::pow(factor, double(rot) / (rot - 2));
    if (!(base > 0) || !std::isfinite(base)) throw Error("rotary_frequencies: the changed base is out of range");
    for (int j = 0; j < rot / 2; ++j) {
      double f = std::pow(base, -2.0 * j / rot);
      if (scaling == MH_ROTARY_LINEAR) f /= factor;
      if (scaling == MH_ROTARY_TURNS) {
        const double r = original * f / (2 * M_PI), g = std::min(1.0, std::max(0.0, (r - low) / (high - low)));
        f = g * f + (1 - g) * f / factor;
      }
      if (!std::isfinite(f)) throw Error("rotary_frequencies: a frequency is out of range");
      freq[j] = f;
    }
    if (magnitude) *magnitude = scaling == MH_ROTARY_TURNS && factor > 1 ? 1 + 0.1 * std::log(factor) : 1.0;
  })
}
int mh_rotary_table(const int32_t *positions, const double *freq, float *table, int n, int half, double magnitude, void *stream) {
  MH_TRY({
    if (n < 0) throw Error("rotary_table: negative size");
    if (half < 1) throw Error("rotary_table: no pairs");
    if (n == 0) return 0;
    if (!positions || !freq || !table) throw Error("rotary_table: null argument");
    aligned16(table, "table");
    if (int64_t(n) * half > int64_t(1) << 56) throw Error("rotary_table: table larger than any memory");
    const RowSet o = whole(table, int64_t(n) * half * 8);
    if (rows_meet(o, whole(positions, int64_t(n) * 4)) || rows_meet(o, whole(freq, int64_t(half) * 8)))
      throw Error("rotary_table: table overlaps positions or freq");
    hip_check(rotary_table(positions, freq, table, n, half, magnitude, S_(stream)), "rotary_table");
  })
}
int mh_rotary(int dt, const void *x, int64_t ldx, const float *table, void *out, int64_t ldo, int n, int heads, int hd, int half,
              int interleaved, int inverse, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (n < 0) throw Error("rotary: negative size");
    if (heads < 1 || hd < 1 || int64_t(heads) * hd > 1 << 30) throw Error("rotary: bad head count or size");
    if (n == 0) return 0;
    check_rotation("rotary", table, hd, half);
    const int64_t es = int64_t(dt_size(dt)), cols = int64_t(heads) * hd;
    check_whole_rows("rotary", "x", es, x, n, ldx, cols);
    check_whole_rows("rotary", "out", es, out, n, ldo, cols);
    if (!(x == out && (ldx == ldo || n == 1)) && rows_meet({x, n, ldx * es, cols * es}, {out, n, ldo * es, cols * es}))
      throw Error("rotary: out overlaps x without being it");
    if (rows_meet({out, n, ldo * es, cols * es}, whole(table, int64_t(n) * half * 8))) throw Error("rotary: out overlaps table");
    Rotary p;
    p.x = x;
    p.out = out;
    p.table = table;
    p.ldx = ldx;
    p.ldo = ldo;
    p.n = n;
    p.heads = heads;
    p.hd = hd;
    p.half = half;
    p.interleaved = interleaved != 0;
    p.inverse = inverse != 0;
    hip_check(rotary(dt, p, nullptr, 0, S_(stream)), "rotary");
  })
}
int mh_kv_store_rotary_paged(int dt, const void *k, const void *v, int64_t ldk, int64_t ldv, const float *table,
                             const int32_t *slots, void *k_cache, void *v_cache, float *k_scale, float *v_scale, int n, int Hkv,
                             int hd, int half, int interleaved, int page, int n_pages, const void *q, int64_t ldq, void *q_out,
                             int64_t ldqo, int Hq, void *stream) {
  MH_TRY({
    const char *op = "kv_store_rotary_paged";
    check_dt(dt);
    check_pool(op, k_cache, v_cache, k_scale, v_scale, Hkv, hd, page, n_pages);
    if (Hkv > 65534) throw Error("kv_store_rotary_paged: bad key/value head count");
    if (n < 0) throw Error("kv_store_rotary_paged: negative size");
    if (n > 1 << 27) throw Error("kv_store_rotary_paged: more tokens than one launch takes (2^27)");
    if (q && (Hq < 1 || int64_t(Hq) * hd > 1 << 30)) throw Error("kv_store_rotary_paged: bad query head count");
    if (n == 0) return 0;
    if (!slots) throw Error("kv_store_rotary_paged: null slots");
    check_rotation(op, table, hd, half);
    check_rows(op, "k", dt, k, ldk, int64_t(Hkv) * hd);
    check_rows(op, "v", dt, v, ldv, int64_t(Hkv) * hd);
    const int64_t es = int64_t(dt_size(dt)), kcols = int64_t(Hkv) * hd * es, angles = int64_t(n) * half * 8;
    const RowSet kr{k, n, ldk * es, kcols}, vr{v, n, ldv * es, kcols};
    RowSet qr{nullptr, 0, 0, 0}, o = qr;
    for (int64_t ld : {ldk, ldv})
      if (ld > (int64_t(1) << 56) / n) throw Error("kv_store_rotary_paged: rows too far apart");
    Rotary p;
    p.table = table;
    p.n = n;
    p.hd = hd;
    p.half = half;
    p.interleaved = interleaved != 0;
    if (q) {
      const int64_t cols = int64_t(Hq) * hd * es;
      check_rows(op, "q", dt, q, ldq, int64_t(Hq) * hd);
      check_rows(op, "q_out", dt, q_out, ldqo, int64_t(Hq) * hd);
      for (int64_t ld : {ldq, ldqo})
        if (ld > (int64_t(1) << 56) / n) throw Error("kv_store_rotary_paged: rows too far apart");
      qr = {q, n, ldq * es, cols};
      o = {q_out, n, ldqo * es, cols};
      if ((!(q == q_out && (ldq == ldqo || n == 1)) && rows_meet(o, qr)) || rows_meet(o, kr) || rows_meet(o, vr))
        throw Error("kv_store_rotary_paged: q_out overlaps q without being it, or k or v");
      if (rows_meet(o, whole(table, angles)) || rows_meet(o, whole(slots, int64_t(n) * 4)))
        throw Error("kv_store_rotary_paged: q_out overlaps table or slots");
      p.x = q;
      p.out = q_out;
      p.ldx = ldq;
      p.ldo = ldqo;
      p.heads = Hq;
    }
    const int64_t pool = int64_t(n_pages) * Hkv * page * hd, scales = int64_t(n_pages) * Hkv * 4;
    const RowSet held[] = {whole(k_cache, pool), whole(v_cache, pool), whole(k_scale, scales), whole(v_scale, scales)};
    for (const RowSet &h : held) {
      for (const RowSet &x : {kr, vr, qr, o, whole(table, angles), whole(slots, int64_t(n) * 4)})
        if (rows_meet(h, x)) throw Error("kv_store_rotary_paged: k, v, q, q_out, table or slots overlap a cache or a scale");
      for (const RowSet *x = held; x < &h; ++x)
        if (rows_meet(h, *x)) throw Error("kv_store_rotary_paged: caches and scales overlap each other");
    }
    hip_check(kv_store_paged(dt, k, v, long(ldk), long(ldv), slots, k_cache, v_cache, k_scale, v_scale, n, Hkv, hd, page, n_pages,
                             serving_error_flag(), S_(stream), &p),
              op);
  })
}

// ---- products in 8-bit integers ---------------------------------------------------
int mh_quantize_rows(int dt, const void *x, int64_t ldx, int8_t *q, int64_t ldq, float *scale, int rows, int cols, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (rows < 0 || cols < 1) throw Error("quantize_rows: bad row count or empty rows");
    if (rows == 0) return 0;
    const int64_t es = int64_t(dt_size(dt));
    check_whole_rows("quantize_rows", "x", es, x, rows, ldx, cols);
    check_whole_rows("quantize_rows", "q", 1, q, rows, ldq, cols);
    if (!scale) throw Error("quantize_rows: null scale");
    if (rows_meet({x, rows, ldx * es, cols * es}, {q, rows, ldq, cols})) throw Error("quantize_rows: q overlaps x");
    check_whole_rows("quantize_rows", "scale", 4, scale, 1, rows, rows);
    const RowSet o = whole(scale, int64_t(rows) * 4);
    if (rows_meet(o, {x, rows, ldx * es, cols * es}) || rows_meet(o, {q, rows, ldq, cols}))
      throw Error("quantize_rows: scale overlaps x or q");
    QuantRows p;
    p.x = x;
    p.q = q;
    p.scale = scale;
    p.ldx = ldx;
    p.ldq = ldq;
    p.rows = rows;
    p.cols = cols;
    hip_check(quantize_rows(dt, p, S_(stream)), "quantize_rows");
  })
}
int mh_dequantize_rows(int dt, const int8_t *q, int64_t ldq, const float *scale, void *out, int64_t ldo, int rows, int cols,
                       void *stream) {
  MH_TRY({
    check_dt(dt);
    if (rows < 0 || cols < 1) throw Error("dequantize_rows: bad row count or empty rows");
    if (rows == 0) return 0;
    const int64_t es = int64_t(dt_size(dt));
    check_whole_rows("dequantize_rows", "q", 1, q, rows, ldq, cols);
    check_whole_rows("dequantize_rows", "out", es, out, rows, ldo, cols);
    if (!scale) throw Error("dequantize_rows: null scale");
    if (rows_meet({out, rows, ldo * es, cols * es}, {q, rows, ldq, cols})) throw Error("dequantize_rows: out overlaps q");
    check_whole_rows("dequantize_rows", "scale", 4, scale, 1, rows, rows);
    if (rows_meet({out, rows, ldo * es, cols * es}, whole(scale, int64_t(rows) * 4)))
      throw Error("dequantize_rows: out overlaps scale");
    QuantRows p;
    p.out = out;
    p.q = const_cast<int8_t *>(q);
    p.scale = const_cast<float *>(scale);
    p.ldx = ldo;
    p.ldq = ldq;
    p.rows = rows;
    p.cols = cols;
    hip_check(dequantize_rows(dt, p, S_(stream)), "dequantize_rows");
  })
}
int mh_linear_i8(int dt, const int8_t *x, int64_t ldx, const float *x_scale, const int8_t *w, int64_t ldw, const float *w_scale,
                 const void *bias, const void *resid, int64_t ldr, void *out, int64_t ldo, int M, int N, int K, int act,
                 void *stream) {
  MH_TRY({
    check_dt(dt);
    if (act < 0 || act > 2) throw Error("linear_i8: bad activation code");
    if (M < 0 || N < 0 || K < 1) throw Error("linear_i8: negative size or empty rows");
    if (K > kI8MaxK) throw Error("linear_i8: the sums of more than 2^17 - 1 products may pass 32 bits");
    if (int64_t((int64_t(M) + 63) / 64) * ((int64_t(N) + 63) / 64) > kI8MaxTiles) throw Error("linear_i8: more outputs than one launch takes (2^34)");
    if (M == 0 || N == 0) return 0;
    const int64_t es = int64_t(dt_size(dt));
    check_whole_rows("linear_i8", "x", 1, x, M, ldx, K);
    check_whole_rows("linear_i8", "w", 1, w, N, ldw, K);
    check_whole_rows("linear_i8", "out", es, out, M, ldo, N);
    if (!x_scale || !w_scale) throw Error("linear_i8: null scale");
    check_whole_rows("linear_i8", "x_scale", 4, x_scale, 1, M, M);
    check_whole_rows("linear_i8", "w_scale", 4, w_scale, 1, N, N);
    if (bias) check_whole_rows("linear_i8", "bias", es, bias, 1, N, N);
    const RowSet o{out, M, ldo * es, N * es};
    if (resid) {
      check_whole_rows("linear_i8", "resid", es, resid, M, ldr, N);
      if (!(resid == out && (ldr == ldo || M == 1)) && rows_meet(o, {resid, M, ldr * es, N * es}))
        throw Error("linear_i8: out overlaps the residual without being it");
    }
    if (rows_meet(o, {x, M, ldx, K}) || rows_meet(o, {w, N, ldw, K})) throw Error("linear_i8: out overlaps x or w");
    if (rows_meet(o, whole(x_scale, int64_t(M) * 4)) || rows_meet(o, whole(w_scale, int64_t(N) * 4)) || rows_meet(o, whole(bias, N * es)))
      throw Error("linear_i8: out overlaps a scale or the bias");
    LinearI8 p;
    p.x = x;
    p.w = w;
    p.sx = x_scale;
    p.sw = w_scale;
    p.bias = bias;
    p.resid = resid;
    p.out = out;
    p.ldx = ldx;
    p.ldw = ldw;
    p.ldo = ldo;
    p.ldr = ldr;
    p.M = M;
    p.N = N;
    p.K = K;
    p.act = act;
    hip_check(linear_i8(dt, p, S_(stream)), "linear_i8");
  })
}

// ---- sampling ------------------------------------------------------------------
int mh_sample_workspace(int dt, int rows, int cols, size_t *bytes) {
  MH_TRY({
    check_dt(dt);
    if (!bytes) throw Error("sample_workspace: null output");
    check_sample_size(rows, cols);
    *bytes = 0;
  })
}
int mh_sample(int dt, const void *logits, int64_t ld, int rows, int cols, const float *u, const float *temperature,
              const int32_t *top_k, const float *top_p, const float *min_p, int32_t *out, float *logprob, void *workspace,
              size_t workspace_bytes, void *stream) {
  MH_TRY({
    check_dt(dt);
    check_sample_size(rows, cols);
    if (rows == 0) return 0;
    if (!logits || !u || !out) throw Error("sample: null argument");
    if (ld < cols) throw Error("sample: rows overlap");
    if (reinterpret_cast<uintptr_t>(logits) % dt_size(dt)) throw Error("sample: logits must be aligned to their type");
    Sampling p;
    p.logits = logits;
    p.ld = long(ld);
    p.rows = rows;
    p.cols = cols;
    p.u = u;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.ids = out;
    p.logprob = logprob;
    hip_check(sample_rows(dt, p, S_(stream)), "sample");
  })
}

// ---- shape -------------------------------------------------------------------
int mh_concat(int dt, const void *const *inputs, int count, void *out, int dim, int ndim, const int *shapes,
              void *stream) {
  MH_TRY({
    check_dt(dt, true);
    if (count <= 0) throw Error("concat: no inputs");
    if (dim < 0 || dim >= ndim) throw Error("concat: dim out of range");
    for (int j = 1; j < count; ++j)
      for (int d = 0; d < ndim; ++d)
        if (d != dim && shapes[j * ndim + d] != shapes[d]) throw Error("concat: shape mismatch");
    size_t outer = 1, inner = 1, total = 0;
    for (int d = 0; d < dim; ++d) outer *= size_t(shapes[d]);
    for (int d = dim + 1; d < ndim; ++d) inner *= size_t(shapes[d]);
    for (int j = 0; j < count; ++j) total += size_t(shapes[j * ndim + dim]);
    size_t off = 0;
    for (int j = 0; j < count; ++j) {
      const size_t len = size_t(shapes[j * ndim + dim]) * inner;
      hip_check(concat_part(dt, inputs[j], out, outer, len, total * inner, off, S_(stream)), "concat");
      off += len;
    }
  })
}
int mh_transpose2d(int dt, const void *in, void *out, int batch, int rows, int cols, void *stream) {
  MH_TRY({
    check_dt(dt, true);
    hip_check(transpose2d(dt, in, out, batch, rows, cols, S_(stream)), "transpose2d");
  })
}

// ---- spatial -----------------------------------------------------------------
static void conv_geom(ConvArgs &cv, int B, int iC, int iH, int iW, int kH, int kW, int s, int p) {
  if (s <= 0 || p < 0 || kH <= 0 || kW <= 0) throw Error("conv2d: bad stride/padding/kernel");
  cv.B = B; cv.iC = iC; cv.iH = iH; cv.iW = iW; cv.kH = kH; cv.kW = kW; cv.s = s; cv.p = p;
  cv.oH = (iH + 2 * p - kH) / s + 1;
  cv.oW = (iW + 2 * p - kW) / s + 1;
  cv.ldx = iC;
  if (cv.oH <= 0 || cv.oW <= 0) throw Error("conv2d: empty output");
}

int mh_pack_conv_weight(int dt, const void *w, void *w_ohwi, int oC, int iC, int kH, int kW, void *stream) {
  MH_TRY({
    check_dt(dt);
    hip_check(transpose2d(dt, w, w_ohwi, oC, iC, kH * kW, S_(stream)), "pack_conv_weight");
  })
}

int mh_conv2d_nhwc(int dt, const void *x, const void *w_ohwi, const void *bias, void *out, int B, int iC, int iH,
                   int iW, int oC, int kH, int kW, int s, int p, int act, void *stream) {
  MH_TRY({
    check_dt(dt);
    ConvArgs cv;
    conv_geom(cv, B, iC, iH, iW, kH, kW, s, p);
    EpiArgs ep;
    ep.out = out;
    ep.ldc = oC;
    ep.bias = bias;
    ep.bias_first = 1;
    ep.act = act;
    hip_check(conv_nhwc(dt, x, w_ohwi, cv, oC, ep, -1, S_(stream)), "conv2d_nhwc");
  })
}

int mh_conv2d(int dt, const void *in, const void *w, const void *bias, void *out, int B, int iC, int iH, int iW,
              int oC, int kH, int kW, int s, int p, void *stream) {
  MH_TRY({
    check_dt(dt);
    ConvArgs cv;
    conv_geom(cv, B, iC, iH, iW, kH, kW, s, p);
    const size_t es = dt_size(dt);
    const size_t xb = (size_t(B) * iC * iH * iW * es + 255) & ~size_t(255);
    const size_t wb = (size_t(oC) * iC * kH * kW * es + 255) & ~size_t(255);
    const size_t ob = size_t(B) * oC * cv.oH * cv.oW * es;
    char *ws = static_cast<char *>(workspace(xb + wb + ob + 256));
    hip_check(nchw_to_nhwc(dt, in, ws, B, iC, iH * iW, S_(stream)), "nchw_to_nhwc");
    hip_check(transpose2d(dt, w, ws + xb, oC, iC, kH * kW, S_(stream)), "pack weight");
    EpiArgs ep;
    ep.out = ws + xb + wb;
    ep.ldc = oC;
    ep.bias = bias;
    ep.bias_first = 1;
    hip_check(conv_nhwc(dt, ws, ws + xb, cv, oC, ep, -1, S_(stream)), "conv2d");
    hip_check(nhwc_to_nchw(dt, ws + xb + wb, out, B, oC, cv.oH * cv.oW, S_(stream)), "nhwc_to_nchw");
  })
}

int mh_pack_convt_weight(int dt, const void *w, void *w_packed, int iC, int oC, int k, void *stream) {
  MH_TRY({
    check_dt(dt);
    // out [kh][kw][oc][ic] gathered from in [ic][oc][kh][kw]
    StridedArgs g;
    g.ndim = 4;
    g.shape[0] = k; g.shape[1] = k; g.shape[2] = oC; g.shape[3] = iC;
    g.strides[0] = k; g.strides[1] = 1; g.strides[2] = long(k) * k; g.strides[3] = long(oC) * k * k;
    g.total = size_t(k) * k * oC * iC;
    hip_check(to_contiguous(dt, w, w_packed, g, S_(stream)), "pack_convt_weight");
  })
}

int mh_conv_transpose2d_nhwc(int dt, const void *x, const void *w_packed, const void *bias, void *out, int B, int iC,
                             int iH, int iW, int oC, int k, int64_t ldc, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (oC % 4 != 0) throw Error("conv_transpose2d: out channels must be a multiple of 4");
    if (ldc < oC) throw Error("conv_transpose2d: ldc < out channels");
    EpiArgs ep;
    ep.mode = EPI_CONVT;
    ep.out = out;
    ep.ldc = long(ldc);
    ep.bias = bias;
    ep.bias_first = 1;
    ep.convt_oc = oC;
    ep.convt_k = k;
    ep.convt_ih = iH;
    ep.convt_iw = iW;
    hip_check(gemm_nt(dt, x, w_packed, B * iH * iW, k * k * oC, iC, iC, iC, 1, 0, 0, 0, ep, -1, S_(stream)),
              "conv_transpose2d");
  })
}

int mh_max_pool2d(int dt, const void *in, void *out, int B, int C, int iH, int iW, int k, int s, int p, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (k <= 0 || s <= 0 || p < 0) throw Error("max_pool2d: bad window");
    hip_check(max_pool2d(dt, 0, in, out, B, C, iH, iW, k, s, p, S_(stream)), "max_pool2d");
  })
}
int mh_max_pool2d_nhwc(int dt, const void *in, void *out, int B, int C, int iH, int iW, int k, int s, int p,
                       void *stream) {
  MH_TRY({
    check_dt(dt);
    if (k <= 0 || s <= 0 || p < 0) throw Error("max_pool2d: bad window");
    hip_check(max_pool2d(dt, 1, in, out, B, C, iH, iW, k, s, p, S_(stream)), "max_pool2d_nhwc");
  })
}
int mh_upsample2d(int dt, const void *in, void *out, int B, int C, int iH, int iW, int scale, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (scale <= 0) throw Error("upsample2d: bad scale");
    hip_check(upsample2d(dt, 0, in, out, B, C, iH, iW, scale, S_(stream)), "upsample2d");
  })
}
int mh_upsample2d_nhwc(int dt, const void *in, void *out, int B, int C, int iH, int iW, int scale, void *stream) {
  MH_TRY({
    check_dt(dt);
    if (scale <= 0) throw Error("upsample2d: bad scale");
    hip_check(upsample2d(dt, 1, in, out, B, C, iH, iW, scale, S_(stream)), "upsample2d_nhwc");
  })
}
int mh_nchw_to_nhwc(int dt, const void *in, void *out, int B, int C, int HW, void *stream) {
  MH_TRY({
    check_dt(dt, true);
    hip_check(nchw_to_nhwc(dt, in, out, B, C, HW, S_(stream)), "nchw_to_nhwc");
  })
}
int mh_nhwc_to_nchw(int dt, const void *in, void *out, int B, int C, int HW, void *stream) {
  MH_TRY({
    check_dt(dt, true);
    hip_check(nhwc_to_nchw(dt, in, out, B, C, HW, S_(stream)), "nhwc_to_nchw");
  })
}

}  // extern "C"
