"""Python mirror of MuNet's ``Backend`` capability interface for the HIP backend.

Method names, argument order and meaning follow the reference's capability
classes (src/core/backend.hpp:190-345); a ``Storage`` here is any torch
tensor living on the GPU (torch only provides device memory and the stream),
and every compute call goes through libmunet_hip.so.  Errors raise
``HipError`` as MuNet's backends raise std::runtime_error.

``query_support`` mirrors Backend::query_support (src/core/backend.hpp:
411-425): fp32/fp16/bf16 are available for every implemented feature and
the fallback policy is always ExplicitUnsupported - this backend never
falls back to the CPU.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import call, i64s, ints
from .synth import BF16, F16, F32, I32

_vp = ctypes.c_void_p


def _torch():
    import torch
    return torch


def torch_dtype(dt):
    t = _torch()
    return {F32: t.float32, F16: t.float16, BF16: t.bfloat16, I32: t.int32}[dt]


def dtype_code(tdtype):
    t = _torch()
    return {t.float32: F32, t.float16: F16, t.bfloat16: BF16, t.int32: I32}[tdtype]


def to_device(arr: np.ndarray, dt: int, device="cuda"):
    """Host storage array (float32 / uint16 bits / int32) -> GPU tensor with the same bits."""
    t = _torch()
    a = np.ascontiguousarray(arr)
    if dt in (F16, BF16):
        host = t.from_numpy(a.astype(np.uint16, copy=False).view(np.int16)).view(torch_dtype(dt))
    elif dt == F32:
        host = t.from_numpy(a.astype(np.float32, copy=False))
    else:
        host = t.from_numpy(a.astype(np.int32, copy=False))
    return host.to(device)


def to_host(x, dt: int) -> np.ndarray:
    """GPU tensor -> host storage array (uint16 bit patterns for 16-bit types)."""
    t = _torch()
    c = x.detach().contiguous().cpu()
    if dt in (F16, BF16):
        return c.view(t.int16).numpy().view(np.uint16).copy()
    return c.numpy().copy()


def empty(shape, dt, device="cuda"):
    return _torch().empty(tuple(shape), dtype=torch_dtype(dt), device=device)


def _p(x):
    return None if x is None else _vp(x.data_ptr())


def _stream():
    return _vp(_torch().cuda.current_stream().cuda_stream)


def _dt(x):
    return dtype_code(x.dtype)


def _operand(op, d, name, x, dtype, shape):
    """Address of a contiguous operand of the given type and shape on GPU d."""
    if x.get_device() != d or x.dtype is not dtype or x.shape != shape or not x.is_contiguous():
        _refuse(op, d, name, x, (dtype,), shape, True)
    return x.data_ptr()


def _optional(op, d, name, x, dtype, shape):
    return None if x is None else _operand(op, d, name, x, dtype, shape)


def _token_rows(op, d, name, x, dtype, shape):
    """(address, values between rows) of [rows, heads, hd] on GPU d whose heads are contiguous."""
    if x.get_device() != d or x.dtype is not dtype or x.shape != shape:
        _refuse(op, d, name, x, (dtype,), shape, False)
    n, h, e = x.stride()
    if (e != 1 and shape[2] > 1) or (h != shape[2] and shape[1] > 1):
        raise ValueError(f"{op}: the heads of {name} must be contiguous")
    return x.data_ptr(), n if shape[0] > 1 else shape[1] * shape[2]


def _rows(op, d, name, x, dtype, shape):
    """(address, values between rows) of a matrix on GPU d whose rows are contiguous."""
    if x.get_device() != d or x.dtype is not dtype or x.shape != shape:
        _refuse(op, d, name, x, (dtype,), shape, False)
    n, e = x.stride()
    if e != 1 and shape[1] > 1:
        raise ValueError(f"{op}: the rows of {name} must be contiguous")
    return x.data_ptr(), n if shape[0] > 1 else shape[1]


def _pool(op, d, k_cache, v_cache, k_scale, v_scale):
    """Addresses and (pages, Hkv, page, hd) of the paged cache's four tensors."""
    if k_cache.dim() != 4:
        _refuse(op, d, "k_cache", k_cache, (k_cache.dtype,), (None,) * 4, True)
    n_pages, Hkv, page, hd = size = k_cache.shape
    t = _torch()
    dt = k_cache.dtype
    if dt is not t.uint8 and dt is not t.float8_e4m3fn:
        _refuse(op, d, "k_cache", k_cache, (t.uint8, t.float8_e4m3fn), size, True)
    return (_operand(op, d, "k_cache", k_cache, dt, size), _operand(op, d, "v_cache", v_cache, dt, (n_pages, Hkv, hd, page)),
            _operand(op, d, "k_scale", k_scale, t.float32, (n_pages, Hkv)),
            _operand(op, d, "v_scale", v_scale, t.float32, (n_pages, Hkv)), n_pages, Hkv, page, hd)


def _refuse(op, d, name, x, dtypes, shape, contiguous):
    """Say what is wrong with an operand."""
    if d < 0 or x.get_device() != d:
        raise ValueError(f"{op}: all tensors must be on one GPU; {name} is on {x.device}")
    if x.dtype not in dtypes:
        raise ValueError(f"{op}: {name} must be {' or '.join(str(t)[6:] for t in dtypes)}, not {str(x.dtype)[6:]}")
    if x.dim() != len(shape) or any(w is not None and w != n for w, n in zip(shape, x.shape)):
        raise ValueError(f"{op}: {name} must be of shape [" + ", ".join("*" if w is None else str(w) for w in shape)
                         + f"], not {list(x.shape)}")
    raise ValueError(f"{op}: {name} must be contiguous")


def _rank(op, d, name, x, rank):
    if d < 0 or x.dim() != rank:
        _refuse(op, d, name, x, (x.dtype,), (None,) * rank, False)
    return x.shape


def _float_dt(op, name, x):
    t = _torch()
    dt = x.dtype
    if dt is t.bfloat16:
        return BF16
    if dt is t.float16:
        return F16
    if dt is not t.float32:
        _refuse(op, x.get_device(), name, x, (t.float32, t.float16, t.bfloat16), x.shape, False)
    return F32


def _workspace(op, d, ws, need):
    """(workspace, its address, its bytes): the caller's, or one of ``need()`` bytes."""
    t = _torch()
    if ws is None:
        n = need()
        ws = t.empty(n, dtype=t.uint8, device=d) if n else None
        return ws, None if ws is None else ws.data_ptr(), n
    n = ws.numel()
    return ws, _operand(op, d, "workspace", ws, t.uint8, (n,)), n


def _launch(name, d, *args):
    """The call with GPU d as the current device, on torch's current stream of it (its
    handle alone: a Stream object around it costs 2.7 us a call)."""
    t = _torch()
    if t.cuda.current_device() == d:
        call(name, *args, t._C._cuda_getCurrentRawStream(d))
    else:
        with t.cuda.device(d):
            call(name, *args, t._C._cuda_getCurrentRawStream(d))


def compute_broadcast(a_shape, a_strides, b_shape, b_strides):
    """compute_broadcast (reference src/types.hpp:436-478)."""
    nd = max(len(a_shape), len(b_shape))
    out, sa, sb = [1] * nd, [0] * nd, [0] * nd
    for i in range(nd):
        ia, ib, o = len(a_shape) - 1 - i, len(b_shape) - 1 - i, nd - 1 - i
        da = a_shape[ia] if ia >= 0 else 1
        db = b_shape[ib] if ib >= 0 else 1
        if da != db and da != 1 and db != 1:
            raise ValueError(f"shape mismatch {tuple(a_shape)} vs {tuple(b_shape)}")
        out[o] = max(da, db)
        sa[o] = (0 if (da == 1 and db != 1) else a_strides[ia]) if ia >= 0 else 0
        sb[o] = (0 if (db == 1 and da != 1) else b_strides[ib]) if ib >= 0 else 0
    return out, sa, sb


def contiguous_strides(shape):
    s, out = 1, []
    for d in reversed(shape):
        out.append(s)
        s *= d
    return list(reversed(out))


@dataclass
class BroadcastInfo:
    out_shape: list
    strides_a: list
    strides_b: list


@dataclass
class BackendSupport:
    available: bool
    fallback_policy: str
    preferred_accumulation_dtype: int


# BackendFeature (reference src/core/backend.hpp:16-30, in its order) and the
# path's functions that have no reference capability: the mh_query_support codes
FEATURES = {"elementwise_binary": 0, "broadcast_row": 1, "matmul": 2, "unary_activation": 3, "softmax": 4,
            "concat": 5, "loss": 6, "convolution": 7, "pooling": 8, "batch_norm": 9, "optimizer_step": 10,
            "random_fill": 11, "reduction": 12, "to_contiguous": 100, "layer_norm": 101, "attention": 102,
            "embedding": 103, "masked_fill": 104}
POLICIES = ("ExplicitUnsupported", "CPUFallback", "ConversionFallback")


def query_support(feature: str, dtype: int) -> BackendSupport:
    """Backend::query_support (src/core/backend.hpp:411-425) of the HIP
    backend, from mh_query_support (no device needed). Unknown features are
    unavailable."""
    av, pol, acc = ctypes.c_int(), ctypes.c_int(), ctypes.c_int()
    call("mh_query_support", FEATURES.get(feature, -1), dtype, ctypes.byref(av), ctypes.byref(pol),
         ctypes.byref(acc))
    return BackendSupport(bool(av.value), POLICIES[pol.value], acc.value)


ROTARY_SCALINGS = {None: 0, "linear": 1, "base": 2, "turns": 3}


def rotary_frequencies(rot, base=10000.0, scaling=None, factor=1.0, original=0, low=1.0, high=32.0):
    """(frequencies, magnitude) for ``rotary_table`` (mh_rotary_frequencies): float64
    [rot / 2] on the host; ``scaling`` None, "linear", "base" or "turns" (whose magnitude
    is for models that were trained with it)."""
    if scaling not in ROTARY_SCALINGS:
        raise ValueError(f"rotary_frequencies: scaling must be None, 'linear', 'base' or 'turns', not {scaling!r}")
    freq, m = (ctypes.c_double * max(1, rot // 2))(), ctypes.c_double()
    call("mh_rotary_frequencies", freq, ctypes.byref(m), rot, base, ROTARY_SCALINGS[scaling], factor, original, low, high)
    return np.array(freq, dtype=np.float64), m.value


class HipBackend:
    """The HIP backend's capability surface (reference class Backend)."""

    def __init__(self, device: int = 0):
        self.device = device
        call("mh_init", device)

    def name(self):
        return "hip"

    def query_support(self, feature: str, dtype: int, shape=None) -> BackendSupport:
        return query_support(feature, dtype)

    # ---- allocation / transfer (backend.hpp:190-205) ----------------------
    def allocate(self, nbytes: int) -> int:
        p = _vp()
        call("mh_allocate", ctypes.byref(p), nbytes)
        return p.value or 0

    def deallocate(self, ptr: int):
        call("mh_deallocate", _vp(ptr))

    def memset(self, x, value: int, nbytes: int):
        call("mh_memset", _p(x), value, nbytes, _stream())

    def synchronize(self):
        call("mh_synchronize", _stream())

    def get_last_kernel_time_us(self) -> float:
        return _lib.load().mh_get_last_kernel_time_us()

    def reports_gpu_kernel_time(self) -> bool:
        return True

    def to_contiguous(self, src, dst, shape, strides, offset=0):
        call("mh_to_contiguous", _dt(src), _p(src), _p(dst), len(shape), ints(shape), i64s(strides), offset,
             _stream())

    # ---- elementwise (backend.hpp:207-238) --------------------------------
    def _bin(self, name, a, b, out, info: BroadcastInfo):
        call(name, _dt(a), _p(a), _p(b), _p(out), len(info.out_shape), ints(info.out_shape), i64s(info.strides_a),
             i64s(info.strides_b), _stream())

    def add(self, a, b, out, info):
        self._bin("mh_add", a, b, out, info)

    def sub(self, a, b, out, info):
        self._bin("mh_sub", a, b, out, info)

    def mul(self, a, b, out, info):
        self._bin("mh_mul", a, b, out, info)

    def div(self, a, b, out, info):
        self._bin("mh_div", a, b, out, info)

    def _un(self, name, x, out, n):
        call(name, _dt(x), _p(x), _p(out), n, _stream())

    def relu(self, x, out, n):
        self._un("mh_relu", x, out, n)

    def sigmoid(self, x, out, n):
        self._un("mh_sigmoid", x, out, n)

    def exp(self, x, out, n):
        self._un("mh_exp", x, out, n)

    def log(self, x, out, n):
        self._un("mh_log", x, out, n)

    def sqrt(self, x, out, n):
        self._un("mh_sqrt", x, out, n)

    def rsqrt(self, x, out, n):
        self._un("mh_rsqrt", x, out, n)

    def sin(self, x, out, n):
        self._un("mh_sin", x, out, n)

    def cos(self, x, out, n):
        self._un("mh_cos", x, out, n)

    def softmax(self, x, out, batch_size, num_classes):
        call("mh_softmax", _dt(x), _p(x), _p(out), batch_size, num_classes, _stream())

    # ---- op-layer functions without a reference backend hook ---------------
    def gelu(self, x, out, n):
        self._un("mh_gelu", x, out, n)

    def masked_fill(self, x, mask, out, n, value):
        call("mh_masked_fill", _dt(x), _p(x), _p(mask), _p(out), n, float(value), _stream())

    def layer_norm(self, x, w, b, out, rows, cols, eps=1e-5):
        call("mh_layer_norm", _dt(x), _p(x), _p(w), _p(b), _p(out), rows, cols, eps, _stream())

    def embedding(self, ids, w, out, n, V, D):
        call("mh_embedding", _dt(w), _p(ids), _p(w), _p(out), n, V, D, _stream())

    def embedding_pos(self, ids, tok_w, pos_w, out, n, V, D, T):
        call("mh_embedding_pos", _dt(tok_w), _p(ids), _p(tok_w), _p(pos_w), _p(out), n, V, D, T, _stream())

    def check_device_errors(self):
        call("mh_check_device_errors")

    def convert(self, x, out, n):
        call("mh_convert", _dt(x), _p(x), _dt(out), _p(out), n, _stream())

    def check_f16_rounding(self) -> int:
        """Float bit patterns (of all 2^32) where the kernels' fast fp16
        rounding differs from the full codec (no reference counterpart)."""
        n = ctypes.c_ulonglong(0)
        call("mh_check_f16_rounding", ctypes.byref(n), _stream())
        return n.value

    def argmax(self, x, out, rows, cols):
        call("mh_argmax", _dt(x), _p(x), _p(out), rows, cols, _stream())

    def measure_mfma_peak(self, dt=2, iters=16000) -> float:
        """Measured matrix-core peak in FLOP/s (mh_measure_mfma_peak; dt 2 =
        bf16, 1 = fp16) on the current torch stream."""
        v = ctypes.c_double(0.0)
        call("mh_measure_mfma_peak", dt, iters, ctypes.byref(v), _stream())
        return v.value

    def measure_hbm_read(self, buf, reps=5) -> float:
        """Measured HBM read rate in bytes/s over the device tensor ``buf``
        (mh_measure_hbm_read)."""
        v = ctypes.c_double()
        call("mh_measure_hbm_read", _p(buf), buf.numel() * buf.element_size(), reps, ctypes.byref(v), _stream())
        return v.value

    # ---- blas (backend.hpp:250-260) ----------------------------------------
    def matmul(self, a, b, out, M, K, N, transA=False, transB=False):
        call("mh_matmul", _dt(a), _p(a), _p(b), _p(out), M, K, N, int(transA), int(transB), _stream())

    def matmul_noalloc(self, a, b, out, M, K, N, transA=False, transB=False):
        """mh_matmul_noalloc: mh_matmul staging its transposes in the
        library's fixed per-device scratch (no device allocation)."""
        call("mh_matmul_noalloc", _dt(a), _p(a), _p(b), _p(out), M, K, N, int(transA), int(transB), _stream())

    def batched_matmul(self, a, b, out, batch, M, K, N, transA, transB, stride_a, stride_b, stride_out):
        call("mh_batched_matmul", _dt(a), _p(a), _p(b), _p(out), batch, M, K, N, int(transA), int(transB),
             stride_a, stride_b, stride_out, _stream())

    def pack_linear_weight(self, w, w_t, in_f, out_f):
        call("mh_pack_linear_weight", _dt(w), _p(w), _p(w_t), in_f, out_f, _stream())

    def linear(self, x, w_t, bias, out, M, K, N, act=0, resid=None):
        call("mh_linear", _dt(x), _p(x), _p(w_t), _p(bias), _p(out), M, K, N, act, _p(resid), _stream())

    def qkv_projection(self, x, wqkv_t, bqkv, q, k, v, B, T, E, H):
        call("mh_qkv_projection", _dt(x), _p(x), _p(wqkv_t), _p(bqkv), _p(q), _p(k), _p(v), B, T, E, H,
             _stream())

    def attention(self, q, k, v, ctx, B, H, T, hd, causal):
        call("mh_attention", _dt(q), _p(q), _p(k), _p(v), _p(ctx), B, H, T, hd, int(causal), _stream())

    def attention_textbook(self, q, k, v, ctx, B, H, T, hd, causal):
        """Textbook keys (key j of a head is row j of its k): the decode
        attention; no MuNet counterpart."""
        call("mh_attention_textbook", _dt(q), _p(q), _p(k), _p(v), _p(ctx), B, H, T, hd, int(causal), _stream())

    # ---- paged 8-bit KV cache (no MuNet counterpart) --------------------------
    # These calls take their sizes from their tensors and check them; all of a
    # call's tensors lie on one GPU, and it runs on torch's current stream there.
    def page_plan(self, lens, new_lens, free_pages, tables, total_lens, cu, slots, positions, used, page, n_pages):
        """Pages and slots of a step's new tokens (mh_page_plan): ``new_lens``
        [B] more tokens behind ``lens`` [B]; ``tables`` [B, width] gets the pages
        taken from ``free_pages``; ``total_lens`` [B], ``cu`` [B + 1], ``slots``,
        ``positions`` (or None) and ``used`` [1] are written.  All int32."""
        op, d, i32 = "page_plan", lens.get_device(), _torch().int32
        (B,), (_, width) = _rank(op, d, "lens", lens, 1), _rank(op, d, "tables", tables, 2)
        (n_free,), (n,) = _rank(op, d, "free_pages", free_pages, 1), _rank(op, d, "slots", slots, 1)
        _launch("mh_page_plan", d, _operand(op, d, "lens", lens, i32, (B,)), _operand(op, d, "new_lens", new_lens, i32, (B,)),
                _operand(op, d, "free_pages", free_pages, i32, (n_free,)), _operand(op, d, "tables", tables, i32, (B, width)),
                _operand(op, d, "total_lens", total_lens, i32, (B,)), _operand(op, d, "cu", cu, i32, (B + 1,)),
                _operand(op, d, "slots", slots, i32, (n,)), _optional(op, d, "positions", positions, i32, (n,)),
                _operand(op, d, "used", used, i32, (1,)), B, n_free, width, page, n_pages, n)

    def kv_store_paged(self, k, v, slots, k_cache, v_cache, k_scale, v_scale):
        """Keys and values [n, Hkv, hd] (heads contiguous, rows any multiple of 16
        bytes apart) into their slots (mh_kv_store_paged): ``k_cache`` [pages,
        Hkv, page, hd] and ``v_cache`` [pages, Hkv, hd, page] of 8-bit
        elements, scales [pages, Hkv] float32."""
        op, d = "kv_store_paged", k.get_device()
        kc, vc, ks, vs, n_pages, Hkv, page, hd = _pool(op, d, k_cache, v_cache, k_scale, v_scale)
        shape = (_rank(op, d, "k", k, 3)[0], Hkv, hd)
        dt = _float_dt(op, "k", k)
        (kp, ldk), (vp, ldv) = _token_rows(op, d, "k", k, k.dtype, shape), _token_rows(op, d, "v", v, k.dtype, shape)
        _launch("mh_kv_store_paged", d, dt, kp, vp, ldk, ldv, _operand(op, d, "slots", slots, _torch().int32, shape[:1]), kc, vc, ks,
                vs, shape[0], Hkv, hd, page, n_pages)

    def attention_paged_workspace(self, q, k_cache, lens, max_q, max_len, window=0) -> int:
        """Bytes of workspace that ``attention_paged`` needs for these sizes."""
        n = ctypes.c_size_t()
        rows, Hq, hd = q.shape
        call("mh_attention_paged_workspace", _float_dt("attention_paged", "q", q), lens.shape[0], rows, Hq, k_cache.shape[1], hd,
             max_q, max_len, window, ctypes.byref(n))
        return n.value

    def attention_paged(self, q, k_cache, v_cache, k_scale, v_scale, tables, lens, cu, out, max_q, max_len, causal=True,
                        window=0, scale=None, workspace=None):
        """Attention of ragged queries over the paged cache (mh_attention_paged):
        request b's queries are rows cu[b]..cu[b+1]-1 of ``q`` and ``out`` [rows,
        Hq, hd], the last of its lens[b] tokens; ``tables`` [B, width].
        ``scale`` None: 1 / sqrt(hd).  ``workspace``: a uint8 tensor of
        ``attention_paged_workspace`` bytes, else one is allocated."""
        op, d, i32 = "attention_paged", q.get_device(), _torch().int32
        kc, vc, ks, vs, n_pages, Hkv, page, hd = _pool(op, d, k_cache, v_cache, k_scale, v_scale)
        shape = (rows, Hq, _) = _rank(op, d, "q", q, 3)
        (B,), (_, width) = _rank(op, d, "lens", lens, 1), _rank(op, d, "tables", tables, 2)
        dt = _float_dt(op, "q", q)
        (qp, ldq), (po, ldo) = _token_rows(op, d, "q", q, q.dtype, (rows, Hq, hd)), _token_rows(op, d, "out", out, q.dtype, shape)
        if scale is None:
            scale = 0.0
        elif not scale:
            raise ValueError("attention_paged: scale 0 (None is 1 / sqrt(hd))")
        workspace, wp, wn = _workspace(op, d, workspace,
                                       lambda: self.attention_paged_workspace(q, k_cache, lens, max_q, max_len, window))
        _launch("mh_attention_paged", d, dt, qp, ldq, kc, vc, ks, vs, _operand(op, d, "tables", tables, i32, (B, width)),
                _operand(op, d, "lens", lens, i32, (B,)), _operand(op, d, "cu", cu, i32, (B + 1,)), po, ldo, B, rows, Hq, Hkv, hd, page,
                n_pages, width, max_q, max_len, causal, window, scale, wp, wn)

    # ---- rotary positions (no MuNet counterpart) --------------------------------
    def rotary_table(self, positions, freq, table, magnitude=1.0):
        """Angles of a step's tokens (mh_rotary_table): ``positions`` [n] int32,
        ``freq`` [pairs] float64 (``rotary_frequencies``) -> ``table`` [n, pairs, 2]
        float32, the cosines and sines times ``magnitude``."""
        op, d, t = "rotary_table", positions.get_device(), _torch()
        (n,), (half,) = _rank(op, d, "positions", positions, 1), _rank(op, d, "freq", freq, 1)
        _launch("mh_rotary_table", d, _operand(op, d, "positions", positions, t.int32, (n,)),
                _operand(op, d, "freq", freq, t.float64, (half,)), _operand(op, d, "table", table, t.float32, (n, half, 2)), n, half,
                magnitude)

    def rotary(self, x, table, out, interleaved=False, inverse=False):
        """The first pairs of each head of ``x`` [n, heads, hd] (heads contiguous)
        turned by ``table`` [n, pairs, 2] into ``out``, which may be ``x``
        (mh_rotary).  Pairs lie half of the rotated part apart, or ``interleaved``
        next to each other; ``inverse`` turns back, which is also the gradient."""
        op, d = "rotary", x.get_device()
        shape = (n, heads, hd) = _rank(op, d, "x", x, 3)
        half = _rank(op, d, "table", table, 3)[1]
        dt = _float_dt(op, "x", x)
        (xp, ldx), (po, ldo) = _token_rows(op, d, "x", x, x.dtype, shape), _token_rows(op, d, "out", out, x.dtype, shape)
        _launch("mh_rotary", d, dt, xp, ldx, _operand(op, d, "table", table, _torch().float32, (n, half, 2)), po, ldo, n, heads, hd,
                half, interleaved, inverse)

    def kv_store_rotary_paged(self, k, v, table, slots, k_cache, v_cache, k_scale, v_scale, q=None, q_out=None, interleaved=False):
        """``kv_store_paged`` of keys rotated by ``table`` [n, pairs, 2] on the way, and
        ``q`` [n, Hq, hd] rotated into ``q_out`` (which may be ``q``) beside them
        (mh_kv_store_rotary_paged).  Rows without a slot are left alone."""
        op, d, t = "kv_store_rotary_paged", k.get_device(), _torch()
        kc, vc, ks, vs, n_pages, Hkv, page, hd = _pool(op, d, k_cache, v_cache, k_scale, v_scale)
        n, half = _rank(op, d, "k", k, 3)[0], _rank(op, d, "table", table, 3)[1]
        shape, dt = (n, Hkv, hd), _float_dt(op, "k", k)
        (kp, ldk), (vp, ldv) = _token_rows(op, d, "k", k, k.dtype, shape), _token_rows(op, d, "v", v, k.dtype, shape)
        qp, ldq, po, ldo, Hq = None, 0, None, 0, 0
        if q is not None:
            Hq = _rank(op, d, "q", q, 3)[1]
            if q_out is None:
                raise ValueError("kv_store_rotary_paged: q needs q_out")
            (qp, ldq), (po, ldo) = (_token_rows(op, d, "q", q, k.dtype, (n, Hq, hd)),
                                    _token_rows(op, d, "q_out", q_out, k.dtype, (n, Hq, hd)))
        _launch("mh_kv_store_rotary_paged", d, dt, kp, vp, ldk, ldv, _operand(op, d, "table", table, t.float32, (n, half, 2)),
                _operand(op, d, "slots", slots, t.int32, (n,)), kc, vc, ks, vs, n, Hkv, hd, half, interleaved, page, n_pages, qp, ldq,
                po, ldo, Hq)

    # ---- products in 8-bit integers (no MuNet counterpart) ------------------------
    def quantize_rows(self, x, q, scale):
        """Rows of ``x`` [rows, cols] as int8 ``q`` with float32 ``scale`` [rows]
        (mh_quantize_rows): a linear_i8's tokens, or its weights [out, in]."""
        op, d, t = "quantize_rows", x.get_device(), _torch()
        shape = _rank(op, d, "x", x, 2)
        dt = _float_dt(op, "x", x)
        (xp, ldx), (qp, ldq) = _rows(op, d, "x", x, x.dtype, shape), _rows(op, d, "q", q, t.int8, shape)
        _launch("mh_quantize_rows", d, dt, xp, ldx, qp, ldq, _operand(op, d, "scale", scale, t.float32, shape[:1]), *shape)

    def dequantize_rows(self, q, scale, out):
        """The values that ``quantize_rows`` left, in ``out``'s type (mh_dequantize_rows)."""
        op, d, t = "dequantize_rows", q.get_device(), _torch()
        shape = _rank(op, d, "q", q, 2)
        dt = _float_dt(op, "out", out)
        (qp, ldq), (po, ldo) = _rows(op, d, "q", q, t.int8, shape), _rows(op, d, "out", out, out.dtype, shape)
        _launch("mh_dequantize_rows", d, dt, qp, ldq, _operand(op, d, "scale", scale, t.float32, shape[:1]), po, ldo, *shape)

    def linear_i8(self, x, x_scale, w, w_scale, out, bias=None, act=0, resid=None):
        """``linear`` of int8 tokens ``x`` [M, K] and weights ``w`` [N, K] with a float32
        scale each (mh_linear_i8): ``out`` [M, N], ``bias`` [N] and ``resid`` [M, N] of
        one floating type; ``resid`` may be ``out``."""
        op, d, t = "linear_i8", x.get_device(), _torch()
        M, K = _rank(op, d, "x", x, 2)
        N = _rank(op, d, "w", w, 2)[0]
        dt, i8, f32 = _float_dt(op, "out", out), t.int8, t.float32
        (xp, ldx), (wp, ldw) = _rows(op, d, "x", x, i8, (M, K)), _rows(op, d, "w", w, i8, (N, K))
        po, ldo = _rows(op, d, "out", out, out.dtype, (M, N))
        rp, ldr = (None, 0) if resid is None else _rows(op, d, "resid", resid, out.dtype, (M, N))
        _launch("mh_linear_i8", d, dt, xp, ldx, _operand(op, d, "x_scale", x_scale, f32, (M,)), wp, ldw,
                _operand(op, d, "w_scale", w_scale, f32, (N,)), _optional(op, d, "bias", bias, out.dtype, (N,)), rp, ldr, po, ldo, M, N,
                K, act)

    # ---- sampling (no MuNet counterpart) ---------------------------------------
    def sample_workspace(self, logits) -> int:
        """Bytes of workspace that ``sample`` needs for these logits."""
        n = ctypes.c_size_t()
        rows, cols = logits.shape
        call("mh_sample_workspace", _float_dt("sample", "logits", logits), rows, cols, ctypes.byref(n))
        return n.value

    def sample(self, logits, u, out, temperature=None, top_k=None, top_p=None, min_p=None, logprob=None, workspace=None):
        """One token per row of ``logits`` [rows, cols], drawn with the uniform
        numbers ``u`` [rows] (mh_sample): ``out`` [rows] int32; ``temperature``,
        ``top_p``, ``min_p`` float32 and ``top_k`` int32 [rows], or None;
        ``logprob`` [rows] float32 optional.  ``workspace``: a uint8 tensor of
        ``sample_workspace`` bytes, else one is allocated."""
        op, d, t = "sample", logits.get_device(), _torch()
        rows, cols = _rank(op, d, "logits", logits, 2)
        dt, f32, each = _float_dt(op, "logits", logits), t.float32, (rows,)
        ld, e = logits.stride()
        if e != 1 and cols > 1:
            raise ValueError("sample: logits must be contiguous along a row")
        workspace, wp, wn = _workspace(op, d, workspace, lambda: self.sample_workspace(logits))
        _launch("mh_sample", d, dt, logits.data_ptr(), ld if rows > 1 else cols, rows, cols, _operand(op, d, "u", u, f32, each),
                _optional(op, d, "temperature", temperature, f32, each), _optional(op, d, "top_k", top_k, t.int32, each),
                _optional(op, d, "top_p", top_p, f32, each), _optional(op, d, "min_p", min_p, f32, each),
                _operand(op, d, "out", out, t.int32, each), _optional(op, d, "logprob", logprob, f32, each), wp, wn)

    # ---- shape (backend.hpp:263-271) ---------------------------------------
    def concat(self, inputs, out, dim, shapes):
        ptrs = (_vp * len(inputs))(*[x.data_ptr() for x in inputs])
        flat = [d for s in shapes for d in s]
        call("mh_concat", _dt(out), ptrs, len(inputs), _p(out), dim, len(shapes[0]), ints(flat), _stream())

    def transpose2d(self, x, out, batch, rows, cols):
        call("mh_transpose2d", _dt(x), _p(x), _p(out), batch, rows, cols, _stream())

    # ---- spatial (backend.hpp:291-311) -------------------------------------
    def conv2d(self, x, w, bias, out, B, iC, iH, iW, oC, kH, kW, s, p):
        call("mh_conv2d", _dt(x), _p(x), _p(w), _p(bias), _p(out), B, iC, iH, iW, oC, kH, kW, s, p, _stream())

    def conv2d_nhwc(self, x, w_ohwi, bias, out, B, iC, iH, iW, oC, kH, kW, s, p, act=0):
        call("mh_conv2d_nhwc", _dt(x), _p(x), _p(w_ohwi), _p(bias), _p(out), B, iC, iH, iW, oC, kH, kW, s, p, act,
             _stream())

    def pack_conv_weight(self, w, w_ohwi, oC, iC, kH, kW):
        call("mh_pack_conv_weight", _dt(w), _p(w), _p(w_ohwi), oC, iC, kH, kW, _stream())

    def conv_transpose2d_nhwc(self, x, w_packed, bias, out, B, iC, iH, iW, oC, k, ldc=None):
        call("mh_conv_transpose2d_nhwc", _dt(x), _p(x), _p(w_packed), _p(bias), _p(out), B, iC, iH, iW, oC, k,
             oC if ldc is None else ldc, _stream())

    def pack_convt_weight(self, w, w_packed, iC, oC, k):
        call("mh_pack_convt_weight", _dt(w), _p(w), _p(w_packed), iC, oC, k, _stream())

    def max_pool2d(self, x, out, B, C, iH, iW, k, s, p):
        call("mh_max_pool2d", _dt(x), _p(x), _p(out), B, C, iH, iW, k, s, p, _stream())

    def max_pool2d_nhwc(self, x, out, B, C, iH, iW, k, s, p):
        call("mh_max_pool2d_nhwc", _dt(x), _p(x), _p(out), B, C, iH, iW, k, s, p, _stream())

    def upsample2d(self, x, out, B, C, iH, iW, scale):
        call("mh_upsample2d", _dt(x), _p(x), _p(out), B, C, iH, iW, scale, _stream())

    def upsample2d_nhwc(self, x, out, B, C, iH, iW, scale):
        call("mh_upsample2d_nhwc", _dt(x), _p(x), _p(out), B, C, iH, iW, scale, _stream())

    def nchw_to_nhwc(self, x, out, B, C, HW):
        call("mh_nchw_to_nhwc", _dt(x), _p(x), _p(out), B, C, HW, _stream())

    def nhwc_to_nchw(self, x, out, B, C, HW):
        call("mh_nhwc_to_nchw", _dt(x), _p(x), _p(out), B, C, HW, _stream())
