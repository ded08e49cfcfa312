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


def _float_dt(op, x):
    t = _torch()
    if x.dtype not in (t.float32, t.float16, t.bfloat16):
        raise ValueError(f"{op}: float32, float16 or bfloat16, not {x.dtype}")
    return dtype_code(x.dtype)


def _size(op, name, x, dim):
    if x.dim() <= dim:
        raise ValueError(f"{op}: {name} has no dimension {dim}")
    return x.shape[dim]


def _nbytes(x):
    return 0 if x is None else x.numel() * x.element_size()


class _Call:
    """The checks of a call whose sizes come from its tensors, and its stream:
    all tensors on one GPU, which is the current device while the call runs, on
    torch's current stream of that device."""

    def __init__(self, op, **tensors):
        self.op = op
        self.t = {k: v for k, v in tensors.items() if v is not None}
        devices = {v.device for v in self.t.values()}
        if len(devices) != 1 or next(iter(devices)).type != "cuda":
            raise ValueError(f"{op}: all tensors must be on one GPU, got {sorted(map(str, devices))}")
        self.guard = _torch().cuda.device(next(iter(devices)))

    def __enter__(self):
        self.guard.__enter__()
        self.stream = _stream()
        return self

    def __exit__(self, *exc):
        return self.guard.__exit__(*exc)

    def _each(self, names, ok, what):
        for n in names:
            if n in self.t and not ok(self.t[n]):
                raise ValueError(f"{self.op}: {n} must be {what}")
        return self

    def int32(self, *names):
        return self._each(names, lambda x: x.dtype == _torch().int32, "int32")

    def float32(self, *names):
        return self._each(names, lambda x: x.dtype == _torch().float32, "float32")

    def contiguous(self, *names):
        return self._each(names, lambda x: x.is_contiguous(), "contiguous")

    def shape(self, name, want):
        def ok(x):
            return x.dim() == len(want) and all(w is None or w == d for w, d in zip(want, x.shape))
        return self._each((name,), ok, "of shape [" + ", ".join("*" if w is None else str(w) for w in want) + "]")

    def pool(self):
        """(pages, Hkv, page, hd) of the cache operands, their shapes and types checked."""
        t = _torch()
        k = self.t["k_cache"]
        self.shape("k_cache", (None, None, None, None))
        n_pages, Hkv, page, hd = k.shape
        self.shape("v_cache", (n_pages, Hkv, hd, page)).shape("k_scale", (n_pages, Hkv)).shape("v_scale", (n_pages, Hkv))
        self._each(("k_cache", "v_cache"), lambda x: x.dtype in (t.uint8, t.float8_e4m3fn), "uint8 or float8_e4m3fn")
        self.float32("k_scale", "v_scale").contiguous("k_cache", "v_cache", "k_scale", "v_scale")
        return n_pages, Hkv, page, hd

    def row_stride(self, name):
        """Values between the rows of [rows, heads, hd] whose heads are contiguous."""
        x = self.t[name]
        rows, heads, hd = x.shape
        if (hd > 1 and x.stride(2) != 1) or (heads > 1 and x.stride(1) != hd):
            raise ValueError(f"{self.op}: the heads of {name} must be contiguous")
        return x.stride(0) if rows > 1 else heads * hd

    def workspace(self, ws, need):
        t = _torch()
        if ws is None:
            return t.empty(need, dtype=t.uint8, device=self.guard.idx) if need else None
        if ws.dtype != t.uint8:
            raise ValueError(f"{self.op}: the workspace must be uint8")
        return ws


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
    def page_plan(self, lens, new_lens, free_pages, tables, total_lens, cu, slots, positions, used, page, n_pages):
        """Pages and slots of a step's new tokens (mh_page_plan): ``new_lens``
        [B] more tokens behind ``lens`` [B]; ``tables`` [B, width] gets the pages taken
        from ``free_pages``; ``total_lens`` [B], ``cu`` [B + 1], ``slots``, ``positions`` (or
        None) and ``used`` [1] are written."""
        B = _size("page_plan", "lens", lens, 0)
        with _Call("page_plan", lens=lens, new_lens=new_lens, free_pages=free_pages, tables=tables, total_lens=total_lens, cu=cu,
                   slots=slots, positions=positions, used=used) as c:
            c.int32("lens", "new_lens", "free_pages", "tables", "total_lens", "cu", "slots", "positions", "used")
            c.contiguous("lens", "new_lens", "free_pages", "tables", "total_lens", "cu", "slots", "positions", "used")
            c.shape("new_lens", (B,)).shape("total_lens", (B,)).shape("cu", (B + 1,)).shape("used", (1,))
            c.shape("tables", (B, None)).shape("free_pages", (None,)).shape("slots", (None,))
            c.shape("positions", tuple(slots.shape))
            call("mh_page_plan", _p(lens), _p(new_lens), _p(free_pages), _p(tables), _p(total_lens), _p(cu), _p(slots),
                 _p(positions), _p(used), B, free_pages.shape[0], tables.shape[1], page, n_pages, slots.shape[0], c.stream)

    def kv_store_paged(self, k, v, slots, k_cache, v_cache, k_scale, v_scale):
        """Keys and values [n, Hkv, hd] (heads contiguous, any row stride of whole
        16 bytes) into their slots (mh_kv_store_paged): ``k_cache`` [pages, Hkv,
        page, hd] and ``v_cache`` [pages, Hkv, hd, page] of 8-bit elements,
        scales [pages, Hkv] float32."""
        with _Call("kv_store_paged", k=k, v=v, slots=slots, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale) as c:
            n_pages, Hkv, page, hd = c.pool()
            n = _size("kv_store_paged", "k", k, 0)
            c.shape("k", (n, Hkv, hd)).shape("v", (n, Hkv, hd)).shape("slots", (n,)).int32("slots").contiguous("slots")
            if v.dtype != k.dtype:
                raise ValueError("kv_store_paged: k and v must have one type")
            call("mh_kv_store_paged", _float_dt("kv_store_paged", k), _p(k), _p(v), c.row_stride("k"), c.row_stride("v"), _p(slots),
                 _p(k_cache), _p(v_cache), _p(k_scale), _p(v_scale), n, Hkv, hd, page, n_pages, c.stream)

    def attention_paged_workspace(self, q, k_cache, lens, max_q, max_len, window=0) -> int:
        """Bytes of workspace that ``attention_paged`` needs for these sizes."""
        n = ctypes.c_size_t()
        call("mh_attention_paged_workspace", _float_dt("attention_paged", q), lens.shape[0], q.shape[0], q.shape[1],
             k_cache.shape[1], q.shape[2], max_q, max_len, window, ctypes.byref(n))
        return n.value

    def attention_paged(self, q, k_cache, v_cache, k_scale, v_scale, tables, lens, cu, out, max_q, max_len, causal=True,
                        window=0, scale=None, workspace=None):
        """Attention of ragged queries over the paged cache (mh_attention_paged):
        request b's queries are rows cu[b]..cu[b+1]-1 of ``q`` and ``out`` [rows, Hq,
        hd], the last of its lens[b] tokens; ``tables`` [B, width].  ``scale`` None:
        1 / sqrt(hd).  ``workspace``: a uint8 tensor of
        ``attention_paged_workspace`` bytes, else one is allocated."""
        B = _size("attention_paged", "lens", lens, 0)
        with _Call("attention_paged", q=q, k_cache=k_cache, v_cache=v_cache, k_scale=k_scale, v_scale=v_scale, tables=tables,
                   lens=lens, cu=cu, out=out, workspace=workspace) as c:
            n_pages, Hkv, page, hd = c.pool()
            c.shape("q", (None, None, hd)).shape("out", tuple(q.shape)).shape("tables", (B, None)).shape("cu", (B + 1,))
            c.int32("tables", "lens", "cu").contiguous("tables", "lens", "cu", "workspace")
            if out.dtype != q.dtype:
                raise ValueError("attention_paged: q and out must have one type")
            if scale is not None and not float(scale):
                raise ValueError("attention_paged: scale 0 (None is 1 / sqrt(hd))")
            need = self.attention_paged_workspace(q, k_cache, lens, max_q, max_len, window)
            workspace = c.workspace(workspace, need)
            call("mh_attention_paged", _float_dt("attention_paged", q), _p(q), c.row_stride("q"), _p(k_cache), _p(v_cache), _p(k_scale),
                 _p(v_scale), _p(tables), _p(lens), _p(cu), _p(out), c.row_stride("out"), B, q.shape[0], q.shape[1], Hkv, hd,
                 page, n_pages, tables.shape[1], max_q, max_len, int(causal), window, 0.0 if scale is None else float(scale),
                 _p(workspace), _nbytes(workspace), c.stream)

    # ---- sampling (no MuNet counterpart) ---------------------------------------
    def sample_workspace(self, logits) -> int:
        """Bytes of workspace that ``sample`` needs for these logits."""
        n = ctypes.c_size_t()
        call("mh_sample_workspace", _float_dt("sample", logits), logits.shape[0], logits.shape[1], ctypes.byref(n))
        return n.value

    def sample(self, logits, u, out, temperature=None, top_k=None, top_p=None, min_p=None, logprob=None, workspace=None):
        """One token per row of ``logits`` [rows, cols], drawn with the uniform
        numbers ``u`` [rows] (mh_sample): ``out`` [rows] int32; ``temperature``, ``top_p``,
        ``min_p`` float32 and ``top_k`` int32 [rows], or None; ``logprob`` [rows] float32
        optional.  ``workspace``: a uint8 tensor of ``sample_workspace`` bytes,
        else one is allocated."""
        rows = _size("sample", "logits", logits, 0)
        with _Call("sample", logits=logits, u=u, out=out, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p,
                   logprob=logprob, workspace=workspace) as c:
            c.shape("logits", (rows, None))
            for name in ("u", "out", "temperature", "top_k", "top_p", "min_p", "logprob"):
                c.shape(name, (rows,))
            c.contiguous("u", "out", "temperature", "top_k", "top_p", "min_p", "logprob", "workspace")
            c.int32("out", "top_k").float32("u", "temperature", "top_p", "min_p", "logprob")
            if logits.shape[1] > 1 and logits.stride(1) != 1:
                raise ValueError("sample: logits must be contiguous along a row")
            ld = logits.stride(0) if rows > 1 else logits.shape[1]
            workspace = c.workspace(workspace, self.sample_workspace(logits))
            call("mh_sample", _float_dt("sample", logits), _p(logits), ld, rows, logits.shape[1], _p(u), _p(temperature),
                 _p(top_k), _p(top_p), _p(min_p), _p(out), _p(logprob), _p(workspace), _nbytes(workspace), c.stream)

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
