"""Device-resident entry points over torch CUDA(HIP) tensors.

torch only provides device memory and the stream here; all computation runs
in libinferno_hip.so.  Each function takes device tensors, launches on
torch's current stream (or ``stream``) and returns without synchronizing.
"""
from __future__ import annotations

import ctypes as C
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import Q4_K, IHIPArgumentError, check, lib
from .synth import BLOCK_BYTES, BLOCK_ELEMS


# torch's current-stream handle without building a Stream object (2-3 us of
# host time per call otherwise); the public API where torch lacks it.
_raw_current_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(stream=None) -> int:
    if stream is not None:
        return stream.cuda_stream
    if _raw_current_stream is not None:
        return _raw_current_stream(torch.cuda.current_device())
    return torch.cuda.current_stream().cuda_stream


def _ptr(t: torch.Tensor, dtype=None, what="tensor") -> int:
    if not t.is_cuda:
        raise IHIPArgumentError(_lib.IHIP_ERR_INVALID, f"{what} must be a device tensor")
    if dtype is not None and t.dtype != dtype:
        raise IHIPArgumentError(_lib.IHIP_ERR_INVALID, f"{what} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise IHIPArgumentError(_lib.IHIP_ERR_INVALID, f"{what} must be contiguous")
    return t.data_ptr()


@dataclass
class DeviceWeight:
    """GGML blocks of an ``outer x inner`` row-major matrix in device memory."""
    data: torch.Tensor        # uint8, device
    ggml_type: int
    inner: int
    outer: int

    @classmethod
    def upload(cls, host_bytes, ggml_type: int, inner: int, outer: int, device="cuda"):
        t = torch.as_tensor(host_bytes, dtype=torch.uint8).to(device)
        w = cls(t, ggml_type, inner, outer)
        w.validate()
        return w

    def validate(self):
        be = BLOCK_ELEMS[self.ggml_type]
        need = self.outer * (self.inner // be) * BLOCK_BYTES[self.ggml_type]
        if self.inner % be or self.data.numel() < need:
            raise IHIPArgumentError(_lib.IHIP_ERR_INVALID, "weight bytes do not match the shape")

    @property
    def nbytes(self) -> int:
        return self.outer * (self.inner // BLOCK_ELEMS[self.ggml_type]) * BLOCK_BYTES[self.ggml_type]


class ArgmaxWorkspace:
    """IHIP_ARGMAX_WS_BYTES of device memory for the per-workgroup partial
    maxima, plus the token/flags outputs.  Calls sharing one workspace must
    not overlap on the GPU."""

    def __init__(self, device="cuda"):
        self.ws = torch.zeros(_lib.ARGMAX_WS_BYTES, dtype=torch.uint8, device=device)
        self.token = torch.zeros(1, dtype=torch.int32, device=device)
        self.flags = torch.zeros(1, dtype=torch.int32, device=device)

    def result(self) -> int:
        """Synchronize and return the 0-based token, raising like
        src/CommonOps.jl:149-152 on NaN/+Inf."""
        torch.cuda.synchronize()
        fl = int(self.flags.item())
        if fl & _lib.FLAG_NAN:
            raise IHIPArgumentError(_lib.IHIP_ERR_NONFINITE, "logits must not contain NaN")
        if fl & _lib.FLAG_POSINF:
            raise IHIPArgumentError(_lib.IHIP_ERR_NONFINITE, "logits must not contain +Inf")
        return int(self.token.item())


class WeightGroup:
    """Host weights of one GGML type and row length uploaded back to back as
    one registered weight (ihip_weight_register_group), e.g. wq, wk and wv:
    `whole` is the group as one DeviceWeight of the summed rows, `members[i]`
    member i's rows inside it, `offsets[i]` its first output row.  Freed by
    release()."""

    def __init__(self, hosts, ggml_type: int, inner: int, outers):
        import numpy as np
        src = [np.ascontiguousarray(h, dtype=np.uint8) for h in hosts]  # alive through the upload
        n = len(src)
        ptrs = (C.c_void_p * n)(*[a.ctypes.data for a in src])
        rows = (C.c_int * n)(*outers)
        h = C.c_uint64(0)
        check(lib().ihip_weight_register_group(ptrs, rows, n, ggml_type, inner, C.byref(h)))
        del src
        self.handle = h.value
        p = C.c_void_p(0)
        check(lib().ihip_weight_device_ptr(self.handle, C.byref(p)))
        self.ptr = p.value
        self.ggml_type, self.inner, self.outers = ggml_type, inner, list(outers)
        self.offsets = [sum(outers[:i]) for i in range(n)]

    def member_ptr(self, i: int) -> int:
        return self.ptr + lib().ihip_weight_bytes(self.ggml_type, self.inner, self.offsets[i])

    def gemv_norm(self, norm_w: torch.Tensor, eps: float, x: torch.Tensor, out: torch.Tensor = None,
                  xn: torch.Tensor = None, stream=None) -> torch.Tensor:
        """Every member's outputs of the normed x in one launch where the norm
        folds (ihip_gemv_norm_dev over the group)."""
        total = sum(self.outers)
        if out is None:
            out = torch.empty(total, dtype=torch.float32, device=x.device)
        if xn is None:
            xn = torch.empty(self.inner, dtype=torch.float32, device=x.device)
        check(lib().ihip_gemv_norm_dev(self.ggml_type, self.ptr, _ptr(norm_w, torch.float32, "norm_w"), eps,
                                       _ptr(x, torch.float32, "x"), _ptr(xn, torch.float32, "xn"),
                                       _ptr(out, torch.float32, "out"), self.inner, total, _stream(stream)))
        return out

    def gemv(self, x: torch.Tensor, out: torch.Tensor = None, stream=None) -> torch.Tensor:
        """Every member's outputs in one launch: out[offsets[i]:][:outers[i]]."""
        total = sum(self.outers)
        if out is None:
            out = torch.empty(total, dtype=torch.float32, device=x.device)
        check(lib().ihip_gemv_dev(self.ggml_type, self.ptr, _ptr(x, torch.float32, "x"),
                                  _ptr(out, torch.float32, "out"), self.inner, total, _stream(stream)))
        return out

    def release(self):
        if self.handle:
            check(lib().ihip_weight_release(self.handle))
            self.handle = 0


def gemv(w: DeviceWeight, x: torch.Tensor, out: torch.Tensor = None, stream=None):
    if out is None:
        out = torch.empty(w.outer, dtype=torch.float32, device=x.device)
    check(lib().ihip_gemv_dev(w.ggml_type, _ptr(w.data, torch.uint8, "w"), _ptr(x, torch.float32, "x"),
                              _ptr(out, torch.float32, "out"), w.inner, w.outer, _stream(stream)))
    return out


def gemv_add(w: DeviceWeight, x: torch.Tensor, resid: torch.Tensor, out: torch.Tensor = None,
             stream=None) -> torch.Tensor:
    """out = resid + W x in one launch (ihip_gemv_add_dev); out defaults to
    resid (in place), as the layer's x .+= residual (src/ModelCPU.jl:909)."""
    if out is None:
        out = resid
    check(lib().ihip_gemv_add_dev(w.ggml_type, _ptr(w.data), _ptr(x, torch.float32, "x"),
                                  _ptr(resid, torch.float32, "resid"), _ptr(out, torch.float32, "out"),
                                  w.inner, w.outer, _stream(stream)))
    return out


def gemv_norm(w: DeviceWeight, norm_w: torch.Tensor, eps: float, x: torch.Tensor,
              out: torch.Tensor = None, xn: torch.Tensor = None, stream=None) -> torch.Tensor:
    """out = W (rmsnorm(x) .* norm_w) (ihip_gemv_norm_dev): one launch where
    the norm folds into the GEMV, else the norm into xn (allocated here when
    not given) and the plain GEMV."""
    if out is None:
        out = torch.empty(w.outer, dtype=torch.float32, device=x.device)
    if xn is None:
        xn = torch.empty(w.inner, dtype=torch.float32, device=x.device)
    check(lib().ihip_gemv_norm_dev(w.ggml_type, _ptr(w.data), _ptr(norm_w, torch.float32, "norm_w"),
                                   eps, _ptr(x, torch.float32, "x"), _ptr(xn, torch.float32, "xn"),
                                   _ptr(out, torch.float32, "out"), w.inner, w.outer, _stream(stream)))
    return out


def dequantize(w: DeviceWeight, out: torch.Tensor = None, stream=None):
    n = w.inner * w.outer
    if out is None:
        out = torch.empty(n, dtype=torch.float32, device=w.data.device)
    check(lib().ihip_dequantize_dev(w.ggml_type, _ptr(w.data, torch.uint8, "w"),
                                    _ptr(out, torch.float32, "out"), n, _stream(stream)))
    return out


def gate_up_swiglu(wg: DeviceWeight, wu: DeviceWeight, x, h=None, stream=None):
    if h is None:
        h = torch.empty(wg.outer, dtype=torch.float32, device=x.device)
    check(lib().ihip_gate_up_swiglu_dev(wg.ggml_type, _ptr(wg.data), wu.ggml_type, _ptr(wu.data),
                                        _ptr(x, torch.float32, "x"), _ptr(h, torch.float32, "h"),
                                        wg.inner, wg.outer, _stream(stream)))
    return h


def ffn_swiglu(wg: DeviceWeight, wu: DeviceWeight, wd: DeviceWeight, x, h=None, y=None, stream=None):
    if h is None:
        h = torch.empty(wg.outer, dtype=torch.float32, device=x.device)
    if y is None:
        y = torch.empty(wd.outer, dtype=torch.float32, device=x.device)
    check(lib().ihip_ffn_swiglu_dev(wg.ggml_type, _ptr(wg.data), wu.ggml_type, _ptr(wu.data),
                                    wd.ggml_type, _ptr(wd.data), _ptr(x, torch.float32, "x"),
                                    _ptr(h, torch.float32, "h"), _ptr(y, torch.float32, "y"),
                                    wg.inner, wg.outer, _stream(stream)))
    return y


def lm_head_argmax(w: DeviceWeight, x, ws: ArgmaxWorkspace, logits=None, stream=None):
    """logits may be None; where the argmax is not fused into the GEMV (other
    types or shapes) a logits buffer is allocated for the call."""
    if logits is None and not lib().ihip_lm_head_fused(w.ggml_type, _ptr(w.data), _ptr(x, torch.float32, "x"),
                                                       w.inner, w.outer):
        logits = torch.empty(w.outer, dtype=torch.float32, device=x.device)
    lp = _ptr(logits, torch.float32, "logits") if logits is not None else None
    check(lib().ihip_lm_head_argmax_dev(w.ggml_type, _ptr(w.data), _ptr(x, torch.float32, "x"), lp,
                                        ws.token.data_ptr(), ws.flags.data_ptr(), w.inner, w.outer,
                                        ws.ws.data_ptr(), _stream(stream)))
    return logits


def argmax(logits: torch.Tensor, ws: ArgmaxWorkspace, stream=None):
    check(lib().ihip_argmax_dev(_ptr(logits, torch.float32, "logits"), logits.numel(),
                                ws.token.data_ptr(), ws.flags.data_ptr(), ws.ws.data_ptr(),
                                _stream(stream)))


def prefill_scratch(T: int, inner: int, device="cuda") -> torch.Tensor:
    """Caller scratch of ihip_prefill_q4_k_dev: the fp16 activations, one
    scale exponent per token and the partial sums of a split over K
    (ihip_prefill_scratch_bytes bytes)."""
    return torch.empty(lib().ihip_prefill_scratch_bytes(T, inner), dtype=torch.uint8, device=device)


def prefill_q4_k(w: DeviceWeight, X: torch.Tensor, Y: torch.Tensor = None, xh: torch.Tensor = None,
                 stream=None):
    if w.ggml_type != Q4_K:
        raise IHIPArgumentError(_lib.IHIP_ERR_INVALID, "prefill takes a Q4_K weight")
    T = X.shape[0]
    if xh is None:
        xh = prefill_scratch(T, w.inner, X.device)
    if Y is None:
        Y = torch.empty(T, w.outer, dtype=torch.float32, device=X.device)
    check(lib().ihip_prefill_q4_k_dev(_ptr(w.data), _ptr(X, torch.float32, "X"), _ptr(xh), _ptr(Y, torch.float32, "Y"),
                                      T, w.inner, w.outer, _stream(stream)))
    return Y


def prefill_convert(X: torch.Tensor, xh: torch.Tensor = None, stream=None) -> torch.Tensor:
    """The rounding half of prefill_q4_k (ihip_prefill_convert_dev): X (T x
    inner, inner > 512) into xh, which prefill_q4_k_xh then multiplies by any
    number of weights."""
    T, inner = X.shape
    if xh is None:
        xh = prefill_scratch(T, inner, device=X.device)
    check(lib().ihip_prefill_convert_dev(_ptr(X, torch.float32, "X"), _ptr(xh, torch.uint8, "xh"),
                                         T, inner, _stream(stream)))
    return xh


def prefill_q4_k_xh(w: DeviceWeight, xh: torch.Tensor, T: int, Y: torch.Tensor = None,
                    stream=None) -> torch.Tensor:
    """The product half (ihip_prefill_q4_k_xh_dev): Y = W X from rows that
    prefill_convert rounded into xh; bit-identical to prefill_q4_k."""
    if w.ggml_type != Q4_K:
        raise IHIPArgumentError(_lib.IHIP_ERR_INVALID, "prefill takes a Q4_K weight")
    if Y is None:
        Y = torch.empty(T, w.outer, dtype=torch.float32, device=xh.device)
    check(lib().ihip_prefill_q4_k_xh_dev(_ptr(w.data), _ptr(xh, torch.uint8, "xh"),
                                         _ptr(Y, torch.float32, "Y"), T, w.inner, w.outer,
                                         _stream(stream)))
    return Y


def prefill_q4_k_f32(w: DeviceWeight, X: torch.Tensor, Y: torch.Tensor = None, stream=None):
    """The prefill on fp32 operands (ihip_prefill_q4_k_f32_dev): within the row
    bound for any finite X, slower than prefill_q4_k on long rows."""
    if w.ggml_type != Q4_K:
        raise IHIPArgumentError(_lib.IHIP_ERR_INVALID, "prefill takes a Q4_K weight")
    T = X.shape[0]
    if Y is None:
        Y = torch.empty(T, w.outer, dtype=torch.float32, device=X.device)
    check(lib().ihip_prefill_q4_k_f32_dev(_ptr(w.data), _ptr(X, torch.float32, "X"),
                                          _ptr(Y, torch.float32, "Y"), T, w.inner, w.outer,
                                          _stream(stream)))
    return Y


def quantize_row_q8k(x: torch.Tensor, y: torch.Tensor = None, stream=None) -> torch.Tensor:
    """x (fp32, a multiple of 256 elements) -> Q8_K blocks (uint8, 292 bytes
    per 256 elements), as quantize_row_q8_K (src/kernels/quant_kernels.c:166-194)."""
    k = x.numel()
    if y is None:
        y = torch.empty(k // 256 * _lib.Q8_K_BYTES, dtype=torch.uint8, device=x.device)
    check(lib().ihip_quantize_row_q8_k_dev(_ptr(x, torch.float32, "x"), _ptr(y, torch.uint8, "y"), k,
                                           _stream(stream)))
    return y


def gemv_q8k(w: DeviceWeight, q8: torch.Tensor, out: torch.Tensor = None, stream=None) -> torch.Tensor:
    """out = W x with x given as Q8_K blocks: the reference C path's numerics
    (vec_dot_q{4,5,6}_K_q8_K per row, src/kernels/quant_kernels.c:204-521)."""
    if out is None:
        out = torch.empty(w.outer, dtype=torch.float32, device=q8.device)
    check(lib().ihip_gemv_q8k_dev(w.ggml_type, _ptr(w.data), _ptr(q8, torch.uint8, "q8"),
                                  _ptr(out, torch.float32, "out"), w.inner, w.outer, _stream(stream)))
    return out


def gemv_q8k_x(w: DeviceWeight, x: torch.Tensor, out: torch.Tensor = None, q8: torch.Tensor = None,
               stream=None) -> torch.Tensor:
    """out = W x in the reference C path's numerics with x given as fp32 (the
    reference's q{4,5,6}_k_gemv, src/kernels/quant_kernels.c:602-650): x is
    quantized to Q8_K inside the call; q8, when given (inner/256 * 292 bytes),
    receives the blocks (Q6_K, and an out that overlaps x, require it)."""
    if out is None:
        out = torch.empty(w.outer, dtype=torch.float32, device=x.device)
    check(lib().ihip_gemv_q8k_x_dev(w.ggml_type, _ptr(w.data), _ptr(x, torch.float32, "x"),
                                    _ptr(out, torch.float32, "out"),
                                    None if q8 is None else _ptr(q8, torch.uint8, "q8"),
                                    w.inner, w.outer, _stream(stream)))
    return out


def rmsnorm(x: torch.Tensor, w: torch.Tensor, eps: float, out: torch.Tensor = None,
            stream=None) -> torch.Tensor:
    """rmsnorm_cpu! (src/ModelCPU.jl:111-123): x * (1/sqrt(mean(x^2) + eps)) .* w."""
    if out is None:
        out = torch.empty_like(x)
    check(lib().ihip_rmsnorm_dev(_ptr(x, torch.float32, "x"), _ptr(w, torch.float32, "w"), eps,
                                 _ptr(out, torch.float32, "out"), x.numel(), _stream(stream)))
    return out


def ffn_block(wg: DeviceWeight, wu: DeviceWeight, wd: DeviceWeight, norm_w: torch.Tensor,
              eps: float, x: torch.Tensor, h: torch.Tensor = None, stream=None) -> torch.Tensor:
    """The MLP half of a decoder layer (src/ModelCPU.jl:913-920), in place on x:
    x += Wd (silu(Wg n) * (Wu n)), n = rmsnorm(x) .* norm_w."""
    if h is None:
        n = lib().ihip_ffn_block_scratch_floats(wg.ggml_type, wu.ggml_type, wg.inner, wg.outer)
        h = torch.empty(n, dtype=torch.float32, device=x.device)
    check(lib().ihip_ffn_block_dev(wg.ggml_type, _ptr(wg.data), wu.ggml_type, _ptr(wu.data),
                                   wd.ggml_type, _ptr(wd.data), _ptr(norm_w, torch.float32, "norm_w"),
                                   eps, _ptr(x, torch.float32, "x"), _ptr(h, torch.float32, "h"),
                                   wg.inner, wg.outer, _stream(stream)))
    return x


def lm_head_argmax_norm(w: DeviceWeight, norm_w: torch.Tensor, eps: float, x: torch.Tensor,
                        ws: "ArgmaxWorkspace", xn: torch.Tensor = None, logits: torch.Tensor = None,
                        stream=None):
    """Final norm + lm_head + greedy token (src/ModelCPU.jl:1014-1015); the
    token and flags land in ws.token / ws.flags (device)."""
    if xn is None:
        xn = torch.empty_like(x)
    if logits is None and not lib().ihip_lm_head_fused(w.ggml_type, _ptr(w.data), _ptr(xn, torch.float32, "xn"),
                                                       w.inner, w.outer):
        logits = torch.empty(w.outer, dtype=torch.float32, device=x.device)
    check(lib().ihip_lm_head_argmax_norm_dev(
        w.ggml_type, _ptr(w.data), _ptr(norm_w, torch.float32, "norm_w"), eps,
        _ptr(x, torch.float32, "x"), _ptr(xn, torch.float32, "xn"),
        None if logits is None else _ptr(logits, torch.float32, "logits"),
        ws.token.data_ptr(), ws.flags.data_ptr(), w.inner, w.outer, ws.ws.data_ptr(), _stream(stream)))
    return xn


# ---- attention over a paged cache ---------------------------------------------
_KV_TYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_ACT_TYPES = {torch.float32: _lib.F32, **_KV_TYPES}


def _invalid(msg: str):
    return IHIPArgumentError(_lib.IHIP_ERR_INVALID, msg)


def _at(t, dtype, what, dev, least=0):
    """Pointer of a contiguous tensor of `dtype` and at least `least` values on device
    `dev` (None: none)."""
    if t is None:
        return None
    if t.get_device() != dev:
        raise _invalid(f"{what} must be on device {dev}, not {t.device}")
    if t.dtype != dtype or not t.is_contiguous():
        raise _invalid(f"{what} must be contiguous {dtype}, got {t.dtype}")
    if least and t.numel() < least:
        raise _invalid(f"{what} holds {t.numel()} values, needs {least}")
    return t.data_ptr()


_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _launch(dev: int, stream, fn, *args):
    """fn(*args, stream) with the tensors' device current (the library launches
    there), on `stream` or that device's current one."""
    if dev == _current_device():
        rc = fn(*args, stream.cuda_stream if stream is not None else _raw_current_stream(dev) if _raw_current_stream
                else torch.cuda.current_stream().cuda_stream)
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, _stream(stream))
    if rc:
        check(rc)


def _same_device(dev: int, *others):
    for t in others:
        if t.index != dev:
            raise _invalid(f"a cache or batch on device {t.index}, tensors on {dev}")


def _fresh(stream, make):
    """make()'s tensor for a call on `stream`: allocated (and filled) there, since
    work that the current stream still has ahead of it may use the same memory, and
    kept from other uses while the current stream reads it."""
    if stream is None:
        return make()
    with torch.cuda.stream(stream):
        t = make()
    t.record_stream(torch.cuda.current_stream(t.device))
    return t


class KVCache:
    """The paged cache of one layer (k, v: pages x kv_heads x page_size x
    head_dim) or of several (layers in front): device tensors of fp16 or bf16
    whose pages are contiguous; layer and page strides are the tensors' own, so
    k and v may be two halves of one tensor."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor):
        for t, what in ((k, "k"), (v, "v")):
            if not t.is_cuda or t.dtype not in _KV_TYPES:
                raise _invalid(f"{what} must be an fp16 or bf16 device tensor")
            if t.dim() not in (4, 5):
                raise _invalid(f"{what} must be [layers x] pages x kv_heads x page_size x head_dim")
            if t.numel() == 0:
                raise _invalid(f"{what} is empty")
            _, heads, page, dim = t.shape[-4:]
            if t.stride()[-3:] != (page * dim, dim, 1):
                raise _invalid(f"a page of {what} must be contiguous")
        if k.shape != v.shape or k.dtype != v.dtype or k.stride()[:-3] != v.stride()[:-3]:
            raise _invalid("k and v differ in shape, type or strides")
        if k.device != v.device:
            raise _invalid("k and v are on different devices")
        self.k, self.v = k, v
        self.layers_dim = k.dim() == 5
        self.layers = k.shape[0] if k.dim() == 5 else 1
        self.layer_stride = k.stride(0) if k.dim() == 5 else 0
        self.pages, self.kv_heads, self.page_size, self.head_dim = k.shape[-4:]
        self.dtype, self.device, self.index = k.dtype, k.device, k.get_device()
        stride = k.stride(-4) if self.pages > 1 else self.kv_heads * self.page_size * self.head_dim
        self.struct = _lib.KVCacheStruct(k.data_ptr(), v.data_ptr(), _KV_TYPES[k.dtype], self.pages, self.page_size,
                                         self.kv_heads, self.head_dim, stride)
        self.ref = C.byref(self.struct)

    def layer(self, i: int) -> "KVCache":
        """Layer i's cache, which rope_kv and attn_paged take."""
        return KVCache(self.k[i], self.v[i]) if self.k.dim() == 5 else self


class KVBatch:
    """The sequences of a call (ihip_kv_batch): int32 device tensors q_starts
    (sequences + 1), kv_lens (sequences), page_table (sequences x pages), and the
    rows of q.  Their contents may change between calls, also under a captured
    graph."""

    def __init__(self, q_starts: torch.Tensor, kv_lens: torch.Tensor, page_table: torch.Tensor, tokens: int):
        n, self.index = kv_lens.numel(), kv_lens.get_device()
        for t, what in ((kv_lens, "kv_lens"), (q_starts, "q_starts"), (page_table, "page_table")):
            _ptr(t, torch.int32, what), _at(t, torch.int32, what, self.index)
        if q_starts.numel() != n + 1 or page_table.dim() != 2 or page_table.shape[0] != n:
            raise _invalid("q_starts has sequences + 1 entries, page_table a row a sequence")
        self.q_starts, self.kv_lens, self.page_table, self.tokens = q_starts, kv_lens, page_table, tokens
        self.sequences = n
        self.struct = _lib.KVBatchStruct(q_starts.data_ptr(), kv_lens.data_ptr(), page_table.data_ptr(), n,
                                         page_table.shape[1], tokens)
        self.ref = C.byref(self.struct)


def rope_turns(rot_dim: int, base: float, scaling: str = "none", factor: float = 1.0, original: int = 0,
               low: float = 1.0, high: float = 32.0, device="cuda"):
    """(turns, mscale) of ihip_rope_turns: rot_dim / 2 doubles on the device, laid
    out once per model, and the factor on the rotated values."""
    if scaling not in _lib.ROPE_SCALING:
        raise _invalid(f"unknown scaling {scaling}")
    host = (C.c_double * max(1, rot_dim // 2))()
    m = C.c_float(1.0)
    check(lib().ihip_rope_turns(_lib.ROPE_SCALING[scaling], rot_dim, base, factor, original, low, high, host,
                                C.byref(m)))
    return torch.tensor(list(host), dtype=torch.float64).to(device), m.value


def _heads(t: torch.Tensor, what, dev, tokens, heads, dim):
    """Pointer, row stride and heads of a tokens x heads x dim fp32 view whose rows
    are contiguous."""
    if t.dtype != torch.float32 or t.get_device() != dev or dev < 0:
        raise _invalid(f"{what} must be float32 on device {dev}")
    shape, stride = t.shape, t.stride()
    if len(shape) != 3:
        raise _invalid(f"{what} is not tokens x heads x head_dim")
    n, h, d = shape
    if n != tokens or d != dim or h != (heads or h) or h == 0:
        raise _invalid(f"{what} is {tuple(shape)}, not {tokens} x {heads or 'heads'} x {dim}")
    if n and (stride[2] != 1 or (stride[1] != d and h > 1)):
        raise _invalid(f"the heads of a token of {what} must be contiguous")
    return t.data_ptr(), stride[0] if n > 1 else h * d, h


def rope_kv(q: torch.Tensor, k, v, turns: torch.Tensor, cache: KVCache, batch: KVBatch, layout: str = "half",
            mscale: float = 1.0, q_norm=None, k_norm=None, eps: float = 1e-6, positions=None,
            out: torch.Tensor = None, out_dtype=None, flags=None, stream=None) -> torch.Tensor:
    """The q and k norms, the rotary positions and the append to the cache
    (ihip_rope_kv_dev).  q, k, v: tokens x heads x head_dim fp32, slices of a
    grouped projection's rows as they are; k and v None for q alone.  The rotated
    part of a head is 2 * turns.numel() values.  Returns q (out_dtype, default
    fp32)."""
    T, D = batch.tokens, cache.head_dim
    if cache.layers_dim:
        raise _invalid("pass one layer of the cache (cache.layer(i))")
    how = _lib.ROPE_LAYOUT.get(layout)
    if how is None:
        raise _invalid(f"unknown layout {layout}")
    if (k is None) != (v is None):
        raise _invalid("k and v go together")
    dev = q.get_device()
    _same_device(dev, cache, batch)
    qp, qs, H = _heads(q, "q", dev, T, None, D)
    kp, ks, vp, vs = None, 0, None, 0
    if k is not None:
        kp, ks, _ = _heads(k, "k", dev, T, cache.kv_heads, D)
        vp, vs, _ = _heads(v, "v", dev, T, cache.kv_heads, D)
    if out is None:
        out = _fresh(stream, lambda: torch.empty(q.shape, dtype=out_dtype or torch.float32, device=q.device))
    elif out.shape != q.shape:
        raise _invalid("out must have q's shape")
    kind = out.dtype
    act = _ACT_TYPES.get(kind)
    if act is None or (out_dtype is not None and kind != out_dtype):
        raise _invalid("out must be fp32, fp16 or bf16, and the type asked for")
    _launch(dev, stream, lib().ihip_rope_kv_dev, qp, qs, kp, ks, vp, vs, H,
            _at(q_norm, torch.float32, "q_norm", dev, D), _at(k_norm, torch.float32, "k_norm", dev, D), eps,
            _at(turns, torch.float64, "turns", dev), 2 * turns.numel(), how, mscale,
            _at(positions, torch.int32, "positions", dev, T), _at(out, kind, "out", dev), act, cache.ref, batch.ref,
            _at(flags, torch.int32, "flags", dev, 1))
    return out


def _counted(n: int, device):
    """n bytes whose front, the counts of attn_paged's parts, is zero."""
    t = torch.empty(n, dtype=torch.uint8, device=device)
    t[:_lib.ATTN_COUNT_BYTES].zero_()
    return t


def attn_workspace(q_heads: int, cache: KVCache, batch: KVBatch):
    """The workspace of attn_paged for a batch of these sizes (q of either type),
    or None where it needs none.  Its counts start as zeros, written on the current
    stream, and every call leaves them so.  Calls that share one must not overlap."""
    n = lib().ihip_attn_paged_scratch_bytes(_lib.F32, q_heads, cache.ref, batch.ref)
    return _counted(n, cache.device) if n else None


def attn_paged(q: torch.Tensor, cache: KVCache, batch: KVBatch, scale: float = None, softcap: float = 0.0,
               window: int = 0, prefix_lens=None, slopes=None, out: torch.Tensor = None, workspace=None, flags=None,
               stream=None) -> torch.Tensor:
    """Attention of the batch's new tokens over their pages (ihip_attn_paged_dev).
    q: tokens x q_heads x head_dim, fp32 or the cache's type, which out has too;
    scale defaults to head_dim ** -0.5.  Rows of out before the first
    sequence's and behind the last one's are not written."""
    T, D = batch.tokens, cache.head_dim
    if cache.layers_dim:
        raise _invalid("pass one layer of the cache (cache.layer(i))")
    shape, act = q.shape, _ACT_TYPES.get(q.dtype)
    if len(shape) != 3 or shape[0] != T or shape[2] != D:
        raise _invalid(f"q is {tuple(shape)}, not {T} x heads x {D}")
    if act is None:
        raise _invalid(f"q must be fp32, fp16 or bf16, got {q.dtype}")
    H, dev = shape[1], q.get_device()
    _same_device(dev, cache, batch)
    if out is None:
        out = _fresh(stream, lambda: torch.empty_like(q))
    elif out.shape != shape:
        raise _invalid("out must have q's shape and type")
    if workspace is None:
        n = lib().ihip_attn_paged_scratch_bytes(_lib.F32, H, cache.ref, batch.ref)
        if n:
            workspace = _fresh(stream, lambda: _counted(n, q.device))
    _launch(dev, stream, lib().ihip_attn_paged_dev, _at(q, q.dtype, "q", dev), act, _at(out, q.dtype, "out", dev), H,
            D ** -0.5 if scale is None else scale, softcap, window,
            _at(prefix_lens, torch.int32, "prefix_lens", dev, batch.sequences),
            _at(slopes, torch.float32, "slopes", dev, H), cache.ref, batch.ref, _at(flags, torch.int32, "flags", dev, 1),
            _at(workspace, torch.uint8, "workspace", dev), 0 if workspace is None else workspace.numel())
    return out


def kv_fork(table: torch.Tensor, lens: torch.Tensor, parents: torch.Tensor, refs: torch.Tensor, page_size: int,
            room: int = 0, flags=None, stream=None):
    """The page tables of the next step (ihip_kv_fork_dev): child c goes on from
    parents[c] (-1: empty) with room for `room` more tokens.  Returns the new
    table and lengths and the page copies that kv_copy has to make; refs is
    updated in place."""
    dev = table.get_device()
    tp = _ptr(table, torch.int32, "table")
    if table.dim() != 2 or lens.numel() != table.shape[0]:
        raise _invalid("table has a row and lens an entry a sequence")
    sequences, width = table.shape
    n, where = parents.numel(), table.device
    # the new table; its lengths, the copies and the scratch
    new = _fresh(stream, lambda: torch.empty(n, width, dtype=torch.int32, device=where))
    ints = _fresh(stream, lambda: torch.empty(5 * n, dtype=torch.int32, device=where))
    p = ints.data_ptr()
    _launch(dev, stream, lib().ihip_kv_fork_dev, tp, _at(lens, torch.int32, "lens", dev), sequences,
            _at(parents, torch.int32, "parents", dev), n, room, width, page_size, refs.numel(),
            _at(refs, torch.int32, "refs", dev), new.data_ptr(), p, p + 4 * n, p + 12 * n,
            _at(flags, torch.int32, "flags", dev, 1))
    return new, ints[:n], ints[n:3 * n].view(n, 2)


def kv_compact(table: torch.Tensor, refs: torch.Tensor, flags=None, stream=None):
    """The used pages moved to the front of the pool (ihip_kv_compact_dev): table
    and refs change in place; returns the moves (pages // 2 pairs, -1 behind the
    last) and their number, both for kv_copy."""
    dev, pages = table.get_device(), refs.numel()
    tp, n = _ptr(table, torch.int32, "table"), pages // 2
    # the moves, the scratch and the moves' number
    ints = _fresh(stream, lambda: torch.empty(2 * n + pages + 1, dtype=torch.int32, device=table.device))
    p = ints.data_ptr()
    _launch(dev, stream, lib().ihip_kv_compact_dev, tp, table.numel(), _at(refs, torch.int32, "refs", dev), pages, p,
            p + 4 * (2 * n + pages), p + 8 * n, _at(flags, torch.int32, "flags", dev, 1))
    return ints[:2 * n].view(n, 2), ints[2 * n + pages:]


def kv_copy(cache: KVCache, copies: torch.Tensor, count: torch.Tensor = None, flags=None, stream=None):
    """Copies pages copies[i, 0] -> copies[i, 1] in every layer of the cache
    (ihip_kv_copy_dev); pairs with a negative entry are skipped, and those from
    *count on."""
    if copies.dim() != 2 or copies.shape[1] != 2:
        raise _invalid("copies is pairs x 2")
    dev = cache.index
    _launch(dev, stream, lib().ihip_kv_copy_dev, cache.ref, cache.layers, cache.layer_stride,
            _at(copies, torch.int32, "copies", dev), copies.shape[0], _at(count, torch.int32, "count", dev, 1),
            _at(flags, torch.int32, "flags", dev, 1))


# ---- layers that keep a state ---------------------------------------------------
class StateBatch:
    """The sequences of a call on layers that keep a state (ihip_state_batch): int32
    device tensors q_starts (sequences + 1), slots (sequences) and, where some begin
    with the call, kv_lens (sequences: all their tokens), and the rows of the call.
    Their contents may change between calls, also under a captured graph.  most: the
    most new tokens of a sequence, 1 in a decode step (a help in the choice of kernels; 0:
    not known, and then a decode step is launched as the prompt that it might be)."""

    def __init__(self, q_starts: torch.Tensor, slots: torch.Tensor, tokens: int, kv_lens=None, most: int = 0):
        n, self.index = slots.numel(), slots.get_device()
        for t, what in ((slots, "slots"), (q_starts, "q_starts"), (kv_lens, "kv_lens")):
            if t is not None:
                _ptr(t, torch.int32, what), _at(t, torch.int32, what, self.index)
        if q_starts.numel() != n + 1 or (kv_lens is not None and kv_lens.numel() != n):
            raise _invalid("q_starts has sequences + 1 entries, kv_lens one a sequence")
        self.q_starts, self.slots, self.kv_lens, self.tokens = q_starts, slots, kv_lens, tokens
        self.sequences = n
        self.struct = _lib.StateBatchStruct(q_starts.data_ptr(), None if kv_lens is None else kv_lens.data_ptr(),
                                            slots.data_ptr(), n, tokens, most)
        self.ref = C.byref(self.struct)


def _slots(state: torch.Tensor, what: str, inner):
    """Floats from one slot of a pool to the next: a float32 tensor slots x inner whose
    slots are contiguous."""
    if not state.is_cuda or state.dtype != torch.float32 or state.dim() != len(inner) + 1 or state.shape[0] == 0:
        raise _invalid(f"{what} must be a float32 device tensor of slots x {' x '.join(inner)}")
    want, n = [], 1
    for d in reversed(state.shape[1:]):
        want.insert(0, n)
        n *= d
    if n == 0 or state.stride()[1:] != tuple(want):
        raise _invalid(f"a slot of {what} must be contiguous")
    return state.stride(0) if state.shape[0] > 1 else n


def _row_step(t: torch.Tensor, what, dev, dtype, tokens, *inner):
    """Pointer and row stride of a tokens x inner view whose rows are contiguous."""
    shape, stride = t.shape, t.stride()
    if t.dtype != dtype or t.get_device() != dev:
        raise _invalid(f"{what} must be {dtype} on device {dev}, got {t.dtype} on {t.device}")
    if shape != (tokens, *inner):
        raise _invalid(f"{what} is {tuple(shape)}, not {(tokens, *inner)}")
    n = 1
    for i in range(len(inner), 0, -1):
        if shape[i] > 1 and stride[i] != n and tokens:
            raise _invalid(f"a row of {what} must be contiguous")
        n *= shape[i]
    return t.data_ptr(), stride[0] if tokens > 1 else n


def _out_like(out, out_dtype, shape, default, device, stream):
    if out is None:
        return _fresh(stream, lambda: torch.empty(shape, dtype=out_dtype or default, device=device))
    if out.shape != shape or (out_dtype is not None and out.dtype != out_dtype):
        raise _invalid(f"out is {out.dtype} {tuple(out.shape)}, not {tuple(shape)} of the type asked for")
    return out


def short_conv(x: torch.Tensor, weight: torch.Tensor, state: torch.Tensor, batch: StateBatch, bias=None,
               silu: bool = True, out: torch.Tensor = None, out_dtype=None, flags=None, stream=None) -> torch.Tensor:
    """The causal convolution of a recurrent layer over each channel's last inputs
    (ihip_short_conv_dev).  x: tokens x channels (rows of a wider projection as they
    are), fp32, fp16 or bf16; weight: channels x width fp32, the newest input's last;
    state: slots x (width - 1) x channels fp32, updated in place.  Returns tokens x
    channels of out_dtype (default: x's type)."""
    dev = x.get_device()
    _same_device(dev, batch)
    act = _ACT_TYPES.get(x.dtype)
    if x.dim() != 2 or weight.dim() != 2 or act is None:
        raise _invalid("x is tokens x channels of fp32, fp16 or bf16, weight channels x width")
    channels, width = weight.shape
    step = _slots(state, "state", ("width - 1", "channels"))
    if state.shape[1:] != (width - 1, channels):
        raise _invalid(f"state is {tuple(state.shape)}, not slots x {width - 1} x {channels}")
    if state.get_device() != dev:
        raise _invalid(f"state must be on device {dev}")
    xp, xs = _row_step(x, "x", dev, x.dtype, batch.tokens, channels)
    out = _out_like(out, out_dtype, x.shape, x.dtype, x.device, stream)
    to = _ACT_TYPES.get(out.dtype)
    if to is None:
        raise _invalid("out must be fp32, fp16 or bf16")
    _launch(dev, stream, lib().ihip_short_conv_dev, xp, act, xs, _at(weight, torch.float32, "weight", dev),
            _at(bias, torch.float32, "bias", dev, channels), channels, width, int(silu), state.data_ptr(), step,
            state.shape[0], _at(out, out.dtype, "out", dev), to, batch.ref, _at(flags, torch.int32, "flags", dev, 1))
    return out


class DeltaLayer:
    """A layer of the gated delta rule (ihip_delta_layer): state (slots x v_heads x
    k_dim x v_dim fp32, updated in place by gated_delta), the heads of q and k, the
    heads' decay (at most 0, as a GGUF file's ssm_a) and dt_bias, and the output
    norm's weights (v_dim) or None.  scale defaults to k_dim ** -0.5."""

    def __init__(self, state: torch.Tensor, k_heads: int, decay: torch.Tensor, dt_bias: torch.Tensor, norm_w=None,
                 norm_eps: float = 1e-6, l2_eps: float = 1e-6, scale: float = None):
        step = _slots(state, "state", ("v_heads", "k_dim", "v_dim"))
        self.slots, self.v_heads, self.k_dim, self.v_dim = state.shape
        self.k_heads, self.index, self.device = k_heads, state.get_device(), state.device
        self.state, self.decay, self.dt_bias, self.norm_w = state, decay, dt_bias, norm_w
        dev = self.index
        self.struct = _lib.DeltaLayerStruct(
            state.data_ptr(), step, self.slots, k_heads, self.v_heads, self.k_dim, self.v_dim,
            _at(decay, torch.float32, "decay", dev, self.v_heads), _at(dt_bias, torch.float32, "dt_bias", dev, self.v_heads),
            _at(norm_w, torch.float32, "norm_w", dev, self.v_dim), norm_eps, l2_eps,
            self.k_dim ** -0.5 if scale is None else scale)
        self.ref = C.byref(self.struct)


def delta_workspace(layer: DeltaLayer, batch: StateBatch, dtype):
    """The workspace of gated_delta for a batch of these sizes, or of smaller ones, with
    q, k and v of `dtype`, or None where it needs none.  Calls that share one must not
    overlap."""
    n = lib().ihip_gated_delta_scratch_bytes(_ACT_TYPES.get(dtype, -1), layer.ref, batch.ref)
    return torch.empty(n, dtype=torch.uint8, device=layer.device) if n else None


def gated_delta(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, a: torch.Tensor, b: torch.Tensor, layer: DeltaLayer,
                batch: StateBatch, gate=None, out: torch.Tensor = None, out_dtype=None, workspace=None, flags=None,
                stream=None) -> torch.Tensor:
    """The gated delta rule over the batch's new tokens (ihip_gated_delta_dev): q, k
    (tokens x k_heads x k_dim) and v (tokens x v_heads x v_dim) of one type, slices of
    the short convolution's rows as they are; a, b: tokens x v_heads fp32; gate:
    tokens x v_heads x v_dim fp32 or None.  The layer's state is updated in place.
    Returns tokens x v_heads x v_dim of out_dtype (fp32 or q's type, the default)."""
    dev, T = q.get_device(), batch.tokens
    _same_device(dev, layer, batch)
    kind = q.dtype
    act = _ACT_TYPES.get(kind)
    if act is None:
        raise _invalid(f"q, k and v must be fp32, fp16 or bf16, got {kind}")
    K, H, dk, dv = layer.k_heads, layer.v_heads, layer.k_dim, layer.v_dim
    qp, qs = _row_step(q, "q", dev, kind, T, K, dk)
    kp, ks = _row_step(k, "k", dev, kind, T, K, dk)
    vp, vs = _row_step(v, "v", dev, kind, T, H, dv)
    ap, as_ = _row_step(a, "a", dev, torch.float32, T, H)
    bp, bs = _row_step(b, "b", dev, torch.float32, T, H)
    gp, gs = (None, 0) if gate is None else _row_step(gate, "gate", dev, torch.float32, T, H, dv)
    out = _out_like(out, out_dtype, v.shape, kind, q.device, stream)
    to = _ACT_TYPES.get(out.dtype)
    if to is None:
        raise _invalid("out must be fp32 or of q's type")
    if workspace is None:
        workspace = _fresh_bytes(stream, lib().ihip_gated_delta_scratch_bytes(act, layer.ref, batch.ref), q.device)
    _launch(dev, stream, lib().ihip_gated_delta_dev, qp, qs, kp, ks, vp, vs, act, ap, as_, bp, bs, gp, gs,
            _at(out, out.dtype, "out", dev), to, layer.ref, batch.ref, _at(flags, torch.int32, "flags", dev, 1),
            _at(workspace, torch.uint8, "workspace", dev), 0 if workspace is None else workspace.numel())
    return out


def _fresh_bytes(stream, n, device):
    return _fresh(stream, lambda: torch.empty(n, dtype=torch.uint8, device=device)) if n else None


# ---- the choice of a token --------------------------------------------------------
def sample_workspace(rows: int, vocab: int, device="cuda"):
    """The workspace of sample for rows x vocab logits, or fewer.  Calls that share one
    must not overlap."""
    n = lib().ihip_sample_scratch_bytes(rows, vocab)
    if not n:
        raise _invalid(f"{rows} rows of {vocab} logits")
    return torch.empty(n, dtype=torch.uint8, device=device)


def sample(logits: torch.Tensor, u: torch.Tensor, temperature=None, top_k=None, top_p=None, min_p=None,
           out: torch.Tensor = None, logprobs=None, flags=None, workspace=None, stream=None) -> torch.Tensor:
    """A token per row of logits (ihip_sample_dev): rows x vocab of fp32, fp16 or bf16,
    u (one number in [0, 1) a row) and, one value a row or None, temperature, top_p,
    min_p (fp32) and top_k (int32), all on the device.  Returns int32 tokens; logprobs
    (fp32) and flags (int32), where given, are written too."""
    if logits.dim() != 2:
        raise _invalid("logits are rows x vocab")
    kind, dev = _ACT_TYPES.get(logits.dtype), logits.get_device()
    rows, vocab = logits.shape
    if kind is None or dev < 0:
        raise _invalid("logits must be an fp32, fp16 or bf16 device tensor")
    if rows and vocab > 1 and logits.stride(1) != 1:
        raise _invalid("a row of logits must be contiguous")
    if out is None:
        out = _fresh(stream, lambda: torch.empty(rows, dtype=torch.int32, device=logits.device))
    if workspace is None:
        workspace = _fresh_bytes(stream, lib().ihip_sample_scratch_bytes(rows, vocab), logits.device)
    _launch(dev, stream, lib().ihip_sample_dev, logits.data_ptr(), kind, logits.stride(0) if rows > 1 else vocab, rows, vocab,
            _at(temperature, torch.float32, "temperature", dev, rows), _at(top_k, torch.int32, "top_k", dev, rows),
            _at(top_p, torch.float32, "top_p", dev, rows), _at(min_p, torch.float32, "min_p", dev, rows),
            _at(u, torch.float32, "u", dev, rows), _at(out, torch.int32, "out", dev, rows),
            _at(logprobs, torch.float32, "logprobs", dev, rows), _at(flags, torch.int32, "flags", dev, rows),
            _at(workspace, torch.uint8, "workspace", dev), 0 if workspace is None else workspace.numel())
    return out
