"""Block operators on torch tensors: norms with a gate, the linear layer in 8-bit integers, shared-prefix attention.

Thin callers of the C entries of the same names (include/condmdi.h, "block operators"): they check shapes, types and devices,
allocate outputs and scratch from torch's allocator and launch on the current stream of the tensors' device.  Nothing
synchronises, so every call can be captured into a graph; a tensor made on another stream is the caller's to order, as with any
torch operator.  There is no CPU path.

    r, h = gated_norm(x, y, gate=gate, scale=scale, shift=shift)        # differentiable
    qkv = linear_i8(h, w_q, w_scale, bias)                              # w_q, w_scale = quantize_rows(w), once
    out = shared_prefix_attention(q, prefix_k, prefix_v, own_k, own_v, own_len)
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _native as N

__all__ = ["gated_norm", "gated_norm_fwd", "gated_norm_vjp", "quantize_rows", "gemm_i8", "linear_i8", "shared_prefix_attention"]

_EPI = {"bias": 0, "gelu": 1, "resid": 3}
_CONTIGUOUS = torch.contiguous_format
# the descriptors' C layouts (native alignment): packing one costs a quarter of a microsecond, a ctypes structure two
_NORM_DESC = struct.Struct("@7i2f2P4q3P3q4P")
_NORM_GRADS = struct.Struct("@2P4q10Pq")
_PREFIX_DESC = struct.Struct("@9if5P13qP")


def _refuse(what: str):
    raise N.NativeError(what)


def _on_device(t: torch.Tensor, name: str) -> int:
    """The HIP device's index of a tensor."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if not t.is_cuda:
        _refuse(f"{name} must be on a HIP device (there is no CPU path), got {t.device}")
    return t.get_device()


def _elsewhere(name: str, t: torch.Tensor, device: int):
    _refuse(f"{name} is on {t.device}, the call's tensors on cuda:{device}")


def _on(device: int, entry, *args) -> int:
    """entry(*args) with `device` current; raises what the entry reports."""
    if torch._C._cuda_getDevice() == device:
        rc = entry(*args)
    else:
        with torch.cuda.device(device):
            rc = entry(*args)
    if rc < 0:
        N.check(int(rc))
    return rc


def _launch(device: int, entry, *args):
    """entry(*args, current stream of `device`)."""
    _on(device, entry, *args, torch._C._cuda_getCurrentRawStream(device))


def _no_tangent(name: str, *tensors):
    """A result without a tangent where an input carries one would be a derivative of zero, silently."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                _refuse(f"{name} has no forward-mode derivative: call it on tensors without a tangent")


def _no_backward(name: str, *tensors):
    """A result without a gradient where one is asked for would train nothing, silently; the same of tangents."""
    _no_tangent(name, *tensors)
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                _refuse(f"{name} has no backward pass: call it under torch.no_grad() or on detached tensors")


# ---- gated norm -------------------------------------------------------------------------------------------------------------

def _rows(t: torch.Tensor, name: str, like: torch.Tensor, device: int) -> torch.Tensor:
    """t as rows like x's that the kernels can read in place (contiguous columns), or a contiguous copy."""
    if t.shape != like.shape or t.dtype != like.dtype:
        _refuse(f"{name} must be {list(like.shape)} {like.dtype}, got {list(t.shape)} {t.dtype}")
    if t.get_device() != device:
        _elsewhere(name, t, device)
    return t if t.stride()[2] == 1 or t.shape[2] == 1 else t.contiguous()


_PARAMS = ("gate", "scale", "shift", "weight", "bias", "post_weight", "post_bias")


def _norm_desc(x, y, gate, scale, shift, weight, bias, post_weight, post_bias, post, pre, residual_scale, eps):
    """(packed descriptor, the tensors it points at in the order x, y, *_PARAMS, device)."""
    device = _on_device(x, "x")
    dtype, shape = x.dtype, x.shape
    code = N.CMDI_DT.get(dtype)
    if code is None or len(shape) != 3:
        _refuse(f"x must be [batch, seq, dim] float32, bfloat16 or float16, got {list(shape)} {dtype}")
    if post not in N.CMDI_NORMS or pre not in ("rms", "layer"):
        _refuse(f"post must be 'none', 'rms' or 'layer' and pre 'rms' or 'layer', got {post!r}, {pre!r}")
    b, s, d = shape
    xs = x.stride()
    if xs[2] != 1 and d != 1:
        x = x.contiguous()
        xs = x.stride()
    tensors, ptrs, strides, pdt = [x, y], [], [], None
    if y is not None:
        tensors[1] = y = _rows(y, "y", x, device)
        ys, yp = y.stride(), y.data_ptr()
    else:
        ys, yp = (0, 0), 0
    vector, of_samples = (d,), (b, d)
    for i, t in enumerate((gate, scale, shift, weight, bias, post_weight, post_bias)):
        if t is None:
            tensors.append(None)
            ptrs.append(0)
            strides.append(0)
            continue
        if pdt is None:
            pdt = t.dtype
            if pdt is not dtype and pdt is not torch.float32:
                _refuse(f"gate, scale, shift, weights and biases must all be float32 or all {dtype}, got {_PARAMS[i]} {pdt}")
        if t.dtype is not pdt:
            _refuse(f"gate, scale, shift, weights and biases must be of one type, got {_PARAMS[i]} {t.dtype} beside {pdt}")
        if t.get_device() != device:
            _elsewhere(_PARAMS[i], t, device)
        ts = t.shape
        if ts == vector:
            if not t.is_contiguous():
                t = t.contiguous()
            step = 0
        elif i < 3 and ts == of_samples:
            st = t.stride()
            if (st[1] != 1 and d > 1) or st[0] == 0:
                t = t.contiguous()
                st = t.stride()
            # a [1, dim] parameter still belongs to its sample (its gradient is [1, dim]): any stride but 0 says so
            step = st[0] if b > 1 else d
        else:
            _refuse(f"{_PARAMS[i]} must be [{d}]{f' or [{b}, {d}]' if i < 3 else ''}, got {list(ts)}")
        tensors.append(t)
        ptrs.append(t.data_ptr())
        strides.append(step)
    desc = _NORM_DESC.pack(b, s, d, code, code if pdt is None or pdt is dtype else 0, N.CMDI_NORMS[post], N.CMDI_NORMS[pre], residual_scale, eps,
                           x.data_ptr(), yp, xs[0], xs[1], ys[0], ys[1], *ptrs[:3], *strides[:3], *ptrs[3:])
    return desc, tensors, device


def _norm_fwd(x, y, gate, scale, shift, weight, bias, post_weight, post_bias, post, pre, residual_scale, eps):
    desc, tensors, device = _norm_desc(x, y, gate, scale, shift, weight, bias, post_weight, post_bias, post, pre, residual_scale, eps)
    x = tensors[0]
    r, h = torch.empty_like(x, memory_format=_CONTIGUOUS), torch.empty_like(x, memory_format=_CONTIGUOUS)
    _launch(device, N.load().cmdi_gated_norm_fwd, desc, r.data_ptr(), h.data_ptr())
    return r, h


_NORM_INPUTS = ("x", "y", "gate", "scale", "shift", "weight", "bias", "post_weight", "post_bias")


def _norm_vjp(args, kw, gr, gh, wanted):
    desc, tensors, device = _norm_desc(*args, **kw)
    x = tensors[0]
    if gr is not None:
        gr = _rows(gr, "grad_r", x, device)
    if gh is not None:
        gh = _rows(gh, "grad_h", x, device)
    make = torch.zeros_like if x.numel() == 0 else torch.empty_like
    out = {n: None if t is None or n not in wanted else make(t, memory_format=_CONTIGUOUS) for n, t in zip(_NORM_INPUTS, tensors)}
    if x.numel() == 0:
        return out
    rs, hs = (0, 0) if gr is None else gr.stride()[:2], (0, 0) if gh is None else gh.stride()[:2]
    lib = N.load()
    grads = [N.ptr(gr), N.ptr(gh), *rs, *hs, *(N.ptr(t) for t in out.values())]
    need = _on(device, lib.cmdi_gated_norm_vjp_workspace, desc, _NORM_GRADS.pack(*grads, 0, 0))
    work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _launch(device, lib.cmdi_gated_norm_vjp, desc, _NORM_GRADS.pack(*grads, N.ptr(work), need))
    return out


def _not_captured():
    if torch.cuda.is_current_stream_capturing():
        _refuse("gated_norm with gradients cannot be captured: use gated_norm_fwd and gated_norm_vjp inside a graph")


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, kw, *args):
        ctx.set_materialize_grads(False)
        ctx.kw = kw
        ctx.save_for_backward(*args)
        return _norm_fwd(*args, **kw)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gr, gh):
        _not_captured()                       # (the forward pass may have run before the capture)
        _no_tangent("gated_norm's backward pass", gr, gh)
        args = ctx.saved_tensors
        if gr is None and gh is None:
            return (None,) * (1 + len(args))
        wanted = [n for n, need in zip(_NORM_INPUTS, ctx.needs_input_grad[1:]) if need]
        out = _norm_vjp(args, ctx.kw, gr, gh, wanted)
        return (None, *(out[n] for n in _NORM_INPUTS))


def gated_norm(x, y=None, *, gate=None, residual_scale=1.0, post="none", post_weight=None, post_bias=None, pre="layer", weight=None, bias=None,
               scale=None, shift=None, eps=1e-5):
    """The norms around a block with its gate and residual scale -> (r, h):

        r = residual_scale * x + gate * N_post(y),    h = (N_pre(r) * weight + bias) * (1 + scale) + shift

    x, y [batch, seq, dim] (float32, bfloat16 or float16; y None: no block in front); gate, scale, shift [dim] or [batch, dim];
    weight, bias, post_weight, post_bias [dim]; the parameters all float32 or all of x's type.  post 'none' | 'rms' | 'layer', pre
    'rms' | 'layer'.  Differentiable (once, in reverse mode) in every tensor; a call that would record or run a backward pass while its
    stream is being captured is refused: the engine accumulates a leaf's gradient on the stream where an eager graph has used it, and
    that work in the midst of a capture ends the process.  Capture gated_norm_fwd and gated_norm_vjp."""
    args = (x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    _no_tangent("gated_norm", *args)
    if torch.is_grad_enabled():
        for t in args:
            if t is not None and t.requires_grad:
                _on_device(x, "x")
                _not_captured()
                return _GatedNorm.apply(dict(post=post, pre=pre, residual_scale=residual_scale, eps=eps), *args)
    return _norm_fwd(*args, post, pre, residual_scale, eps)


def gated_norm_fwd(x, y=None, *, gate=None, residual_scale=1.0, post="none", post_weight=None, post_bias=None, pre="layer", weight=None, bias=None,
                   scale=None, shift=None, eps=1e-5):
    """gated_norm without a backward pass -> (r, h)."""
    _no_tangent("gated_norm_fwd", x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    return _norm_fwd(x, y, gate, scale, shift, weight, bias, post_weight, post_bias, post, pre, residual_scale, eps)


def gated_norm_vjp(grad_r, grad_h, x, y=None, *, gate=None, residual_scale=1.0, post="none", post_weight=None, post_bias=None, pre="layer", weight=None,
                   bias=None, scale=None, shift=None, eps=1e-5, wanted=_NORM_INPUTS):
    """Gradients of gated_norm's inputs for those of (r, h), either of which may be None -> {name: gradient, None where there is
    no such input or it is not `wanted`}.  Explicit counterpart of the autograd path, for graphs and hand-written loops."""
    unknown = set(wanted) - set(_NORM_INPUTS)
    if unknown:
        _refuse(f"no such inputs: {sorted(unknown)}")
    args = (x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    _no_tangent("gated_norm_vjp", grad_r, grad_h, *args)
    return _norm_vjp(args, dict(post=post, pre=pre, residual_scale=residual_scale, eps=eps),
                     grad_r, grad_h, wanted)


# ---- the linear layer in 8-bit integers ---------------------------------------------------------------------------------------

def _float_rows(x: torch.Tensor):
    """(x [rows, cols] with contiguous columns, its type's code, device)."""
    device = _on_device(x, "x")
    code = N.CMDI_DT.get(x.dtype)
    if code is None or x.dim() != 2:
        _refuse(f"x must be [rows, cols] float32, bfloat16 or float16, got {list(x.shape)} {x.dtype}")
    return x if x.stride()[1] == 1 or x.shape[1] == 1 else x.contiguous(), code, device


def quantize_rows(x: torch.Tensor):
    """Rows of x [rows, cols] in 8 bits -> (q int8 [rows, cols rounded up to 128] with zeros behind the columns, scale float32
    [rows]); x ~ q * scale, without a backward pass.  For weights [out, in] once (a parameter's .detach()), for activations
    [tokens, in] in every call."""
    x, code, device = _float_rows(x)
    _no_backward("quantize_rows", x)
    rows, cols = x.shape
    kp = (cols + 127) // 128 * 128
    q = torch.empty((rows, kp), dtype=torch.int8, device=x.device)
    scale = torch.empty((rows,), dtype=torch.float32, device=x.device)
    _launch(device, N.load().cmdi_quant_rows_i8, x.data_ptr(), code, rows, cols, x.stride()[0], q.data_ptr(), kp, scale.data_ptr())
    return q, scale


def _bytes_rows(t: torch.Tensor, name: str, device: int) -> torch.Tensor:
    if t.dtype != torch.int8 or t.dim() != 2:
        _refuse(f"{name} must be int8 [rows, k], got {list(t.shape)} {t.dtype}")
    if t.get_device() != device:
        _elsewhere(name, t, device)
    st = t.stride()
    if st[1] != 1 or st[0] % 16 or st[0] < t.shape[1] or st[0] > 1 << 22 or t.data_ptr() % 16:
        t = t.clone(memory_format=_CONTIGUOUS)          # (.contiguous() leaves a contiguous tensor where it is)
    return t


def _scales(t: torch.Tensor, name: str, size: int, device: int) -> torch.Tensor:
    if t.dtype != torch.float32 or t.shape != (size,):
        _refuse(f"{name} must be float32 [{size}], got {list(t.shape)} {t.dtype}")
    if t.get_device() != device:
        _elsewhere(name, t, device)
    return t if t.is_contiguous() else t.contiguous()


def _epilogue(epi, resid, m: int, n: int, dtype, device: int):
    """(code, resid that the kernels can read in place, its row stride)."""
    code = _EPI.get(epi)
    if code is None or (code == 3) != (resid is not None):
        _refuse(f"epi must be 'bias', 'gelu' or 'resid', the last with a resid tensor, got {epi!r}")
    if resid is None:
        return code, None, n
    if resid.shape != (m, n) or resid.dtype != dtype:
        _refuse(f"resid must be [{m}, {n}] {dtype}, got {list(resid.shape)} {resid.dtype}")
    if resid.get_device() != device:
        _elsewhere("resid", resid, device)
    if (n > 1 and resid.stride()[1] != 1) or (m > 1 and resid.stride()[0] < n):
        resid = resid.contiguous()
    return code, resid, resid.stride()[0] if m > 1 else n


def gemm_i8(a, a_scale, w, w_scale, bias=None, *, epi="bias", resid=None, dtype=torch.float32) -> torch.Tensor:
    """C = epi((a wᵀ) * a_scale[:, None] * w_scale + bias) for int8 rows a [M, K], w [N, K] (K a multiple of 128, as
    quantize_rows pads it), the sum exact in 32-bit integers.  epi 'bias', 'gelu' or 'resid' (+ resid [M, N] of `dtype`); C of
    `dtype`, without a backward pass."""
    device = _on_device(a, "a")
    _no_backward("gemm_i8", a_scale, w_scale, bias, resid)
    out = N.CMDI_DT.get(dtype)
    if out is None:
        _refuse(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    a, w = _bytes_rows(a, "a", device), _bytes_rows(w, "w", device)
    (m, k), n = a.shape, w.shape[0]
    if w.shape[1] != k:
        _refuse(f"a has {k} columns, w {w.shape[1]}")
    a_scale, w_scale = _scales(a_scale, "a_scale", m, device), _scales(w_scale, "w_scale", n, device)
    if bias is not None:
        bias = _scales(bias, "bias", n, device)
    code, resid, ldr = _epilogue(epi, resid, m, n, dtype, device)
    c = torch.empty((m, n), dtype=dtype, device=a.device)
    _launch(device, N.load().cmdi_gemm_i8, a.data_ptr(), a_scale.data_ptr(), w.data_ptr(), w_scale.data_ptr(), N.ptr(bias), N.ptr(resid), c.data_ptr(),
            m, n, k, a.stride()[0] if m > 1 else k, w.stride()[0] if n > 1 else k, n, ldr, out, code)
    return c


def linear_i8(x, w, w_scale, bias=None, *, epi="bias", resid=None) -> torch.Tensor:
    """A linear layer in 8-bit integers: rows of x [M, in] are quantised in the call, (w, w_scale) = quantize_rows(weight [out, in])
    once -> [M, out] of x's type, without a backward pass.  epi 'bias', 'gelu' or 'resid' (+ resid [M, out]); the same bits as
    gemm_i8 behind quantize_rows."""
    x, dt, device = _float_rows(x)
    _no_backward("linear_i8", x, w_scale, bias, resid)
    w = _bytes_rows(w, "w", device)
    (m, cols), (n, kp) = x.shape, w.shape
    if kp != (cols + 127) // 128 * 128:
        _refuse(f"w must be quantize_rows of a weight [out, {cols}], got {list(w.shape)}")
    w_scale = _scales(w_scale, "w_scale", n, device)
    if bias is not None:
        bias = _scales(bias, "bias", n, device)
    code, resid, ldr = _epilogue(epi, resid, m, n, x.dtype, device)
    where = x.device
    c = torch.empty((m, n), dtype=x.dtype, device=where)
    need = m * (kp + 4)                       # cmdi_linear_i8's scratch: the rows in 8 bits, then their scales
    work = torch.empty(need, dtype=torch.uint8, device=where)
    _launch(device, N.load().cmdi_linear_i8, x.data_ptr(), dt, m, cols, x.stride()[0], w.data_ptr(), w_scale.data_ptr(), N.ptr(bias), N.ptr(resid),
            c.data_ptr(), n, kp, w.stride()[0] if n > 1 else kp, n, ldr, code, work.data_ptr(), need)
    return c


# ---- shared-prefix attention ----------------------------------------------------------------------------------------------------

def _heads(t: torch.Tensor, name: str, shape, dtype, device: int, limit=1 << 62):
    """(t of `shape` with rows of contiguous, 16-byte aligned dims that the kernels can read in place, or a contiguous copy; its
    address; its strides without the last).  A dimension of one element may carry any stride: 0 stands for it."""
    if t.shape != shape or t.dtype is not dtype:
        _refuse(f"{name} must be {list(shape)} {dtype}, got {list(t.shape)} {t.dtype}")
    if t.get_device() != device:
        _elsewhere(name, t, device)
    st, at = t.stride(), t.data_ptr()
    if st[-1] == 1 and not at & 15 and st[-3] <= limit and not (st[0] | st[-2] | st[-3]) & 7 and at:
        return t, at, st[:-1]
    if not t.numel():
        return t, 0, (0,) * (len(shape) - 1)
    for again in (False, True):
        st, at = t.stride(), t.data_ptr()
        fine = st[-1] == 1 and at % 16 == 0
        if 1 in shape:
            st = [0 if n == 1 else s for n, s in zip(shape, st)]
        for s in st[:-1]:
            fine = fine and s % 8 == 0
        if again or (fine and st[-3] <= limit):
            return t, at, st[:-1]
        t = t.clone(memory_format=_CONTIGUOUS)          # (.contiguous() leaves a contiguous tensor where it is)


def shared_prefix_attention(q, prefix_k, prefix_v, own_k=None, own_v=None, own_len=None, *, causal=True, scale=None, return_lse=False):
    """Attention of sequences that share a prefix: out[b, i, h] = softmax(scale * q[b, i, h] · k) v over the prefix's keys and sample
    b's own first ``own_len[b]`` keys; with ``causal`` query i sees own keys 0 .. own_len[b] - queries + i (the queries are the
    sequence's newest tokens, their keys among the own ones), otherwise all own_len[b].

    q [batch, queries, heads, dim]; prefix_k, prefix_v [prefix, kv_heads, dim] (or None); own_k, own_v [batch, own_max, kv_heads,
    dim] (or None); own_len int32 [batch] on the device (None: own_max); bfloat16 or float16, dim 64 or 128, heads a multiple of
    kv_heads.  scale None: 1 / sqrt(dim).  -> out [batch, queries, heads, dim], with return_lse also the log-sums float32 [batch,
    heads, queries].  A query that sees no key (or scores of -inf alone) gives 0 and -inf.  Scores, maxima and sums
    are fp32; the softmax's weights meet the values in q's type (half a step of it relative each, in float16 also 2^-32 of the
    query's largest).  For serving: there is no backward pass."""
    device = _on_device(q, "q")
    _no_backward("shared_prefix_attention", q, prefix_k, prefix_v, own_k, own_v)
    dtype, shape = q.dtype, q.shape
    if len(shape) != 4 or dtype not in (torch.bfloat16, torch.float16):
        _refuse(f"q must be [batch, queries, heads, dim] bfloat16 or float16, got {list(shape)} {dtype}")
    if (prefix_k is None) != (prefix_v is None) or (own_k is None) != (own_v is None):
        _refuse("keys and values come together")
    b, n, h, d = shape
    pk = pv = ok = ov = p = o = 0
    ps = pvs = (0, 0)
    os_ = ovs = (0, 0, 0)
    hk = None
    if prefix_k is not None:
        if prefix_k.dim() != 3:
            _refuse(f"prefix_k must be [prefix, kv_heads, dim], got {list(prefix_k.shape)}")
        p, hk = prefix_k.shape[:2]
        prefix_k, pk, ps = _heads(prefix_k, "prefix_k", (p, hk, d), dtype, device, 1 << 23)
        prefix_v, pv, pvs = _heads(prefix_v, "prefix_v", (p, hk, d), dtype, device, 1 << 23)
    if own_k is not None:
        if own_k.dim() != 4:
            _refuse(f"own_k must be [batch, own_max, kv_heads, dim], got {list(own_k.shape)}")
        o = own_k.shape[1]
        hk = own_k.shape[2] if hk is None else hk
        own_k, ok, os_ = _heads(own_k, "own_k", (b, o, hk, d), dtype, device, 1 << 23)
        own_v, ov, ovs = _heads(own_v, "own_v", (b, o, hk, d), dtype, device, 1 << 23)
    if hk is None:
        _refuse("no keys: give a prefix, own keys or both")
    lens = 0
    if own_len is not None:
        if own_k is None or own_len.shape != (b,) or own_len.dtype != torch.int32:
            _refuse(f"own_len must be int32 [{b}] beside own keys, got {list(own_len.shape)} {own_len.dtype}")
        if own_len.get_device() != device:
            _elsewhere("own_len", own_len, device)
        own_len = own_len if own_len.is_contiguous() else own_len.contiguous()
        lens = own_len.data_ptr()
    q, qp, qs = _heads(q, "q", shape, dtype, device)
    desc = _PREFIX_DESC.pack(b, n, h, hk, d, p, o, 1 if causal else 0, N.CMDI_DT[dtype], 1.0 / math.sqrt(d) if scale is None else scale, qp, pk, pv, ok, ov,
                             *qs, *ps, *pvs, *os_, *ovs, lens)
    out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    lse = torch.empty((b, h, n), dtype=torch.float32, device=q.device) if return_lse else None
    lib = N.load()
    need = _on(device, lib.cmdi_prefix_attention_workspace, desc)
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    _launch(device, lib.cmdi_prefix_attention, desc, out.data_ptr(), N.ptr(lse), N.ptr(work), need)
    return (out, lse) if return_lse else out
