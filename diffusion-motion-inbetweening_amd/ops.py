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
from typing import Optional

import torch

from . import _native as N

__all__ = ["gated_norm", "gated_norm_fwd", "gated_norm_vjp", "quantize_rows", "gemm_i8", "linear_i8", "shared_prefix_attention"]

_EPI = {"bias": 0, "gelu": 1, "resid": 3}


def _refuse(what: str):
    raise N.NativeError(what)


def _on_device(t: torch.Tensor, name: str) -> torch.device:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.device.type != "cuda":
        _refuse(f"{name} must be on a HIP device (there is no CPU path), got {t.device}")
    return t.device


def _same_device(device: torch.device, **tensors):
    for name, t in tensors.items():
        if t is not None and t.device != device:
            _refuse(f"{name} is on {t.device}, the call's tensors on {device}")


class _On:
    """The tensors' device made current for the launches (nothing to do where it is already)."""

    def __init__(self, device):
        self.device = device

    def __enter__(self):
        self.before = torch.cuda.current_device()
        if self.before != self.device.index:
            torch.cuda.set_device(self.device)
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.before != self.device.index:
            torch.cuda.set_device(self.before)


# ---- gated norm -------------------------------------------------------------------------------------------------------------

def _rows(t: torch.Tensor, name: str, like: Optional[torch.Tensor] = None) -> torch.Tensor:
    """t as [batch, seq, dim] rows that the kernels can read in place (contiguous columns), or a contiguous copy."""
    if t.dim() != 3:
        _refuse(f"{name} must be [batch, seq, dim], got {tuple(t.shape)}")
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype):
        _refuse(f"{name} must be {tuple(like.shape)} {like.dtype}, got {tuple(t.shape)} {t.dtype}")
    return t if t.shape[2] == 1 or t.stride(2) == 1 else t.contiguous()


def _param(t: Optional[torch.Tensor], name: str, x: torch.Tensor, dtype, per_sample: bool) -> Optional[torch.Tensor]:
    if t is None:
        return None
    b, _, d = x.shape
    if t.dtype != dtype:
        _refuse(f"{name} must be {dtype} like the other parameters, got {t.dtype}")
    if t.shape != (d,) and not (per_sample and t.shape == (b, d)):
        _refuse(f"{name} must be [{d}]{f' or [{b}, {d}]' if per_sample else ''}, got {tuple(t.shape)}")
    if (d > 1 and t.stride(-1) != 1) or (t.dim() == 2 and t.stride(0) == 0):
        t = t.contiguous()
    return t


def _stride(t: Optional[torch.Tensor]) -> int:
    # a [1, dim] parameter still belongs to its sample (its gradient is [1, dim]): any stride but 0 says so
    return 0 if t is None or t.dim() == 1 else max(1, t.stride(0)) if t.shape[0] > 1 else t.shape[1]


def _norm_desc(x, y, gate, scale, shift, weight, bias, post_weight, post_bias, post, pre, residual_scale, eps):
    """(desc, the tensors it points at in the order x, y, gate, scale, shift, weight, bias, post_weight, post_bias)."""
    device = _on_device(x, "x")
    if x.dtype not in N.CMDI_DT:
        _refuse(f"x must be float32, bfloat16 or float16, got {x.dtype}")
    if post not in N.CMDI_NORMS or pre not in ("rms", "layer"):
        _refuse(f"post must be 'none', 'rms' or 'layer' and pre 'rms' or 'layer', got {post!r}, {pre!r}")
    x = _rows(x, "x")
    if y is not None:
        y = _rows(y, "y", x)
    params = dict(gate=gate, scale=scale, shift=shift, weight=weight, bias=bias, post_weight=post_weight, post_bias=post_bias)
    _same_device(device, y=y, **params)
    dtypes = {t.dtype for t in params.values() if t is not None}
    dtype = dtypes.pop() if dtypes else x.dtype
    if dtypes or dtype not in (x.dtype, torch.float32):
        _refuse(f"gate, scale, shift, weights and biases must all be float32 or all {x.dtype}")
    p = {k: _param(t, k, x, dtype, k in ("gate", "scale", "shift")) for k, t in params.items()}
    b, s, d = x.shape
    desc = N.GatedNormDesc(b, s, d, N.CMDI_DT[x.dtype], N.CMDI_DT[dtype], N.CMDI_NORMS[post], N.CMDI_NORMS[pre], float(residual_scale),
                           float(eps), N.ptr(x), N.ptr(y), (C.c_int64 * 2)(x.stride(0), x.stride(1)),
                           (C.c_int64 * 2)(*((y.stride(0), y.stride(1)) if y is not None else (0, 0))), N.ptr(p["gate"]), N.ptr(p["scale"]),
                           N.ptr(p["shift"]), _stride(p["gate"]), _stride(p["scale"]), _stride(p["shift"]), N.ptr(p["weight"]), N.ptr(p["bias"]),
                           N.ptr(p["post_weight"]), N.ptr(p["post_bias"]))
    return desc, (x, y, *p.values())


def _norm_fwd(args, kw):
    desc, tensors = _norm_desc(*args, **kw)
    x = tensors[0]
    r, h = torch.empty(x.shape, dtype=x.dtype, device=x.device), torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _On(x.device) as stream:
        N.check(N.load().cmdi_gated_norm_fwd(C.byref(desc), N.ptr(r), N.ptr(h), stream))
    return r, h


_NORM_INPUTS = ("x", "y", "gate", "scale", "shift", "weight", "bias", "post_weight", "post_bias")


def _norm_vjp(args, kw, gr, gh, wanted):
    desc, tensors = _norm_desc(*args, **kw)
    x = tensors[0]
    _same_device(x.device, grad_r=gr, grad_h=gh)
    gr, gh = (None if g is None else _rows(g, n, x) for g, n in ((gr, "grad_r"), (gh, "grad_h")))
    empty = x.numel() == 0
    out = {n: None if t is None or n not in wanted else torch.zeros(t.shape, dtype=t.dtype, device=t.device) if empty else
           torch.empty(t.shape, dtype=t.dtype, device=t.device) for n, t in zip(_NORM_INPUTS, tensors)}
    if empty:
        return out
    pair = lambda g: (C.c_int64 * 2)(*((g.stride(0), g.stride(1)) if g is not None else (0, 0)))  # noqa: E731
    grads = N.GatedNormGrads(N.ptr(gr), N.ptr(gh), pair(gr), pair(gh), *(N.ptr(out[n]) for n in _NORM_INPUTS), 0, 0)
    lib = N.load()
    need = lib.cmdi_gated_norm_vjp_workspace(C.byref(desc), C.byref(grads))
    if need < 0:
        N.check(int(need))
    work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    grads.d_work, grads.work_bytes = N.ptr(work), need
    with _On(x.device) as stream:
        N.check(lib.cmdi_gated_norm_vjp(C.byref(desc), C.byref(grads), stream))
    return out


class _GatedNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, kw, *args):
        ctx.set_materialize_grads(False)
        ctx.kw = kw
        ctx.save_for_backward(*args)
        return _norm_fwd(args, kw)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gr, gh):
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
    'rms' | 'layer'.  Differentiable (once) in every tensor; a call that would record a backward pass while its stream is
    being captured is refused: capture gated_norm_fwd and gated_norm_vjp."""
    args = (x, y, gate, scale, shift, weight, bias, post_weight, post_bias)
    kw = dict(post=post, pre=pre, residual_scale=residual_scale, eps=eps)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args):
        if torch.cuda.is_current_stream_capturing():
            _refuse("gated_norm with gradients cannot be captured: use gated_norm_fwd and gated_norm_vjp inside a graph")
        return _GatedNorm.apply(kw, *args)
    return _norm_fwd(args, kw)


def gated_norm_fwd(x, y=None, *, gate=None, residual_scale=1.0, post="none", post_weight=None, post_bias=None, pre="layer", weight=None, bias=None,
                   scale=None, shift=None, eps=1e-5):
    """gated_norm without a backward pass -> (r, h)."""
    return _norm_fwd((x, y, gate, scale, shift, weight, bias, post_weight, post_bias), dict(post=post, pre=pre, residual_scale=residual_scale, eps=eps))


def gated_norm_vjp(grad_r, grad_h, x, y=None, *, gate=None, residual_scale=1.0, post="none", post_weight=None, post_bias=None, pre="layer", weight=None,
                   bias=None, scale=None, shift=None, eps=1e-5, wanted=_NORM_INPUTS):
    """Gradients of gated_norm's inputs for those of (r, h), either of which may be None -> {name: gradient, None where there is
    no such input or it is not `wanted`}.  Explicit counterpart of the autograd path, for graphs and hand-written loops."""
    unknown = set(wanted) - set(_NORM_INPUTS)
    if unknown:
        _refuse(f"no such inputs: {sorted(unknown)}")
    return _norm_vjp((x, y, gate, scale, shift, weight, bias, post_weight, post_bias), dict(post=post, pre=pre, residual_scale=residual_scale, eps=eps),
                     grad_r, grad_h, wanted)


# ---- the linear layer in 8-bit integers ---------------------------------------------------------------------------------------

def quantize_rows(x: torch.Tensor):
    """Rows of x [rows, cols] in 8 bits -> (q int8 [rows, cols rounded up to 128] with zeros behind the columns, scale float32
    [rows]); x ~ q * scale.  For weights [out, in] once, for activations [tokens, in] in every call."""
    device = _on_device(x, "x")
    if x.dim() != 2 or x.dtype not in N.CMDI_DT:
        _refuse(f"x must be [rows, cols] float32, bfloat16 or float16, got {tuple(x.shape)} {x.dtype}")
    rows, cols = x.shape
    if cols > 1 and x.stride(1) != 1:
        x = x.contiguous()
    kp = (cols + 127) // 128 * 128
    q = torch.empty((rows, kp), dtype=torch.int8, device=device)
    scale = torch.empty((rows,), dtype=torch.float32, device=device)
    with _On(device) as stream:
        N.check(N.load().cmdi_quant_rows_i8(N.ptr(x), N.CMDI_DT[x.dtype], rows, cols, x.stride(0), N.ptr(q), kp, N.ptr(scale), stream))
    return q, scale


def _bytes_rows(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 2 or t.dtype != torch.int8:
        _refuse(f"{name} must be int8 [rows, k], got {tuple(t.shape)} {t.dtype}")
    if t.stride(1) != 1 or t.stride(0) % 16 or t.stride(0) < t.shape[1] or t.data_ptr() % 16:
        t = t.contiguous()
    return t


def gemm_i8(a, a_scale, w, w_scale, bias=None, *, epi="bias", resid=None, dtype=torch.float32) -> torch.Tensor:
    """C = epi((a wᵀ) * a_scale[:, None] * w_scale + bias) for int8 rows a [M, K], w [N, K] (K a multiple of 128, as
    quantize_rows pads it), the sum exact in 32-bit integers.  epi 'bias', 'gelu' or 'resid' (+ resid [M, N] of `dtype`); C of
    `dtype`."""
    device = _on_device(a, "a")
    _same_device(device, a_scale=a_scale, w=w, w_scale=w_scale, bias=bias, resid=resid)
    if epi not in _EPI or (epi == "resid") != (resid is not None):
        _refuse(f"epi must be 'bias', 'gelu' or 'resid', the last with a resid tensor, got {epi!r}")
    if dtype not in N.CMDI_DT:
        _refuse(f"dtype must be float32, bfloat16 or float16, got {dtype}")
    a, w = _bytes_rows(a, "a"), _bytes_rows(w, "w")
    (m, k), n = a.shape, w.shape[0]
    if w.shape[1] != k:
        _refuse(f"a has {k} columns, w {w.shape[1]}")
    for name, t, size in (("a_scale", a_scale, m), ("w_scale", w_scale, n), ("bias", bias, n)):
        if t is not None and (t.shape != (size,) or t.dtype != torch.float32):
            _refuse(f"{name} must be float32 [{size}], got {tuple(t.shape)} {t.dtype}")
    a_scale, w_scale = a_scale.contiguous(), w_scale.contiguous()
    bias = None if bias is None else bias.contiguous()
    if resid is not None:
        if resid.shape != (m, n) or resid.dtype != dtype:
            _refuse(f"resid must be [{m}, {n}] {dtype}, got {tuple(resid.shape)} {resid.dtype}")
        if (n > 1 and resid.stride(1) != 1) or (m > 1 and resid.stride(0) < n):
            resid = resid.contiguous()
    c = torch.empty((m, n), dtype=dtype, device=device)
    with _On(device) as stream:
        N.check(N.load().cmdi_gemm_i8(N.ptr(a), N.ptr(a_scale), N.ptr(w), N.ptr(w_scale), N.ptr(bias), N.ptr(resid), N.ptr(c), m, n, k,
                                      max(a.stride(0), k) if m > 1 else k, max(w.stride(0), k) if n > 1 else k, n,
                                      n if resid is None or m <= 1 else resid.stride(0), N.CMDI_DT[dtype], _EPI[epi], stream))
    return c


def linear_i8(x, w, w_scale, bias=None, *, epi="bias", resid=None) -> torch.Tensor:
    """A linear layer in 8-bit integers: rows of x [M, in] are quantised in the call, (w, w_scale) = quantize_rows(weight [out, in])
    once -> [M, out] of x's type.  epi 'bias', 'gelu' or 'resid' (+ resid [M, out])."""
    _on_device(x, "x")
    if x.dim() != 2 or x.dtype not in N.CMDI_DT:
        _refuse(f"x must be [rows, cols] float32, bfloat16 or float16, got {tuple(x.shape)} {x.dtype}")
    if w.dim() != 2 or w.shape[1] != (x.shape[1] + 127) // 128 * 128:
        _refuse(f"w must be quantize_rows of a weight [out, {x.shape[1]}], got {tuple(w.shape)}")
    q, scale = quantize_rows(x)
    return gemm_i8(q, scale, w, w_scale, bias, epi=epi, resid=resid, dtype=x.dtype)


# ---- shared-prefix attention ----------------------------------------------------------------------------------------------------

def _heads(t: torch.Tensor, name: str, shape, dtype) -> torch.Tensor:
    """t of `shape` with rows of contiguous, 16-byte aligned dims that the kernels can read in place, or a contiguous copy."""
    if tuple(t.shape) != tuple(shape) or t.dtype != dtype:
        _refuse(f"{name} must be {list(shape)} {dtype}, got {list(t.shape)} {t.dtype}")
    if t.numel() and (t.stride(-1) != 1 or t.data_ptr() % 16 or any(s % 8 for s in t.stride()[:-1]) or t.stride(-3) > 1 << 23):
        t = t.contiguous()
    return t


def _strides(t: Optional[torch.Tensor], n: int):
    # a dimension of one element may carry any stride: its own does not matter
    return (C.c_int64 * n)(*([0] * n if t is None else [0 if t.shape[i] <= 1 else t.stride(i) for i in range(n)]))


def shared_prefix_attention(q, prefix_k, prefix_v, own_k=None, own_v=None, own_len=None, *, causal=True, scale=None, return_lse=False):
    """Attention of sequences that share a prefix: out[b, i, h] = softmax(scale * q[b, i, h] · k) v over the prefix's keys and sample
    b's own first ``own_len[b]`` keys; with ``causal`` query i sees own keys 0 .. own_len[b] - queries + i (the queries are the
    sequence's newest tokens, their keys among the own ones), otherwise all own_len[b].

    q [batch, queries, heads, dim]; prefix_k, prefix_v [prefix, kv_heads, dim] (or None); own_k, own_v [batch, own_max, kv_heads,
    dim] (or None); own_len int32 [batch] on the device (None: own_max); bfloat16 or float16, dim 64 or 128, heads a multiple of
    kv_heads.  scale None: 1 / sqrt(dim).  -> out [batch, queries, heads, dim], with return_lse also the log-sums float32 [batch,
    heads, queries].  A query that sees no key gives 0 and -inf."""
    device = _on_device(q, "q")
    if q.dim() != 4 or q.dtype not in (torch.bfloat16, torch.float16):
        _refuse(f"q must be [batch, queries, heads, dim] bfloat16 or float16, got {tuple(q.shape)} {q.dtype}")
    if (prefix_k is None) != (prefix_v is None) or (own_k is None) != (own_v is None):
        _refuse("keys and values come together")
    if prefix_k is None and own_k is None:
        _refuse("no keys: give a prefix, own keys or both")
    _same_device(device, prefix_k=prefix_k, prefix_v=prefix_v, own_k=own_k, own_v=own_v, own_len=own_len)
    b, n, h, d = q.shape
    kv = prefix_k if prefix_k is not None else own_k
    if kv.dim() != (3 if prefix_k is not None else 4):
        _refuse("prefix keys must be [prefix, kv_heads, dim], own keys [batch, own_max, kv_heads, dim]")
    hk = kv.shape[-2]
    if prefix_k is not None:
        prefix_k, prefix_v = (_heads(t, m, (prefix_k.shape[0], hk, d), q.dtype) for t, m in ((prefix_k, "prefix_k"), (prefix_v, "prefix_v")))
    if own_k is not None:
        if own_k.dim() != 4:
            _refuse(f"own_k must be [batch, own_max, kv_heads, dim], got {tuple(own_k.shape)}")
        own_k, own_v = (_heads(t, m, (b, own_k.shape[1], hk, d), q.dtype) for t, m in ((own_k, "own_k"), (own_v, "own_v")))
    if own_len is not None:
        if own_k is None or own_len.shape != (b,) or own_len.dtype != torch.int32:
            _refuse(f"own_len must be int32 [{b}] beside own keys, got {tuple(own_len.shape)} {own_len.dtype}")
        own_len = own_len.contiguous()
    if q.numel() and (q.stride(-1) != 1 or q.data_ptr() % 16 or any(s % 8 for s in q.stride()[:-1])):
        q = q.contiguous()
    desc = N.PrefixAttentionDesc(b, n, h, hk, d, 0 if prefix_k is None else prefix_k.shape[0], 0 if own_k is None else own_k.shape[1], int(bool(causal)),
                                 N.CMDI_DT[q.dtype], 1.0 / math.sqrt(d) if scale is None else float(scale), N.ptr(q), N.ptr(prefix_k), N.ptr(prefix_v),
                                 N.ptr(own_k), N.ptr(own_v), _strides(q, 3), _strides(prefix_k, 2), _strides(prefix_v, 2), _strides(own_k, 3),
                                 _strides(own_v, 3), N.ptr(own_len))
    out = torch.empty((b, n, h, d), dtype=q.dtype, device=device)
    lse = torch.empty((b, h, n), dtype=torch.float32, device=device) if return_lse else None
    lib = N.load()
    with _On(device) as stream:
        need = lib.cmdi_prefix_attention_workspace(C.byref(desc))
        if need < 0:
            N.check(int(need))
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        N.check(lib.cmdi_prefix_attention(C.byref(desc), N.ptr(out), N.ptr(lse), N.ptr(work), need, stream))
    return (out, lse) if return_lse else out
