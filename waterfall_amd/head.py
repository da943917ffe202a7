"""The output head: what stands between an encoder and the losses.  The reference's models end in normalisation -> Linear ->
log_softmax and hand ``log_probs [B, T, V]`` to the loss (``rnnp.py:116-122``); here every step of it, and the softmax cross
entropy on the same projection, is a kernel of the library with its own gradient.

    y  = layer_norm(x, weight, bias)              rows of the last dimension
    y  = dropout(x, p, seed)                      counter-based: the mask is never stored
    lp = linear_log_softmax(x, weight, bias)      fp32 log-probabilities, what DenseFsaVec takes
    ce = linear_cross_entropy(x, weight, targets, bias)   the logits are never kept

``OutputHead`` is the module over them.  All run on the current stream of the tensors' device and can be captured in a graph.
"""
import ctypes as C

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .graph import _on, _ptr, _stream

__all__ = ["layer_norm", "dropout"]

_TYPES = {torch.float32: _lib.WF_F32, torch.bfloat16: _lib.WF_BF16, torch.float16: _lib.WF_F16}


def _check(t, name, like=None, dtype=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")
    if t.dtype not in _TYPES:
        raise TypeError(f"{name} must be float32, bfloat16 or float16, got {t.dtype}")
    if t.device.type != "cuda":
        raise _lib.WfError(f"{name} must live on the GPU: waterfall_amd has no CPU path")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, x is on {like.device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} is {t.dtype}, expected {dtype}")
    return t


def _rows(t):
    """(t as rows of its last dimension with unit stride inside a row, elements from row to row).  A view where the leading
    dimensions collapse into one, a contiguous copy otherwise."""
    D = t.shape[-1]
    n = t.numel() // D if D else 0
    if t.stride(-1) != 1 and D > 1:
        t = t.contiguous()
    try:
        v = t.view(n, D)
    except RuntimeError:
        v = t.contiguous().view(n, D)
    return v, v.stride(0) if n > 1 else D


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        lib, dev = _lib.lib(), x.device
        v, ld = _rows(x)
        N, D = v.shape
        y = torch.empty(x.shape, dtype=x.dtype, device=dev)
        keep = any(ctx.needs_input_grad)
        stats = torch.empty((N, 2), dtype=torch.float32, device=dev) if keep else None
        params = weight if weight is not None else bias
        ptype = _TYPES[params.dtype if params is not None else x.dtype]
        with _on(dev):
            _lib.check(lib.wf_layer_norm(_ptr(v), ld, N, D, _TYPES[x.dtype], _ptr(weight), _ptr(bias), ptype, eps, _ptr(y),
                                         _ptr(stats), _stream(dev)))
        if keep:
            ctx.save_for_backward(x, weight, stats)
            ctx.ptype, ctx.bias = ptype, bias is not None
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, stats = ctx.saved_tensors
        lib, dev = _lib.lib(), x.device
        v, ld = _rows(x)
        g, ldg = _rows(dy)
        N, D = v.shape
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev)
        pt = next(k for k, n in _TYPES.items() if n == ctx.ptype)
        dw = torch.empty(D, dtype=pt, device=dev) if weight is not None and ctx.needs_input_grad[1] else None
        db = torch.empty(D, dtype=pt, device=dev) if ctx.bias and ctx.needs_input_grad[2] else None
        ws, n = None, C.c_size_t(0)
        if dw is not None or db is not None:
            _lib.check(lib.wf_layer_norm_backward_workspace_bytes(N, D, _TYPES[x.dtype], C.byref(n)))
            ws = torch.empty(n.value, dtype=torch.uint8, device=dev)
        with _on(dev):
            _lib.check(lib.wf_layer_norm_backward(_ptr(g), ldg, _ptr(v), ld, N, D, _TYPES[x.dtype], _ptr(weight), ctx.ptype,
                                                  _ptr(stats), _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n.value, _stream(dev)))
        return dx, dw, db, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of ``x`` (at most 32768 elements).

    x: float32, bfloat16 or float16, any leading dimensions.  weight, bias: [D] or None, both of one of these types (fp32
    weights beside bfloat16 activations are fine).  The result is contiguous and of x's type; statistics are fp32."""
    _check(x, "x")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("layer_norm: x needs a last dimension of at least one element")
    if x.shape[-1] > 32768:
        raise ValueError(f"layer_norm: rows of {x.shape[-1]} elements (at most 32768)")
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None:
            _check(t, name, like=x)
            if t.shape != x.shape[-1:]:
                raise ValueError(f"layer_norm: {name} has shape {tuple(t.shape)}, expected {tuple(x.shape[-1:])}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"layer_norm: weight is {weight.dtype}, bias is {bias.dtype}")
    return _LayerNorm.apply(x, None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous(),
                            float(eps))


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed):
        ctx.p = p
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
            ctx.seed = None
        else:
            ctx.seed = seed
        return _drop(x, p, seed)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        return _drop(dy, ctx.p, ctx.saved_tensors[0] if ctx.seed is None else ctx.seed), None, None


def _drop(x, p, seed):
    x = x.contiguous()
    y = torch.empty_like(x)
    key, at = (0, seed) if isinstance(seed, torch.Tensor) else (seed, None)
    with _on(x.device):
        _lib.check(_lib.lib().wf_dropout(_ptr(x), x.numel(), _TYPES[x.dtype], p, key, _ptr(at), _ptr(y), _stream(x.device)))
    return y


def dropout(x, p, seed):
    """x / (1 - p) where element i (row-major) is kept, 0 elsewhere; the mask is a function of (seed, i) alone (Philox4x32-7,
    word i % 4 of counter i / 4, kept iff word >= floor(p 2^32)), so backward needs no stored mask and equal seeds give equal
    masks whatever the type or the strides.

    seed: an integer (64 bits are used), or a one-element int64 tensor on x's device that is read when the kernel runs: a
    captured graph takes a new mask on a replay that finds a new seed there.  That tensor must not change between forward and
    backward.  Call it in training only: there is no evaluation mode."""
    _check(x, "x")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p must be in [0, 1], got {p}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise TypeError("dropout: seed must be an integer or an int64 tensor of one element")
        if seed.device != x.device:
            raise ValueError(f"dropout: seed is on {seed.device}, x is on {x.device}")
    else:
        seed = int(seed) & 0xFFFFFFFFFFFFFFFF
    return _Dropout.apply(x, p, seed)
