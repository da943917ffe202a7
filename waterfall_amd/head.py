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

__all__ = ["layer_norm", "dropout", "linear_log_softmax", "linear_cross_entropy", "OutputHead"]

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


# ---- the projection ---------------------------------------------------------------------------------------------------

_LOG_FWD, _LOG_BWD, _CE_FWD, _CE_BWD = range(4)


def _linear_ws(what, N, D, V, x):
    n = C.c_size_t(0)
    _lib.check(_lib.lib().wf_linear_workspace_bytes(what, N, D, V, _TYPES[x.dtype], C.byref(n)))
    return torch.empty(n.value, dtype=torch.uint8, device=x.device), n.value


def _check_linear(who, x, weight, bias):
    _check(x, "x")
    _check(weight, "weight", like=x, dtype=x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"{who}: x needs a last dimension of at least one element")
    if weight.dim() != 2 or weight.shape[1] != x.shape[-1] or weight.shape[0] < 1:
        raise ValueError(f"{who}: weight has shape {tuple(weight.shape)}, expected [V, {x.shape[-1]}]")
    if bias is not None:
        _check(bias, "bias", like=x)
        if bias.shape != weight.shape[:1]:
            raise ValueError(f"{who}: bias has shape {tuple(bias.shape)}, expected [{weight.shape[0]}]")


def _linear_args(x, weight, bias):
    """(what keeps the tensors alive, the arguments x .. type)"""
    v, ldx = _rows(x)
    w, ldw = _rows(weight)
    N, D = v.shape
    return (v, w), (_ptr(v), ldx, N, D, _ptr(w), ldw, w.shape[0], _TYPES[x.dtype])


class _LinearLogSoftmax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        dev = x.device
        keep, a = _linear_args(x, weight, bias)
        N, D, V = a[2], a[3], a[6]
        bt = _TYPES[bias.dtype] if bias is not None else 0
        lp = torch.empty(x.shape[:-1] + (V,), dtype=torch.float32, device=dev)
        with _on(dev):
            ws, n = _linear_ws(_LOG_FWD, N, D, V, x)
            _lib.check(_lib.lib().wf_linear_log_softmax(*a, _ptr(bias), bt, _ptr(lp), _ptr(ws), n, _stream(dev)))
        ctx.save_for_backward(x, weight, bias, lp)
        return lp

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, bias, lp = ctx.saved_tensors
        dev = x.device
        keep, a = _linear_args(x, weight, bias)
        N, D, V = a[2], a[3], a[6]
        g, ldg = _rows(grad)
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty(weight.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[1] else None
        db = torch.empty(V, dtype=bias.dtype, device=dev) if ctx.needs_input_grad[2] else None
        with _on(dev):
            ws, n = _linear_ws(_LOG_BWD, N, D, V, x)
            _lib.check(_lib.lib().wf_linear_log_softmax_backward(
                _ptr(lp), _ptr(g), ldg, *a, _TYPES[bias.dtype] if bias is not None else 0, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n,
                _stream(dev)))
        return dx, dw, db


def linear_log_softmax(x, weight, bias=None):
    """log_softmax(x weight^T + bias) as float32 [..., V]: the log-probabilities that ``DenseFsaVec`` takes.

    x [..., D], weight [V, D]: float32, bfloat16 or float16, both of one type; bias [V] or None, any of the three.  float32 is
    computed to float32's accuracy (no reduced-precision product).  A bias of -inf masks an output; a row whose every output
    is masked is all -inf and has no gradient.  In the backward pass rows whose incoming gradient is all zero (frames behind an
    utterance's end) are left out whatever they hold; 16-bit types round the gradient of a logit to x's type before it enters
    the products."""
    _check_linear("linear_log_softmax", x, weight, bias)
    return _LinearLogSoftmax.apply(x, weight, None if bias is None else bias.contiguous())


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, bias, ignore_index, smoothing, reduction):
        dev = x.device
        keep, a = _linear_args(x, weight, bias)
        N, D, V = a[2], a[3], a[6]
        ctx.rest = (_TYPES[bias.dtype] if bias is not None else 0, 1 if targets.dtype == torch.int64 else 0, ignore_index, smoothing)
        ctx.reduction = reduction
        bt, wide = ctx.rest[:2]
        loss = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
        lse = torch.empty(N, dtype=torch.float32, device=dev)
        total = torch.empty((), dtype=torch.float32, device=dev) if reduction != "none" else None
        with _on(dev):
            ws, n = _linear_ws(_CE_FWD, N, D, V, x)
            _lib.check(_lib.lib().wf_linear_cross_entropy(*a, _ptr(bias), bt, _ptr(targets), wide, ignore_index, smoothing, _ptr(loss),
                                                          _ptr(lse), _ptr(total), 1 if reduction == "mean" else 0, _ptr(ws), n,
                                                          _stream(dev)))
        ctx.save_for_backward(x, weight, targets, bias, lse)
        return loss if total is None else total

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, weight, targets, bias, lse = ctx.saved_tensors
        dev = x.device
        keep, a = _linear_args(x, weight, bias)
        N, D, V = a[2], a[3], a[6]
        bt, wide, ignore_index, smoothing = ctx.rest
        g = grad.contiguous()
        dx = torch.empty(x.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[0] else None
        dw = torch.empty(weight.shape, dtype=x.dtype, device=dev) if ctx.needs_input_grad[1] else None
        db = torch.empty(V, dtype=bias.dtype, device=dev) if ctx.needs_input_grad[3] else None
        with _on(dev):
            ws, n = _linear_ws(_CE_BWD, N, D, V, x)
            _lib.check(_lib.lib().wf_linear_cross_entropy_backward(
                _ptr(g), 1 if ctx.reduction == "none" else 0, 1 if ctx.reduction == "mean" else 0, _ptr(lse), *a, _ptr(bias), bt,
                _ptr(targets), wide, ignore_index, smoothing, _ptr(dx), _ptr(dw), _ptr(db), _ptr(ws), n, _stream(dev)))
        return dx, dw, None, db, None, None, None


def linear_cross_entropy(x, weight, targets, bias=None, ignore_index=-1, label_smoothing=0.0, reduction="mean"):
    """Softmax cross entropy of x weight^T + bias against ``targets``, without keeping the logits: forward leaves one number per
    row, backward computes the logits again piece by piece.

    x [..., D], weight [V, D], bias as for ``linear_log_softmax``; targets [...]: int32 or int64.  Rows whose target is
    ``ignore_index`` (by default -1, the label of the arcs that take no frame) have no loss, no gradient and may hold anything.
    A target that is neither it nor an output makes its row's loss NaN (nothing is read out of range) and has no gradient.

    reduction: 'none' (float32 [...]), 'sum', or 'mean' over the rows that take part (0 where there are none)."""
    _check_linear("linear_cross_entropy", x, weight, bias)
    if not isinstance(targets, torch.Tensor) or targets.dtype not in (torch.int32, torch.int64):
        raise TypeError("linear_cross_entropy: targets must be an int32 or int64 tensor")
    if targets.device != x.device:
        raise ValueError(f"linear_cross_entropy: targets are on {targets.device}, x is on {x.device}")
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets have shape {tuple(targets.shape)}, expected {tuple(x.shape[:-1])}")
    if not 0.0 <= float(label_smoothing) <= 1.0:
        raise ValueError(f"linear_cross_entropy: label_smoothing must be in [0, 1], got {label_smoothing}")
    if reduction not in ("none", "sum", "mean"):
        raise ValueError(f"linear_cross_entropy: unknown reduction {reduction!r}")
    return _LinearCrossEntropy.apply(x, weight, targets.contiguous(), None if bias is None else bias.contiguous(), int(ignore_index),
                                     float(label_smoothing), reduction)


class OutputHead(nn.Module):
    """Encoder output [..., D] -> log-probabilities [..., V] for ``DenseFsaVec`` / ``graphloss``: layer norm, dropout (in
    training), projection with log-softmax (the tail of the reference's models, ``rnnp.py:116-122``).

        head = wf.OutputHead(encoder_dim, lang.num_nn_output, dropout=0.1)
        loss = wf.graphloss(decoding_graph=graphs, dense_fsa_vec=wf.DenseFsaVec(head(enc), segments), ...)
        loss = loss + 0.1 * head.cross_entropy(enc, frame_targets)         # on the same projection

    Parameters may be float32 beside 16-bit activations: the projection's are cast to the activations' type.  Dropout takes
    its seed from torch's generator of the device (``torch.manual_seed``), on the device: it can be captured in a graph."""

    def __init__(self, idim, num_outputs, dropout=0.0, norm=True, bias=True, eps=1e-5, device=None, dtype=None):
        super().__init__()
        if not 0.0 <= dropout <= 1.0:
            raise ValueError(f"OutputHead: dropout must be in [0, 1], got {dropout}")
        kw = dict(device=device, dtype=dtype)
        self.dropout, self.eps = float(dropout), float(eps)
        self.norm_weight = nn.Parameter(torch.ones(idim, **kw)) if norm else None
        self.norm_bias = nn.Parameter(torch.zeros(idim, **kw)) if norm else None
        self.weight = nn.Parameter(torch.empty(num_outputs, idim, **kw))
        self.bias = nn.Parameter(torch.zeros(num_outputs, **kw)) if bias else None
        nn.init.normal_(self.weight, std=idim ** -0.5)

    def features(self, x):
        if self.norm_weight is not None:
            x = layer_norm(x, self.norm_weight, self.norm_bias, self.eps)
        if self.training and self.dropout > 0.0:
            seed = torch.empty(1, dtype=torch.int64, device=x.device).random_()
            x = dropout(x, self.dropout, seed)
        return x

    def forward(self, x):
        x = self.features(x)
        return linear_log_softmax(x, self.weight.to(x.dtype), self.bias)

    def cross_entropy(self, x, targets, ignore_index=-1, label_smoothing=0.0, reduction="mean"):
        x = self.features(x)
        return linear_cross_entropy(x, self.weight.to(x.dtype), targets, self.bias, ignore_index, label_smoothing, reduction)
