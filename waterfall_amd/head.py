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
import functools

import torch
from torch import nn
from torch.autograd.function import once_differentiable

from . import _lib
from .graph import _on

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


# The calls' host time counts: a backward pass runs on the autograd engine's own thread (with the forward's device and stream
# current), where every Python operation takes several times as long.  Pointers go to the library as plain integers; they and
# the strides are taken from the saved tensors again, which hooks may have moved in between.

def _p(t):
    return None if t is None else t.data_ptr()


def _raw_stream(device):
    return torch._C._cuda_getCurrentRawStream(device.index)


def _rows(t):
    """(t as rows of its last dimension with unit stride inside a row, elements from row to row).  A view where the leading
    dimensions collapse into one, a contiguous copy otherwise."""
    D = t.shape[-1]
    if t.is_contiguous():
        return t, D
    n = t.numel() // D if D else 0
    if t.stride(-1) != 1 and D > 1:
        t = t.contiguous()
    try:
        v = t.view(n, D)
    except RuntimeError:
        v = t.contiguous().view(n, D)
    return v, v.stride(0) if n > 1 else D


@functools.lru_cache(maxsize=256)
def _norm_bytes(N, D, t):
    n = C.c_size_t(0)
    _lib.check(_lib.lib().wf_layer_norm_backward_workspace_bytes(N, D, t, C.byref(n)))
    return n.value


def _wanted(*tensors):
    """Whether a gradient may be asked for: without one the call skips autograd's own work (a third of a short call)."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _norm(x, weight, bias, eps, keep):
    dev, D = x.device, x.shape[-1]
    v, ld = _rows(x)
    N = x.numel() // D
    y = torch.empty(x.shape, dtype=x.dtype, device=dev)
    stats = torch.empty((N, 2), dtype=torch.float32, device=dev) if keep else None
    params = weight if weight is not None else bias
    pdtype = x.dtype if params is None else params.dtype
    with _on(dev):
        _lib.check(_lib.lib().wf_layer_norm(v.data_ptr(), ld, N, D, _TYPES[x.dtype], _p(weight), _p(bias), _TYPES[pdtype], eps,
                                            y.data_ptr(), _p(stats), _raw_stream(dev)))
    return y, v, ld, N, D, pdtype, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, v, ld, N, D, pdtype, stats = _norm(x, weight, bias, eps, True)
        need = ctx.needs_input_grad
        ctx.save_for_backward(v, weight, stats)
        ctx.rest = (x.shape, N, D, pdtype, weight is not None and need[1], bias is not None and need[2])
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        v, weight, stats = ctx.saved_tensors
        shape, N, D, pdtype, want_w, want_b = ctx.rest
        dev, t = v.device, _TYPES[v.dtype]
        v, ld = _rows(v)
        g, ldg = _rows(dy)
        dx = torch.empty(shape, dtype=v.dtype, device=dev)
        dw = torch.empty(D, dtype=pdtype, device=dev) if want_w else None
        db = torch.empty(D, dtype=pdtype, device=dev) if want_b else None
        n = _norm_bytes(N, D, t) if want_w or want_b else 0
        ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
        _lib.check(_lib.lib().wf_layer_norm_backward(g.data_ptr(), ldg, v.data_ptr(), ld, N, D, t, _p(weight), _TYPES[pdtype],
                                                     stats.data_ptr(), dx.data_ptr(), _p(dw), _p(db), _p(ws), n, _raw_stream(dev)))
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
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    if _wanted(x, weight, bias):
        return _LayerNorm.apply(x, weight, bias, float(eps))
    return _norm(x, weight, bias, float(eps), False)[0]


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, seed):
        if isinstance(seed, torch.Tensor):
            ctx.save_for_backward(seed)
            ctx.rest = (p, None)
        else:
            ctx.rest = (p, seed)
        return _drop(x, p, seed)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        p, seed = ctx.rest
        return _drop(dy, p, ctx.saved_tensors[0] if seed is None else seed), None, None


def _drop(x, p, seed):
    if not x.is_contiguous():
        x = x.contiguous()
    y, dev = torch.empty_like(x), x.device
    key, at = (0, seed.data_ptr()) if isinstance(seed, torch.Tensor) else (seed, None)
    with _on(dev):
        _lib.check(_lib.lib().wf_dropout(x.data_ptr(), x.numel(), _TYPES[x.dtype], p, key, at, y.data_ptr(), _raw_stream(dev)))
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
    return _Dropout.apply(x, p, seed) if _wanted(x) else _drop(x, p, seed)


# ---- the projection ---------------------------------------------------------------------------------------------------

_LOG_FWD, _LOG_BWD, _CE_FWD, _CE_BWD = range(4)


@functools.lru_cache(maxsize=256)
def _linear_bytes(what, N, D, V, dtype):
    n = C.c_size_t(0)
    _lib.check(_lib.lib().wf_linear_workspace_bytes(what, N, D, V, _TYPES[dtype], C.byref(n)))
    return n.value


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


def _linear_args(x, weight):
    """x and weight as rows, and the arguments x .. type of the library's calls"""
    v, ldx = _rows(x)
    w, ldw = _rows(weight)
    D = x.shape[-1]
    return v, w, (v.data_ptr(), ldx, x.numel() // D, D, w.data_ptr(), ldw, weight.shape[0], _TYPES[x.dtype])


def _entropy_args(bias, targets, rest):
    """the arguments bias .. smoothing; rest: (ignore_index, smoothing)"""
    return (_p(bias), _TYPES[bias.dtype] if bias is not None else 0, targets.data_ptr(), 1 if targets.dtype == torch.int64 else 0) + rest


def _log_softmax(x, weight, bias):
    dev = x.device
    v, w, a = _linear_args(x, weight)
    V = a[6]
    bt = _TYPES[bias.dtype] if bias is not None else 0
    lp = torch.empty(x.shape[:-1] + (V,), dtype=torch.float32, device=dev)
    n = _linear_bytes(_LOG_FWD, a[2], a[3], V, x.dtype)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    with _on(dev):
        _lib.check(_lib.lib().wf_linear_log_softmax(*a, _p(bias), bt, lp.data_ptr(), ws.data_ptr(), n, _raw_stream(dev)))
    return lp, v, w, a, bt


class _LinearLogSoftmax(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        lp, v, w, a, bt = _log_softmax(x, weight, bias)
        ctx.save_for_backward(v, w, bias, lp)
        ctx.shapes = (x.shape, weight.shape)
        return lp

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        v, w, bias, lp = ctx.saved_tensors
        xshape, wshape = ctx.shapes
        v, w, a = _linear_args(v, w)
        bt = _TYPES[bias.dtype] if bias is not None else 0
        dev, need = v.device, ctx.needs_input_grad
        g, ldg = _rows(grad)
        dx = torch.empty(xshape, dtype=v.dtype, device=dev) if need[0] else None
        dw = torch.empty(wshape, dtype=v.dtype, device=dev) if need[1] else None
        db = torch.empty(wshape[:1], dtype=bias.dtype, device=dev) if need[2] else None
        n = _linear_bytes(_LOG_BWD, a[2], a[3], a[6], v.dtype)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.check(_lib.lib().wf_linear_log_softmax_backward(lp.data_ptr(), g.data_ptr(), ldg, *a, bt, _p(dx), _p(dw), _p(db),
                                                             ws.data_ptr(), n, _raw_stream(dev)))
        return dx, dw, db


def linear_log_softmax(x, weight, bias=None):
    """log_softmax(x weight^T + bias) as float32 [..., V]: the log-probabilities that ``DenseFsaVec`` takes.

    x [..., D], weight [V, D]: float32, bfloat16 or float16, both of one type; bias [V] or None, any of the three.  float32 is
    computed to float32's accuracy (no reduced-precision product).  A bias of -inf masks an output; a row whose every output
    is masked is all -inf and has no gradient.  In the backward pass rows whose incoming gradient is all zero (frames behind an
    utterance's end) are left out whatever they hold; 16-bit types round the gradient of a logit to x's type before it enters
    the products."""
    _check_linear("linear_log_softmax", x, weight, bias)
    bias = None if bias is None else bias.contiguous()
    return _LinearLogSoftmax.apply(x, weight, bias) if _wanted(x, weight, bias) else _log_softmax(x, weight, bias)[0]


def _entropy(x, weight, targets, bias, ignore_index, smoothing, reduction):
    dev = x.device
    v, w, a = _linear_args(x, weight)
    N = a[2]
    rest = (ignore_index, smoothing)
    rows, mean = 1 if reduction == "none" else 0, 1 if reduction == "mean" else 0
    loss = torch.empty(x.shape[:-1], dtype=torch.float32, device=dev)
    lse = torch.empty(N, dtype=torch.float32, device=dev)
    total = None if rows else torch.empty((), dtype=torch.float32, device=dev)
    n = _linear_bytes(_CE_FWD, N, a[3], a[6], x.dtype)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    with _on(dev):
        _lib.check(_lib.lib().wf_linear_cross_entropy(*a, *_entropy_args(bias, targets, rest), loss.data_ptr(), lse.data_ptr(),
                                                      _p(total), mean, ws.data_ptr(), n, _raw_stream(dev)))
    return loss if rows else total, v, w, rest, rows, mean, lse


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, targets, bias, ignore_index, smoothing, reduction):
        loss, v, w, rest, rows, mean, lse = _entropy(x, weight, targets, bias, ignore_index, smoothing, reduction)
        ctx.save_for_backward(v, w, targets, bias, lse)
        ctx.rest = (x.shape, weight.shape, rest, rows, mean)
        return loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        v, w, targets, bias, lse = ctx.saved_tensors
        xshape, wshape, rest, rows, mean = ctx.rest
        v, w, a = _linear_args(v, w)
        dev, need = v.device, ctx.needs_input_grad
        if not grad.is_contiguous():
            grad = grad.contiguous()
        dx = torch.empty(xshape, dtype=v.dtype, device=dev) if need[0] else None
        dw = torch.empty(wshape, dtype=v.dtype, device=dev) if need[1] else None
        db = torch.empty(wshape[:1], dtype=bias.dtype, device=dev) if need[3] else None
        n = _linear_bytes(_CE_BWD, a[2], a[3], a[6], v.dtype)
        ws = torch.empty(n, dtype=torch.uint8, device=dev)
        _lib.check(_lib.lib().wf_linear_cross_entropy_backward(grad.data_ptr(), rows, mean, lse.data_ptr(), *a,
                                                               *_entropy_args(bias, targets, rest), _p(dx), _p(dw), _p(db),
                                                               ws.data_ptr(), n, _raw_stream(dev)))
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
    args = (x, weight, targets.contiguous(), None if bias is None else bias.contiguous(), int(ignore_index), float(label_smoothing),
            reduction)
    return _LinearCrossEntropy.apply(*args) if _wanted(x, weight, bias) else _entropy(*args)[0]


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
