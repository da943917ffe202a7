"""The output head: what stands between an encoder and the losses.  The reference's models end in normalisation -> Linear ->
log_softmax and hand ``log_probs [B, T, V]`` to the loss (``rnnp.py:116-122``); here every step of it, and the softmax cross
entropy on the same projection, is a kernel of the library with its own gradient.

    y  = layer_norm(x, weight, bias)              rows of the last dimension
    y  = dropout(x, p, seed)                      counter-based: the mask is never stored
    lp = linear_log_softmax(x, weight, bias)      fp32 log-probabilities, what DenseFsaVec takes
    ce = linear_cross_entropy(x, weight, targets, bias)   the logits are never kept

``OutputHead`` is the module over them.  All run on the current stream of the tensors' device and can be captured in a graph; a
backward pass only while no eager graph of the same leaves is alive (a loss that was kept, say): it raises, since torch's engine would
draw that graph's stream into the capture.
"""
import torch
from torch import nn

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


# The autograd nodes are C++ (csrc/wf_head_torch.cpp over the C entry points): short calls are bound by the host.

_ext = None


def _nodes():
    global _ext
    if _ext is None:
        _lib.lib()
        try:
            from . import _head
        except ImportError as e:
            raise _lib.WfError(f"waterfall_amd/_head.so cannot be loaded ({e}): build it first "
                               "(python -c 'import __graft_entry__ as g; g.build()').") from None
        _ext = _head
    return _ext


def _run(name, x, *args):
    """One of the nodes on x's device and its current stream."""
    dev = x.device
    with _on(dev):
        try:
            return getattr(_ext or _nodes(), name)(*args, torch._C._cuda_getCurrentRawStream(dev.index))
        except RuntimeError as e:
            if str(e).startswith("libwfdwfst error"):
                raise _lib.WfError(str(e).split("\n")[0]) from None
            raise


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension of ``x`` (at most 32768 elements).

    x: float32, bfloat16 or float16, any leading dimensions.  weight, bias: [D] or None, both of one of these types (fp32
    weights beside bfloat16 activations are fine).  The result is contiguous and of x's type; statistics are fp32.  In the
    backward pass rows whose incoming gradient is all zero take no part, whatever they hold."""
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
    return _run("layer_norm", x, x, None if weight is None else weight.contiguous(), None if bias is None else bias.contiguous(),
                float(eps))


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
        return _run("dropout", x, x, p, 0, seed)
    return _run("dropout", x, x, p, int(seed) & 0xFFFFFFFFFFFFFFFF, None)


# ---- the projection ---------------------------------------------------------------------------------------------------

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


def linear_log_softmax(x, weight, bias=None):
    """log_softmax(x weight^T + bias) as float32 [..., V]: the log-probabilities that ``DenseFsaVec`` takes.

    x [..., D], weight [V, D]: float32, bfloat16 or float16, both of one type; bias [V] or None, any of the three.  float32
    products are off by less than 2^-21 of themselves, 2^-24.5 on average (about one rounding of float32).  A bias of -inf masks
    an output; a row whose every output is masked is all -inf and has no gradient.  In the backward pass rows whose incoming
    gradient is all zero (frames behind an utterance's end) are left out whatever they hold; 16-bit types round the gradient of a logit to x's type before it enters
    the products (float16: scaled to the upper end of the type's range, bits are lost below 2^-26 of the largest)."""
    _check_linear("linear_log_softmax", x, weight, bias)
    return _run("linear_log_softmax", x, x, weight, None if bias is None else bias.contiguous())


_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(x, weight, targets, bias=None, ignore_index=-1, label_smoothing=0.0, reduction="mean"):
    """Softmax cross entropy of x weight^T + bias against ``targets``, without keeping the logits: forward leaves one number per
    row, backward computes the logits again piece by piece.

    x [..., D], weight [V, D], bias as for ``linear_log_softmax``; targets [...]: int32 or int64.  Rows whose target is
    ``ignore_index`` (by default -1, the label of the arcs that take no frame) have no loss, no gradient and may hold anything.
    A target that is neither it nor an output makes its row's loss NaN (nothing is read out of range) and has no gradient.
    ``label_smoothing`` spreads its share over all outputs, those masked by a bias of -inf too: the loss is then infinite.

    reduction: 'none' (float32 [...]; rows whose incoming gradient is zero are left out of the backward pass whatever they
    hold), 'sum', or 'mean' over the rows that take part (0 where there are none)."""
    _check_linear("linear_cross_entropy", x, weight, bias)
    if not isinstance(targets, torch.Tensor) or targets.dtype not in (torch.int32, torch.int64):
        raise TypeError("linear_cross_entropy: targets must be an int32 or int64 tensor")
    if targets.device != x.device:
        raise ValueError(f"linear_cross_entropy: targets are on {targets.device}, x is on {x.device}")
    if targets.shape != x.shape[:-1]:
        raise ValueError(f"linear_cross_entropy: targets have shape {tuple(targets.shape)}, expected {tuple(x.shape[:-1])}")
    if not 0.0 <= float(label_smoothing) <= 1.0:
        raise ValueError(f"linear_cross_entropy: label_smoothing must be in [0, 1], got {label_smoothing}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"linear_cross_entropy: unknown reduction {reduction!r}")
    return _run("linear_cross_entropy", x, x, weight, targets.contiguous(), None if bias is None else bias.contiguous(),
                int(ignore_index), float(label_smoothing), _REDUCTIONS[reduction])


class OutputHead(nn.Module):
    """Encoder output [..., D] -> log-probabilities [..., V] for ``DenseFsaVec`` / ``graphloss``: layer norm, dropout (in
    training), projection with log-softmax (the tail of the reference's models, ``rnnp.py:116-122``).

        head = wf.OutputHead(encoder_dim, lang.num_nn_output, dropout=0.1)
        loss = wf.graphloss(decoding_graph=graphs, dense_fsa_vec=wf.DenseFsaVec(head(enc), segments), ...)

    ``cross_entropy`` takes the same path to a loss of its own.  Each of the two calls norms and draws a dropout mask; both losses
    of one step share them like this:

        x, w = head.features(enc), head.weight.to(enc.dtype)
        loss = wf.graphloss(dense_fsa_vec=wf.DenseFsaVec(wf.linear_log_softmax(x, w, head.bias), segments), ...)
        loss = loss + 0.1 * wf.linear_cross_entropy(x, w, frame_targets, head.bias)

    Parameters may be float32 beside 16-bit activations: the projection's weight is cast to the activations' type (and its
    gradient comes back in it).  Frames without a target, or whose incoming gradient is zero, may hold anything.  Dropout takes
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
