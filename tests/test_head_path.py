"""OutputHead: layer norm, dropout and projection together in front of the losses that are there, and the calls around them that
a training program makes: saved tensors moved by hooks, two calls at once, a captured step, mixed precision.

Gradients of the whole head are compared as vectors: |error| <= r |want| in the 2-norm.  fp32: every entry comes out of a chain
of at most about 1000 roundings of 2^-24 (row statistics of 96 features, products over 96 features or 59 outputs in six
parts, sums over 120 rows), which cancellation may raise by a factor of 4: r = 2^-12.  bfloat16: five roundings of 2^-8 on the way
(norm, dropout, gradient of a logit, gradient of the features twice), which add up: r = 5 * 2^-8 and the same 2^-12."""
import numpy as np
import pytest
import torch

import waterfall_amd as wf
from tests import util

DEV = "cuda:0"
pytestmark = pytest.mark.gpu


def near(got, want, r, what):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), what
    assert (got - want).norm() <= r * want.norm(), (what, ((got - want).norm() / want.norm()).item())


def plain(head, x, mask, dtype):
    """the head in 64 bits on its own parameters; rounds to `dtype` nowhere"""
    p = {k: v.detach().double().requires_grad_() for k, v in head.named_parameters()}
    x = x.detach().double().requires_grad_()
    mu = x.mean(-1, keepdim=True)
    h = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + head.eps) * p["norm_weight"] + p["norm_bias"]
    z = (h * mask) @ p["weight"].t() + p["bias"]
    return torch.log_softmax(z, -1), x, p


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_training_step_of_graph_loss_and_cross_entropy(dtype):
    c = util.random_case(77, "ctc", B=4, T=30, L=5, P=58)
    B, T, V = c["lp"].shape
    torch.manual_seed(3)
    head = wf.OutputHead(96, V, dropout=0.2, device=DEV)                   # fp32 parameters
    with torch.no_grad():
        for q in (head.norm_weight, head.norm_bias, head.bias):
            q.add_(0.1 * torch.randn_like(q))
        if dtype == torch.bfloat16:
            head.weight.copy_(head.weight.bfloat16())
    enc = torch.randn(B, T, 96, device=DEV).to(dtype)
    x = enc.clone().requires_grad_()
    segs = torch.from_numpy(c["segs"])
    frames = torch.arange(T, device=DEV)[None, :] < segs[:, 2].to(DEV)[:, None]
    torch.manual_seed(11)
    feats = head.features(x)                                               # one dropout mask for both losses
    w = head.weight.to(x.dtype)
    lp = wf.linear_log_softmax(feats, w, head.bias)
    assert lp.dtype == torch.float32
    gl = wf.graphloss(c["fsa"], wf.DenseFsaVec(lp, segs), reduction="sum")
    best = wf.best_path(c["fsa"], wf.DenseFsaVec(lp.detach(), segs))
    targets = torch.full((B, T), -1, dtype=torch.int32, device=DEV)
    for i in range(B):
        targets[i, :int(segs[i, 2])] = torch.tensor(best["labels"][i], dtype=torch.int32, device=DEV)
    assert (targets[frames] >= 0).all()
    ce = wf.linear_cross_entropy(feats, w, targets, head.bias, label_smoothing=0.1, reduction="sum")
    (gl + 0.3 * ce).backward()
    # the same in 64 bits, the graph loss by its gradient with respect to these log-probabilities
    torch.manual_seed(11)
    seed = torch.empty(1, dtype=torch.int64, device=DEV).random_()
    mask = wf.dropout(torch.ones(B, T, 96, device=DEV), 0.2, seed).double()
    ref, rx, rp = plain(head, enc, mask, dtype)
    r = 2.0 ** -12 + (5 * 2.0 ** -8 if dtype == torch.bfloat16 else 0)
    near(lp.detach()[frames], ref.detach()[frames], r, "log_probs")
    leaf = lp.detach().clone().requires_grad_()
    wf.graphloss(c["fsa"], wf.DenseFsaVec(leaf, segs), reduction="sum").backward()
    t = targets.long().clamp(min=0)
    want_ce = (-(0.9 * ref.gather(-1, t[..., None])[..., 0] + 0.1 * ref.mean(-1)) * frames).sum()
    near(ce.detach(), want_ce.detach(), r, "cross entropy")
    ((ref * leaf.grad.double()).sum() + 0.3 * want_ce).backward()
    near(x.grad, rx.grad, r, "dx")
    for k, v in head.named_parameters():
        near(v.grad, rp[k].grad, r, k)
    assert not x.grad[~frames].any()


def test_evaluation_and_the_methods_of_the_module():
    torch.manual_seed(0)
    head = wf.OutputHead(40, 70, dropout=0.5, device=DEV)
    x = torch.randn(3, 5, 40, device=DEV)
    t = torch.randint(0, 70, (3, 5), device=DEV)
    head.eval()
    lp, ref = head(x), plain(head, x, 1.0, torch.float32)[0]
    near(lp.detach(), ref.detach(), 2.0 ** -12, "eval")
    with torch.no_grad():
        assert torch.equal(head(x), lp) and torch.equal(head.cross_entropy(x, t), head.cross_entropy(x, t))
    near(head.cross_entropy(x, t).detach(), torch.nn.functional.nll_loss(ref.reshape(-1, 70), t.reshape(-1)).detach(), 2.0 ** -12, "ce")
    head.train()
    torch.manual_seed(5)
    a = head(x)
    torch.manual_seed(5)
    assert torch.equal(head(x), a) and not torch.equal(head(x), a)         # the generator's seed, another mask per call
    bare = wf.OutputHead(40, 70, norm=False, bias=False, device=DEV)
    assert sorted(k for k, _ in bare.named_parameters()) == ["weight"]
    bare(x).sum().backward()
    assert bare.weight.grad.shape == (70, 40)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensors_that_hooks_moved(dtype):
    """save_on_cpu hands backward copies at other addresses and with other strides."""
    wide = torch.randn(6, 7, 200, device=DEV).to(dtype)
    args = [wide[..., 5:133], torch.randn(128, device=DEV), torch.randn(128, device=DEV)]
    w, b = (torch.randn(90, 300, device=DEV) * 0.1).to(dtype)[:, 100:228], torch.randn(90, device=DEV)
    t = torch.randint(-1, 90, (6, 7), device=DEV)

    def step():
        a = [v.detach().requires_grad_() for v in args + [w, b]]
        y = wf.dropout(wf.layer_norm(*a[:3]), 0.25, torch.tensor([9], device=DEV))
        x = torch.cat([y, y], -1)[..., 64:192]                             # rows with a stride of their own
        loss = wf.linear_log_softmax(x, *a[3:]).square().sum() + wf.linear_cross_entropy(x, a[3], t, a[4])
        return loss, a

    loss, a = step()
    want = torch.autograd.grad(loss, a)
    with torch.autograd.graph.save_on_cpu():
        loss, a = step()
    junk = [torch.full((6, 7, 256), float("nan"), device=DEV, dtype=dtype) for _ in range(20)]     # what was freed is used again
    got = torch.autograd.grad(loss, a)
    del junk
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def test_saved_tensors_that_come_back_as_something_else():
    """Hooks that hand back other devices, types or sizes: an error on the host, nothing is launched."""
    x, w = torch.randn(4, 64, device=DEV, requires_grad=True), torch.randn(50, 64, device=DEV, requires_grad=True)
    t, one = torch.randint(0, 50, (4,), device=DEV), torch.ones(64, device=DEV)
    for wrong in (lambda v: v.cpu(), lambda v: v.double() if v.is_floating_point() else v.short(), lambda v: v.reshape(-1)[:-1] if v.numel() > 1 else v.short()):
        for f in (lambda: wf.layer_norm(x, one, one), lambda: wf.linear_log_softmax(x, w), lambda: wf.linear_cross_entropy(x, w, t),
                  lambda: wf.dropout(x, 0.5, torch.tensor([3], device=DEV))):
            with torch.autograd.graph.saved_tensors_hooks(lambda v: v, wrong):
                y = f()
                with pytest.raises(RuntimeError, match="came back"):
                    y.sum().backward()
    # other strides are fine
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: torch.stack((v, v), -1)[..., 0]):
        got = torch.autograd.grad(wf.linear_cross_entropy(wf.layer_norm(x, one, one), w, t), (x, w))
    want = torch.autograd.grad(wf.linear_cross_entropy(wf.layer_norm(x, one, one), w, t), (x, w))
    for p, q in zip(got, want):
        assert torch.equal(p, q)


def test_what_autograd_has_to_notice():
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    w = torch.randn(50, 64, device=DEV, requires_grad=True)
    t = torch.randint(0, 50, (4,), device=DEV)
    y = x * 1.0
    loss = wf.linear_cross_entropy(y, w, t)
    with torch.no_grad():
        y.zero_()                                                          # the saved features change
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()
    lp = wf.linear_log_softmax(x, w)
    g, = torch.autograd.grad(lp.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()                                                 # no second derivative: said, not made up


def test_two_calls_at_once_share_nothing():
    torch.manual_seed(1)
    cases = []
    for k in range(2):
        x = torch.randn(700, 192, device=DEV).bfloat16()
        w = (torch.randn(1500 + 333 * k, 192, device=DEV) * 0.1).bfloat16()
        cases.append((x, w, torch.randint(0, 1500, (700,), device=DEV)))

    def step(x, w, t):
        a = [x.clone().requires_grad_(), w.clone().requires_grad_()]
        h = wf.dropout(wf.layer_norm(a[0]), 0.1, 7)
        loss = wf.linear_cross_entropy(h, a[1], t)
        return [loss.detach(), *torch.autograd.grad(loss, a)]

    want = [step(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [None, None]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k] = step(*cases[k])
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        for p, q in zip(a, b):
            assert torch.equal(p, q)


def test_a_captured_step_of_the_module():
    torch.manual_seed(2)
    head = wf.OutputHead(64, 200, dropout=0.3, device=DEV)
    x = torch.randn(5, 40, 64, device=DEV)
    t = torch.randint(-1, 200, (5, 40), device=DEV)
    params = list(head.parameters())

    def step():
        loss = head.cross_entropy(x, t, label_smoothing=0.1)
        return [loss.detach(), *torch.autograd.grad(loss, params)]

    def capture():
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        return graph, out

    graph, out = capture()
    seen = []
    for _ in range(3):                                                     # every replay draws another mask
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.isfinite(v).all() for v in out)
        seen.append(out[0].item())
    assert len(set(seen)) == 3
    head.eval()
    graph, out = capture()
    for k in range(4):
        x.copy_(torch.randn(5, 40, 64, device=DEV))
        t.copy_(torch.randint(-1, 200, (5, 40), device=DEV) if k else torch.full((5, 40), -1, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step()):
            assert torch.equal(p, q), k


def test_longer_than_any_tile_and_odd_everywhere():
    """One row, one feature, one output up to sizes beyond every tile, all odd: against 64 bits as vectors."""
    g = torch.Generator().manual_seed(8)
    for N, D, V in ((1, 1, 1), (1, 3, 5), (2, 1, 129), (513, 1, 1027), (33, 2051, 7), (1025, 5, 130), (4099, 65, 257)):
        x, w = torch.randn(N, D, generator=g).to(DEV).requires_grad_(), torch.randn(V, D, generator=g).to(DEV).requires_grad_()
        t = torch.randint(0, V, (N,), generator=g).to(DEV)
        got = torch.autograd.grad(wf.linear_cross_entropy(x, w, t), (x, w))
        rx, rw = x.detach().double().requires_grad_(), w.detach().double().requires_grad_()
        want = torch.autograd.grad(torch.nn.functional.cross_entropy(rx @ rw.t(), t), (rx, rw))
        for p, q, what in zip(got, want, ("dx", "dw")):
            if V == 1:
                # p - 1 is a difference of equal numbers: zero up to the roundings of exp and log
                assert (p.double() - q).abs().max() <= 2.0 ** -18 * 8, what
            else:
                near(p, q, 2.0 ** -12, (N, D, V, what))
