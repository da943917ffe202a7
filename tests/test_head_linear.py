"""linear_log_softmax and linear_cross_entropy against float64 restatements of their formulas, with elementwise bounds that
count roundings.

u = 2^-24 / 2^-8 / 2^-11 is one rounding of float32 / bfloat16 / float16.  A product of K terms a_k b_k:
  * 16-bit operands are exact in fp32; the running sum is rounded once per 16 terms at most (matrix instructions), counted
    twice for the rounding inside one: (K / 8 + 32) u_32 sum |a_k b_k|;
  * float32 operands are three bf16 parts by truncation, |second| < 2^-7, |third| < 2^-15 of the value: the products left out
    are below 2 * 2^-22 + 2^-30 of |a b|, and there are six times the roundings: 2^-20.9 + (6 K / 8 + 32) u_32.
With e the bound of a logit, log-sum-exp is off by at most max e plus the exponentials' and logarithm's own errors (relative
2^-20 covers an fp32 exponential with an argument up to 16 beyond its unit, and the sums of up to 118 partial sums), the
probability p by p (expm1 of both).  Then rounding to 16 bits of the gradient of a logit, and of the result."""
import math

import pytest
import torch

import waterfall_amd as wf
from waterfall_amd import _lib

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
DEV = "cuda:0"
gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
# one of everything; below and above a tile of 128 / 256, odd ones, a K tail, a K that is not a multiple of 8
SIZES = [(1, 1, 1), (1, 512, 5001), (3, 64, 2), (5, 7, 59), (64, 65, 128), (127, 72, 129), (128, 128, 256), (129, 257, 255),
         (300, 64, 513), (513, 192, 300), (1000, 80, 59), (2, 1030, 1), (296, 257, 5001),
         # outputs in whole 64s and around them, features around the 32 and 64 columns of a workgroup, splits over many rows
         (40, 33, 64), (100, 63, 65), (5000, 31, 33), (4099, 95, 127), (40000, 33, 50),
         # more work than the direct kernels take: tiles, with rows, outputs and features that end inside one
         (300, 1031, 6007), (700, 641, 5003), (2049, 257, 4099), (20003, 700, 131)]


def k_error(dtype, K):
    return (2.0 ** -20.9 + (6 * K / 8 + 32) * 2.0 ** -24) if dtype == torch.float32 else (K / 8 + 32) * 2.0 ** -24


class Case:
    def __init__(self, N, D, V, dtype, bias=True, seed=0, scale=1.0):
        g = torch.Generator().manual_seed(1000 * N + 10 * D + V + seed)
        self.x = (scale * torch.randn(N, D, generator=g)).to(dtype).to(DEV)
        self.w = (2.0 / math.sqrt(D) * torch.randn(V, D, generator=g)).to(dtype).to(DEV)
        self.b = (0.5 * torch.randn(V, generator=g)).to(dtype).to(DEV) if bias else None
        self.t = torch.randint(0, V, (N,), generator=g).to(DEV)
        self.g = g
        self.dtype, self.N, self.D, self.V = dtype, N, D, V

    def logits(self, rows=None):
        """z, its log-softmax and the bounds of both, in 64 bits"""
        x = self.x.double() if rows is None else self.x[rows].double()
        z = x @ self.w.double().t()
        size = x.abs() @ self.w.double().abs().t()
        if self.b is not None:
            z = z + self.b.double()
            size = size + torch.nan_to_num(self.b.double().abs(), posinf=0.0)
        e = k_error(self.dtype, self.D) * size + 2.0 ** -24 * torch.nan_to_num(z.abs(), posinf=0.0)
        lse = torch.logsumexp(z, 1, keepdim=True)
        el = e.amax(1, keepdim=True) + 2.0 ** -20 + 4 * 2.0 ** -24 * lse.abs()
        return z, lse, e, el

    def products(self, dz, edz, scale=0.0):
        """dx, dw, db of d loss / d z = dz known to within edz, and their bounds.  scale: what fp16 gradients are relative to."""
        x, w, u = self.x.double(), self.w.double(), U[self.dtype]
        if self.dtype != torch.float32:
            edz = edz + u * (dz.abs() + edz) + HALF_STEP[self.dtype] * scale
        out = []
        for want, spread, size, K in ((dz @ w, edz @ w.abs(), dz.abs() @ w.abs(), self.V),
                                      (dz.t() @ x, edz.t() @ x.abs(), dz.abs().t() @ x.abs(), self.N),
                                      (dz.sum(0), edz.sum(0), dz.abs().sum(0), self.N)):
            # K is summed in pieces and splits: a handful of additions more, inside the 32
            bound = spread + k_error(self.dtype, K) * size
            out.append((want, bound + u * (want.abs() + bound) + HALF_STEP[self.dtype]))
        return out


def within(got, want, bound, what):
    assert got.shape == want.shape, what
    over = ((got.double() - want).abs() - bound)
    assert torch.isfinite(got).all(), what
    assert over.max().item() <= 0, (what, over.max().item(), (over > 0).sum().item())


def check_grads(got, wants, what):
    for g, (want, bound), name in zip(got, wants, ("dx", "dweight", "dbias")):
        if g is not None:
            within(g, want, bound, (what, name))


def dz_of_log_softmax(c, G):
    z, lse, e, el = c.logits()
    p = torch.exp(z - lse)
    s = G.double().sum(1, keepdim=True)
    abs_s = G.double().abs().sum(1, keepdim=True)
    ep = p * torch.expm1(e + el + 2.0 ** -20)
    # the sum of V terms by 256 threads and a tree: chains of V / 256 + 8
    es = (c.V / 256 + 16) * 2.0 ** -24 * abs_s
    return G.double() - p * s, ep * s.abs() + (p + ep) * es + 3 * 2.0 ** -24 * (G.double().abs() + p * s.abs())


def dz_of_entropy(c, g, eps):
    z, lse, e, el = c.logits()
    p = torch.exp(z - lse)
    ep = p * torch.expm1(e + el + 2.0 ** -20)
    valid = (c.t >= 0) & (c.t < c.V)
    hot = torch.zeros_like(p)
    hot[valid, c.t[valid]] = 1 - eps
    g = torch.where(valid, g.double(), torch.zeros((), dtype=torch.float64, device=DEV))[:, None]
    # g relative to the largest, the target's share taken out and put back behind the products: ten roundings at most
    return g * (p - hot - eps / c.V), g.abs() * (ep + 10 * 2.0 ** -24 * (p + hot + eps / c.V))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", SIZES)
def test_log_softmax_and_gradients(N, D, V, dtype):
    c = Case(N, D, V, dtype, bias=V != 59)
    leaves = [t.requires_grad_() for t in (c.x, c.w, c.b) if t is not None]
    lp = wf.linear_log_softmax(c.x, c.w, c.b)
    assert lp.dtype == torch.float32 and lp.shape == (N, V)
    with torch.no_grad():
        z, lse, e, el = c.logits()
        within(lp.detach(), z - lse, e + el + 2.0 ** -24 * (z - lse).abs(), "log_probs")
        G = torch.randn(N, V, generator=c.g).to(DEV) * 0.01
        G[N // 2:, :] *= (torch.rand(N - N // 2, 1, generator=c.g) < 0.7).to(DEV)       # some rows without a gradient
    got = torch.autograd.grad(lp, leaves, G)
    with torch.no_grad():
        check_grads(got, c.products(*dz_of_log_softmax(c, G), 2 * G.abs().max().item()), (N, D, V))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", SIZES)
def test_cross_entropy_and_gradients(N, D, V, dtype):
    c = Case(N, D, V, dtype, bias=V != 300)
    with torch.no_grad():
        if N > 2:
            c.t[torch.rand(N, generator=c.g).to(DEV) < 0.3] = -1
        z, lse, e, el = c.logits()
    live = c.t >= 0
    n = max(1, int(live.sum()))
    for eps in (0.0, 0.1, 1.0):
        with torch.no_grad():
            zt = z.gather(1, c.t.clamp(min=0)[:, None])
            want = (lse - (1 - eps) * zt - eps * z.mean(1, keepdim=True))[:, 0]
            # the mean of V logits: V / 16 + 128 additions deep at most, 2^-24 of the running sum each
            bound = (el + e.amax(1, keepdim=True) + 8 * 2.0 ** -24 * (lse.abs() + zt.abs()))[:, 0] + eps * (V / 16 + 128) * 2.0 ** -24 * z.abs().mean(1)
            want, bound = want * live, bound * live
        for reduction in ("none", "sum", "mean"):
            leaves = [t.detach().requires_grad_() for t in (c.x, c.w, c.b) if t is not None]
            t = c.t.int() if reduction == "sum" else c.t
            loss = wf.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2] if c.b is not None else None, label_smoothing=eps, reduction=reduction)
            assert loss.dtype == torch.float32
            with torch.no_grad():
                if reduction == "none":
                    within(loss.detach(), want, bound, "loss")
                    up = torch.randn(N, generator=c.g).to(DEV)
                    g = up
                else:
                    k = n if reduction == "mean" else 1
                    within(loss.detach(), want.sum() / k, (bound.sum() + (N / 1024 + 32) * 2.0 ** -24 * want.abs().sum()) / k, reduction)
                    up = torch.tensor(1.7, device=DEV)
                    g = (up / k).expand(N)
            got = torch.autograd.grad(loss, leaves, up)
            with torch.no_grad():
                check_grads(got, c.products(*dz_of_entropy(c, torch.where(live, g, 0.0), eps), 2 * g.abs().max().item()), (N, D, V, eps, reduction))
                assert not got[0][~live].any()


@gpu
@pytest.mark.parametrize("dtype,N,D,V", [(torch.bfloat16, 16384, 64, 10001), (torch.float16, 9000, 128, 20000), (torch.float32, 6000, 96, 10001)])
def test_several_pieces_of_the_outputs(dtype, N, D, V):
    """More than 256 MB of logit gradients: dx is summed over pieces; large tiles; targets in every piece."""
    c = Case(N, D, V, dtype)
    with torch.no_grad():
        c.t[N - N // 8:] = -1
        dz, edz = dz_of_entropy(c, torch.where(c.t >= 0, 1.0 / (N - N // 8), 0.0), 0.1)
        wants = c.products(dz, edz, 2.0 / (N - N // 8))
        del dz, edz
    leaves = [t.detach().requires_grad_() for t in (c.x, c.w, c.b)]
    got = torch.autograd.grad(wf.linear_cross_entropy(leaves[0], leaves[1], c.t, leaves[2], label_smoothing=0.1), leaves)
    check_grads(got, wants, (N, D, V))
    lp = wf.linear_log_softmax(*leaves)
    with torch.no_grad():
        z, lse, e, el = c.logits()
        within(lp.detach(), z - lse, e + el + 2.0 ** -24 * (z - lse).abs(), "log_probs")
        del z, lse, e, el
        G = torch.randn(N, V, device=DEV) * 1e-3
        G[::5] = 0
        wants = c.products(*dz_of_log_softmax(c, G), 2 * G.abs().max().item())
    check_grads(torch.autograd.grad(lp, leaves, G), wants, (N, D, V))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_take_no_part_may_hold_anything(dtype):
    c = Case(200, 96, 700, dtype)
    dead = torch.zeros(200, dtype=torch.bool, device=DEV)
    dead[[0, 3, 77, 198, 199]] = True
    dead[100:140] = True
    x = c.x.clone()
    x[dead] = float("nan")
    x[3] = float("inf")
    t = torch.where(dead, -100, c.t)
    a = [v.detach().requires_grad_() for v in (x, c.w, c.b)]
    loss = wf.linear_cross_entropy(a[0], a[1], t, a[2], ignore_index=-100, reduction="none")
    got = torch.autograd.grad(loss.sum(), a)
    b = [v.detach().requires_grad_() for v in (c.x[~dead], c.w, c.b)]
    ref = wf.linear_cross_entropy(b[0], b[1], c.t[~dead], b[2], reduction="none")
    want = torch.autograd.grad(ref.sum(), b)
    assert torch.equal(loss[~dead], ref) and not loss[dead].any()
    assert torch.equal(got[0][~dead], want[0]) and not got[0][dead].any()
    # sums over the rows are split by the number of rows of the call: not bit by bit, but both within the formula's bound
    few = Case(200, 96, 700, dtype)
    few.x, few.t, few.N = c.x[~dead], c.t[~dead], 200
    bounds = few.products(*dz_of_entropy(few, torch.ones(len(few.t), device=DEV), 0.0), 2.0)
    check_grads((None,) + got[1:], bounds, "entropy, masked rows")
    check_grads(want, bounds, "entropy, live rows alone")
    # the same for log-probabilities: rows without an incoming gradient
    lp = wf.linear_log_softmax(*a)
    G = torch.randn(200, 700, device=DEV)
    G[dead] = 0
    got = torch.autograd.grad(lp, a, G)
    want = torch.autograd.grad(wf.linear_log_softmax(*b), b, G[~dead])
    assert torch.equal(got[0][~dead], want[0]) and not got[0][dead].any()
    bounds = few.products(*dz_of_log_softmax(few, G[~dead]), 2 * G.abs().max().item())
    check_grads((None,) + got[1:], bounds, "log-probabilities, masked rows")
    check_grads(want, bounds, "log-probabilities, live rows alone")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_nothing_left_of_the_rows_or_of_the_outputs(dtype):
    c = Case(40, 64, 130, dtype)
    a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    none = torch.full_like(c.t, -1)
    for reduction in ("mean", "sum", "none"):
        loss = wf.linear_cross_entropy(a[0], a[1], none, a[2], reduction=reduction)
        assert not loss.detach().any()
        for g in torch.autograd.grad(loss.sum(), a):
            assert not g.any()
    for g in torch.autograd.grad(wf.linear_log_softmax(*a), a, torch.zeros(40, 130, device=DEV)):
        assert not g.any()
    # no rows at all
    e = [a[0].detach()[:0].reshape(0, 3, 64).requires_grad_(), a[1], a[2]]
    for y in (wf.linear_log_softmax(*e), wf.linear_cross_entropy(e[0], e[1], none[:0].reshape(0, 3), e[2]),
              wf.linear_cross_entropy(e[0], e[1], none[:0].reshape(0, 3), e[2], reduction="none")):
        assert not y.detach().any()
        for g in torch.autograd.grad(y.sum(), e):
            assert not g.any()
    # outputs masked by their bias: probability 0, as if they were not there
    keep = torch.ones(130, dtype=torch.bool, device=DEV)
    keep[[0, 5, 64, 127, 128]] = False
    b = torch.where(keep, c.b, float("-inf")).requires_grad_()
    lp = wf.linear_log_softmax(a[0], a[1], b)
    assert (lp.detach()[:, ~keep] == float("-inf")).all()
    sub = Case(40, 64, 130, dtype)
    sub.w, sub.b = c.w[keep], c.b[keep]
    sub.V = 125
    z, lse, e2, el = sub.logits()
    within(lp.detach()[:, keep], (z - lse), e2 + el + 2.0 ** -24 * (z - lse).abs(), "masked")
    t = torch.nonzero(keep)[torch.arange(40, device=DEV) % 125, 0]
    for g in torch.autograd.grad(wf.linear_cross_entropy(a[0], a[1], t, b), (a[0], a[1], b)):
        assert torch.isfinite(g).all()
    # every output masked: -inf, an infinite loss, no gradient
    gone = torch.full((130,), float("-inf"), device=DEV, dtype=dtype).requires_grad_()
    lp = wf.linear_log_softmax(a[0], a[1], gone)
    assert (lp.detach() == float("-inf")).all()
    loss = wf.linear_cross_entropy(a[0], a[1], c.t, gone, reduction="none")
    assert (loss.detach() == float("inf")).all()
    for g in torch.autograd.grad(loss, (a[0], a[1], gone), torch.ones(40, device=DEV)) + torch.autograd.grad(lp, (a[0], a[1], gone), torch.ones(40, 130, device=DEV)):
        assert torch.isfinite(g).all()


@gpu
def test_targets_that_are_no_output_and_values_that_are_not_finite_stay_in_their_row():
    c = Case(50, 64, 300, torch.bfloat16)
    t = c.t.clone()
    t[4], t[5], t[6] = 300, -2, 1 << 40
    a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    loss = wf.linear_cross_entropy(a[0], a[1], t, a[2], reduction="none")
    bad = torch.zeros(50, dtype=torch.bool, device=DEV)
    bad[[4, 5, 6]] = True
    assert torch.isnan(loss[bad]).all() and torch.isfinite(loss[~bad]).all()
    dx, dw, db = torch.autograd.grad(loss, a, torch.ones(50, device=DEV))
    assert not dx[bad].any() and torch.isfinite(dw).all()
    x = c.x.detach().clone()
    x[7, 3] = float("inf")
    x[9, 0] = float("nan")
    lp = wf.linear_log_softmax(x, c.w, c.b)
    loss = wf.linear_cross_entropy(x, c.w, c.t, c.b, reduction="none")
    rows = torch.ones(50, dtype=torch.bool, device=DEV)
    rows[[7, 9]] = False
    assert torch.isfinite(lp[rows]).all() and torch.isfinite(loss[rows]).all()
    assert torch.isnan(loss[9]) and torch.isnan(lp[9]).all()
    assert not torch.isfinite(lp[7]).any() and not torch.isfinite(loss[7])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layouts_strides_and_partial_gradients(dtype):
    g = torch.Generator().manual_seed(11)
    big = torch.randn(9, 8, 200, generator=g).to(dtype).to(DEV)
    wide = (torch.randn(333, 264, generator=g) * 0.1).to(dtype).to(DEV)
    b = torch.randn(333, generator=g).to(DEV)                                 # fp32 bias beside 16-bit operands
    t = torch.randint(0, 333, (9, 8), generator=g).to(DEV)
    for x, w, tt in ((big[..., :128], wide[:, 3:131], t), (big.transpose(0, 1)[..., 8:136], wide[:, 128:256], t.t()),
                     (big[::2, 1:, 64:192], wide[:, :128], t[::2, 1:]), (big[:1, :1, :128].expand(9, 8, 128), wide[:, 8:136], t),
                     (big.permute(2, 1, 0)[:128].permute(1, 2, 0), wide.t()[:128].t(), t.t())):
        a = [v.detach().requires_grad_() for v in (x, w, b)]
        d = [v.detach().contiguous().requires_grad_() for v in (x, w, b)]
        y, z = wf.linear_log_softmax(*a), wf.linear_log_softmax(*d)
        assert torch.equal(y, z)
        box = torch.randn(y.shape[:-1] + (400,), generator=g).to(DEV)
        for p, q in zip(torch.autograd.grad(y, a, box[..., 7:340]), torch.autograd.grad(z, d, box[..., 7:340].contiguous())):
            assert p.shape == q.shape and torch.equal(p, q)
        y, z = wf.linear_cross_entropy(a[0], a[1], tt, a[2]), wf.linear_cross_entropy(d[0], d[1], tt.contiguous(), d[2])
        assert torch.equal(y, z)
        whole = torch.autograd.grad(z, d, retain_graph=True)
        for p, q in zip(torch.autograd.grad(y, a), whole):
            assert torch.equal(p, q)
        for k in range(3):                                                    # one gradient alone, twice through one node
            for _ in range(2):
                assert torch.equal(torch.autograd.grad(z, d[k], retain_graph=True)[0], whole[k])
    x, w = big[..., :128].contiguous().requires_grad_(), wide[:, :128].contiguous()
    for y in (wf.linear_log_softmax(x, w)[..., :2].sum(), wf.linear_log_softmax(x, w).sum(), wf.linear_cross_entropy(x, w, t, reduction="none").sum()):
        assert torch.isfinite(torch.autograd.grad(y, x)[0]).all()             # expanded and partly filled gradients


@gpu
def test_gradients_against_differences():
    c = Case(6, 20, 33, torch.float32)
    t = c.t.clone()
    t[2] = -1
    up = torch.randn(6, 33, generator=c.g).double().to(DEV)

    def both(x, w, b):
        lp = torch.log_softmax(x @ w.t() + b, -1)
        m = (t >= 0).double()
        ce = -(0.9 * lp.gather(1, t.clamp(min=0)[:, None])[:, 0] + 0.1 * lp.mean(1)) * m
        return (lp * up).sum(), ce.sum() / m.sum()

    leaves = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    got = (torch.autograd.grad(wf.linear_log_softmax(*leaves), leaves, up.float()),
           torch.autograd.grad(wf.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], label_smoothing=0.1), leaves))
    for k in range(3):
        for i in range(0, leaves[k].numel(), 17):
            v = []
            for h in (1e-4, -1e-4):
                args = [u.detach().double().clone() for u in leaves]
                args[k].reshape(-1)[i] += h
                v.append(both(*args))
            for q in range(2):
                d = ((v[0][q] - v[1][q]) / 2e-4).item()
                # h^2 / 6 times a third derivative of order |up| |x|^3 <= 100: below 1e-6; fp32 arithmetic of ~1e3 terms: 1e-5
                assert abs(d - got[q][k].reshape(-1)[i].item()) <= 2e-5 * (1 + abs(d)), (k, i, q)


@gpu
def test_the_same_inputs_give_the_same_bits_on_any_stream():
    c = Case(777, 320, 2000, torch.bfloat16)
    c.t[::9] = -1
    G = torch.randn(777, 2000, device=DEV)

    def step():
        a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
        lp, ce = wf.linear_log_softmax(*a), wf.linear_cross_entropy(a[0], a[1], c.t, a[2])
        return [lp, ce, *torch.autograd.grad(lp, a, G), *torch.autograd.grad(ce, a)]

    want = step()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(step())
    torch.cuda.synchronize()
    for r in got:
        for a, b in zip(r, want):
            assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_the_projection_in_a_captured_graph(dtype):
    c = Case(150, 96, 400, dtype)
    G = torch.randn(150, 400, device=DEV)
    t = c.t.clone()

    def step(a):
        lp, ce = wf.linear_log_softmax(*a), wf.linear_cross_entropy(a[0], a[1], t, a[2], label_smoothing=0.1)
        return [lp, ce, *torch.autograd.grad(lp, a, G), *torch.autograd.grad(ce, a)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [v.detach().clone().requires_grad_() for v in (c.x, c.w, c.b)]
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
    for k in range(4):
        t.copy_(torch.where(torch.rand(150, device=DEV) < 0.2 * k, -1, (c.t + k) % 400))      # other rows take part
        with torch.no_grad():
            leaves[0].copy_(c.x * (1 + 0.1 * k))
        graph.replay()
        torch.cuda.synchronize()
        want = step([v.detach().clone().requires_grad_() for v in leaves])
        for p, q in zip(out, want):
            assert torch.equal(p, q), k


def test_the_projection_refuses_what_it_cannot_do():
    x, w = torch.zeros(2, 8), torch.zeros(3, 8)
    with pytest.raises(_lib.WfError, match="GPU"):
        wf.linear_log_softmax(x, w)
    with pytest.raises(_lib.WfError, match="GPU"):
        wf.linear_cross_entropy(x, w, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        wf.linear_log_softmax(x.double(), w.double())
    with pytest.raises(ValueError):
        wf.OutputHead(4, 5, dropout=2.0)
    import ctypes as C
    lib, n = _lib.lib(), C.c_size_t(0)
    for what, N, D, V, t, rc in ((0, 5, 8, 3, 0, 0), (4, 5, 8, 3, 0, -1), (0, -1, 8, 3, 0, -1), (1, 5, 0, 3, 0, -1), (2, 5, 8, 0, 0, -1),
                                 (3, 5, 8, 3, 9, -1), (0, 1 << 31, 8, 3, 0, -5), (0, 5, 1 << 21, 3, 0, -5), (0, 5, 8, (1 << 21) + 1, 0, -5)):
        assert lib.wf_linear_workspace_bytes(what, N, D, V, t, C.byref(n)) == rc, (what, N, D, V, t)
    # too small a workspace, null pointers, a bad smoothing: an error before anything is launched
    assert lib.wf_linear_log_softmax(1, 8, 2, 8, 1, 8, 3, 0, None, 0, 1, 256, 10, None) == -2
    assert lib.wf_linear_log_softmax(None, 8, 2, 8, 1, 8, 3, 0, None, 0, 1, 256, 1 << 40, None) == -1
    assert lib.wf_linear_log_softmax(1, 8, 2, 8, 1, -8, 3, 0, None, 0, 1, 256, 1 << 40, None) == -1
    assert lib.wf_linear_log_softmax(1, 1 << 30, 2, 8, 1, 8, 3, 0, None, 0, 1, 256, 1 << 40, None) == -5
    assert lib.wf_linear_cross_entropy(1, 8, 2, 8, 1, 1 << 30, 3, 0, None, 0, 1, 1, -1, 0.0, 1, 1, None, 0, 256, 1 << 40, None) == -5
    assert lib.wf_linear_cross_entropy(1, 8, 2, 8, 1, 8, 3, 0, None, 0, 1, 1, -1, 1.5, 1, 1, None, 0, 256, 1 << 40, None) == -1
    assert lib.wf_linear_cross_entropy(1, 8, 2, 8, 1, 8, 3, 0, None, 0, None, 1, -1, 0.0, 1, 1, None, 0, 256, 1 << 40, None) == -1
    assert lib.wf_linear_cross_entropy(1, 8, 2, 8, 1, 8, 3, 0, 1, 8, 1, 1, -1, 0.0, 1, 1, None, 0, 256, 1 << 40, None) == -1
    assert lib.wf_linear_cross_entropy_backward(1, 0, 0, None, 1, 8, 2, 8, 1, 8, 3, 0, None, 0, 1, 1, -1, 0.0, 1, 1, None, 256, 1 << 40, None) == -1
    assert lib.wf_linear_log_softmax_backward(1, None, 3, 1, 8, 2, 8, 1, 8, 3, 0, 0, 1, 1, None, 256, 1 << 40, None) == -1


@gpu
def test_rows_that_lie_more_than_2_30_elements_apart():
    big = torch.empty((1 << 30) + 64, dtype=torch.bfloat16, device=DEV)
    x = big.as_strided((2, 64), (1 << 30, 1))
    c = Case(2, 64, 40, torch.bfloat16)
    x.copy_(c.x)
    y = x.detach().requires_grad_()
    out = wf.linear_cross_entropy(y, c.w, c.t)
    assert torch.equal(out, wf.linear_cross_entropy(c.x, c.w, c.t))
    dx, = torch.autograd.grad(out, y)
    d = c.x.detach().requires_grad_()
    assert torch.equal(dx, torch.autograd.grad(wf.linear_cross_entropy(d, c.w, c.t), d)[0])
    same = c.x[:1].expand(5, 64)                                             # the other end: one row five times
    assert torch.equal(wf.linear_log_softmax(same, c.w), wf.linear_log_softmax(same.contiguous(), c.w))


@gpu
def test_boxes_and_rows_beyond_2_31_elements():
    dtype, u = torch.bfloat16, U[torch.bfloat16]
    N, D, V = 429500, 64, 5001                                                # N V passes 2^31
    c = Case(N, D, V, dtype)
    with torch.no_grad():
        G = torch.empty(N, V, device=DEV)
        for n in range(0, N, 20000):
            G[n:n + 20000].normal_(std=0.01)
        G[::7] = 0
    leaves = [t.requires_grad_() for t in (c.x, c.w, c.b)]
    lp = wf.linear_log_softmax(*leaves)
    dx, dw, db = torch.autograd.grad(lp, leaves, G)
    lp = lp.detach()
    want = [torch.zeros(V, D, device=DEV, dtype=torch.float64) for _ in range(3)] + [torch.zeros(V, device=DEV, dtype=torch.float64) for _ in range(3)]
    with torch.no_grad():
        for n in range(0, N, 20000):
            part = Case.__new__(Case)
            part.x, part.w, part.b, part.dtype, part.D, part.V = c.x[n:n + 20000].detach(), c.w.detach(), c.b.detach(), dtype, D, V
            part.N = part.x.shape[0]
            z, lse, e, el = part.logits()
            within(lp[n:n + 20000], z - lse, e + el + 2.0 ** -24 * (z - lse).abs(), ("log_probs", n))
            del z, lse, e, el
            dz, edz = dz_of_log_softmax(part, G[n:n + 20000])
            within(dx[n:n + 20000], *part.products(dz, edz)[0], ("dx", n))
            edz = edz + u * (dz.abs() + edz)
            x = part.x.double()
            for k, (m, b) in enumerate(((dz, x), (edz, x.abs()), (dz.abs(), x.abs()))):
                want[k] += m.t() @ b
                want[3 + k] += m.sum(0)
            del dz, edz
        for got, (w, spread, size), what in ((dw, want[:3], "dweight"), (db, want[3:], "dbias")):
            bound = spread + k_error(dtype, N) * size
            within(got, w, bound + u * (w.abs() + bound), what)
    del G, lp, c, leaves, dx
    torch.cuda.empty_cache()
    N, D, V = (1 << 21) - 64, 1040, 50                                        # N D passes 2^31: the most rows the direct kernels take
    g = torch.Generator(device=DEV).manual_seed(5)
    x = torch.empty(N, D, dtype=dtype, device=DEV).normal_(generator=g)
    few = Case(300, D, V, dtype)
    at = torch.cat((torch.arange(100), torch.arange(N // 2, N // 2 + 100), torch.arange(N - 100, N))).to(DEV)
    x[at] = few.x
    t = torch.full((N,), -1, device=DEV)
    t[at] = few.t
    assert torch.equal(wf.linear_log_softmax(x, few.w, few.b)[at], wf.linear_log_softmax(few.x, few.w, few.b))
    y = x.detach().requires_grad_()
    w, b = few.w.detach().requires_grad_(), few.b.detach().requires_grad_()
    got = torch.autograd.grad(wf.linear_cross_entropy(y, w, t, b), (y, w, b))
    f = few.x.detach().requires_grad_()
    ref = torch.autograd.grad(wf.linear_cross_entropy(f, w, few.t, b), (f, w, b))
    assert torch.equal(got[0][at], ref[0])                                    # the same rows, alone in a small batch
    assert got[0].ne(0).any(1).sum().item() <= 300
    with torch.no_grad():
        check_grads(got[1:], few.products(*dz_of_entropy(few, torch.full((300,), 1 / 300, device=DEV), 0.0))[1:], "weights")


@gpu
def test_the_projection_refuses_mismatches():
    x, w, b = torch.zeros(2, 8, device=DEV), torch.zeros(3, 8, device=DEV), torch.zeros(3, device=DEV)
    t = torch.zeros(2, dtype=torch.int64, device=DEV)
    for args in ((x, w[:, :7]), (x, w[None]), (x, w, b[:2]), (x, w[:0])):
        with pytest.raises(ValueError):
            wf.linear_log_softmax(*args)
    with pytest.raises(TypeError):
        wf.linear_log_softmax(x, w.bfloat16())
    for bad, kw in ((t[:1], {}), (t, dict(label_smoothing=-0.1)), (t, dict(reduction="max")), (t.cpu(), {})):
        with pytest.raises(ValueError):
            wf.linear_cross_entropy(x, w, bad, b, **kw)
    with pytest.raises(TypeError):
        wf.linear_cross_entropy(x, w, t.float(), b)
