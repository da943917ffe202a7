"""layer_norm and dropout against plain float64 restatements: sizes at the edges of the kernels' row shapes, odd lengths,
strides, parameter types, masked infinities, refusals.

Tolerances count roundings.  u = 2^-24 (fp32), 2^-8 (bfloat16), 2^-11 (float16) is the relative error of one rounding.  A
result of type t is computed in fp32 and rounded once: |error| <= u_t |y| plus the fp32 arithmetic, whose errors are relative
to the terms that were added: 32 u_32 times their size covers the chain (a sum of n terms by lanes and a tree takes a
dozen additions deep at the widths tested here, the mean and the inverse deviation a handful of operations more).  Below its
smallest normal number 2^-14 float16 has steps of 2^-24: a result there is off by up to half of one, 2^-25, whatever its size."""
import numpy as np
import pytest
import torch

import waterfall_amd as wf
from waterfall_amd import _lib

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
HALF_STEP = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}      # of the subnormal numbers, where it counts
DEV = "cuda:0"
gpu = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def philox7(n, seed):
    """Words of Philox4x32-7 for counters 0, 1, ... by Python's own integers in numpy's unsigned 64 bits."""
    c = [np.arange((n + 3) // 4, dtype=np.uint64) for _ in range(1)] + [np.zeros((n + 3) // 4, np.uint64) for _ in range(3)]
    k = [seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF]
    lo = np.uint64(0xFFFFFFFF)
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & lo, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & lo]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, 1).reshape(-1)[:n]


def norm64(x, w, b, eps, dy=None):
    x = x.double().cpu()
    mean = x.mean(-1, keepdim=True)
    d = x - mean
    r = 1 / torch.sqrt((d * d).mean(-1, keepdim=True) + eps)
    h = d * r
    w = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.double().cpu()
    y = h * w + (0 if b is None else b.double().cpu())
    if dy is None:
        return y
    g = dy.double().cpu()
    gw = g * w
    dx = r * (gw - gw.mean(-1, keepdim=True) - h * (gw * h).mean(-1, keepdim=True))
    lead = tuple(range(x.dim() - 1))
    return y, dx, (g * h).sum(lead), g.sum(lead), (g * h).abs().sum(lead), g.abs().sum(lead), r, gw, h


def within(got, want, bound, what):
    bound = bound + HALF_STEP[got.dtype]
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = ((got - want).abs() - bound).max().item()
    assert over <= 0, (what, over)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1), (1, 512), (3, 2), (5, 1, 63), (2, 7, 255), (4, 513), (1000, 256), (9, 1023), (3, 2049),
                                   (2, 4097), (2, 8193), (1, 16385), (2, 32768), (0, 16), (2, 0, 16), (4097, 80)])
def test_layer_norm_and_gradients(shape, dtype):
    g = torch.Generator().manual_seed(hash((shape, 3)) & 0xFFFF)
    D = shape[-1]
    x = (torch.randn(shape, generator=g) * 1.5 + 0.7).to(dtype)
    w, b = (torch.randn(D, generator=g) + 1).to(dtype), torch.randn(D, generator=g).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    lx, lw, lb = (t.to(DEV).requires_grad_() for t in (x, w, b))
    y = wf.layer_norm(lx, lw, lb)
    assert y.dtype == dtype and y.shape == x.shape and y.is_contiguous()
    y.backward(dy.to(DEV))
    want, dx, dw, db, adw, adb, r, gw, h = norm64(x, w, b, 1e-5, dy)
    u, f = U[dtype], 32 * U[torch.float32]
    if x.numel() == 0:
        assert lx.grad.shape == x.shape and not lw.grad.any() and not lb.grad.any()
        return
    # (x - mean): an error of the mean of f |x| counts with rstd; the terms of dx are of size r (|gw| + means)
    big = x.double().abs().amax(-1, keepdim=True)
    within(y, want, u * want.abs() + f * ((big * r + h.abs()) * w.double().abs() + want.abs()) + 1e-30, "y")
    size = r * (gw.abs() + gw.abs().mean(-1, keepdim=True) + (h.abs() + big * r) * (1 + (gw * h).abs().mean(-1, keepdim=True) + gw.abs().amax(-1, keepdim=True)))
    within(lx.grad, dx, u * dx.abs() + f * size, "dx")
    # a sum over N rows: chains of at most N / 256 / 16 + 16 + 6 additions; f covers 32 roundings of the running sum
    rows = max(1, x.numel() // D)
    fr = f * (1 + rows / 4096)
    within(lw.grad, dw, u * dw.abs() + fr * (adw + (dy.double().abs() * big * r).sum(tuple(range(x.dim() - 1)))), "dweight")
    within(lb.grad, db, u * db.abs() + fr * adb, "dbias")


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_layer_norm_rows_of_other_layouts_and_parameters(dtype):
    g = torch.Generator().manual_seed(5)
    big = torch.randn(6, 5, 96, generator=g).to(dtype).to(DEV)
    w, b = torch.randn(70, generator=g).to(DEV), torch.randn(70, generator=g).to(DEV)      # fp32 parameters
    for view in (big[..., 3:73], big[::2, :, :70], big.transpose(0, 1)[..., 1:71], big[:1, :1, :70].expand(4, 3, 70),
                 big.permute(1, 2, 0)[:, :70, :].transpose(1, 2)):
        x = view.detach().requires_grad_()
        lw, lb = w.clone().requires_grad_(), b.clone().requires_grad_()
        y = wf.layer_norm(x, lw, lb)
        dense = view.contiguous().requires_grad_()
        dw, db = w.clone().requires_grad_(), b.clone().requires_grad_()
        z = wf.layer_norm(dense, dw, db)
        assert torch.equal(y, z)
        dy = torch.randn(y.shape, generator=g).to(dtype).to(DEV)
        wide = torch.zeros(y.shape[:-1] + (80,), dtype=dtype, device=DEV)
        wide[..., 5:75] = dy
        gx, gw, gb = torch.autograd.grad(y, (x, lw, lb), wide[..., 5:75])          # a gradient with strides of its own
        hx, hw, hb = torch.autograd.grad(z, (dense, dw, db), dy)
        assert torch.equal(gx, hx) and torch.equal(gw, hw) and torch.equal(gb, hb)
    x = big[..., :70].contiguous()
    none = wf.layer_norm(x)
    assert torch.equal(none, wf.layer_norm(x, torch.ones(70, device=DEV), torch.zeros(70, device=DEV)))
    xb = x.detach().requires_grad_()
    only = b.clone().requires_grad_()
    wf.layer_norm(xb, None, only).sum().backward()                                   # an expanded gradient, no weight
    assert torch.equal(only.grad, torch.full((70,), 30.0, device=DEV))


@gpu
def test_layer_norm_a_row_of_infinities_or_equal_values_stays_in_its_row():
    x = torch.randn(40, 300, device=DEV)
    x[3] = 7.5                  # no variance: rstd = 1 / sqrt(eps), y = 0
    x[5, 2] = float("inf")
    x[6, 9] = float("nan")
    y = wf.layer_norm(x)
    assert not y[3].any()
    assert torch.isnan(y[5]).all() and torch.isnan(y[6]).all()
    keep = [i for i in range(40) if i not in (5, 6)]
    assert torch.isfinite(y[keep]).all()


@gpu
def test_layer_norm_beyond_2_31_elements():
    N, D = 2200000, 1000
    x = torch.empty(N, D, dtype=torch.bfloat16, device=DEV).normal_()
    at = torch.cat((torch.arange(50), torch.arange(N // 2, N // 2 + 50), torch.arange(N - 50, N))).to(DEV)
    w, b = torch.randn(D, device=DEV), torch.randn(D, device=DEV)
    big, few = x.requires_grad_(), x.detach()[at].requires_grad_()
    y, z = wf.layer_norm(big, w, b), wf.layer_norm(few, w, b)
    assert torch.equal(y[at], z)
    g = torch.randn(150, D, device=DEV).bfloat16()
    up = torch.zeros_like(x)
    up[at] = g
    dx, = torch.autograd.grad(y, big, up)
    assert torch.equal(dx[at], torch.autograd.grad(z, few, g)[0])
    assert dx.ne(0).any(1).sum().item() <= 150


@gpu
def test_layer_norm_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    x, w, b = torch.randn(3, 37, generator=g), torch.randn(37, generator=g), torch.randn(37, generator=g)
    c = torch.randn(3, 37, generator=g)
    leaves = [t.to(DEV).requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad((wf.layer_norm(*leaves) * c.to(DEV)).sum(), leaves)
    for k, t in enumerate((x, w, b)):
        flat = t.double().reshape(-1)
        for i in range(0, flat.numel(), 11):
            v = []
            for h in (1e-4, -1e-4):
                args = [u.double().clone() for u in (x, w, b)]
                args[k].reshape(-1)[i] += h
                v.append((norm64(*args, 1e-5) * c.double()).sum().item())
            d = (v[0] - v[1]) / 2e-4
            # second-order differences: O(h^2) times the third derivative (about r^3 |c|), and 64-bit cancellation: 1e-6
            assert abs(d - grads[k].reshape(-1)[i].item()) <= 1e-5 * (1 + abs(d)), (k, i)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [0, 1, 3, 4, 5, 7, 8, 9, 2047, 2048, 2049, 100003, 8500001])
def test_dropout_is_the_generator_s_mask_bit_for_bit(n, dtype):
    g = torch.Generator().manual_seed(n)
    x = torch.randn(n, generator=g).to(dtype)
    for p, seed in ((0.1, 12345678901234567890), (0.5, 0), (0.999, -3)):
        lx = x.to(DEV).requires_grad_()
        y = wf.dropout(lx, p, seed)
        keep = torch.from_numpy(philox7(n, seed & 0xFFFFFFFFFFFFFFFF) >= np.uint64(int(p * 2.0 ** 32)))
        scale = torch.tensor(1 / (1 - p), dtype=torch.float32)
        want = torch.where(keep, x.float() * scale, torch.zeros(())).to(dtype)
        assert torch.equal(y.detach().cpu(), want)
        dy = torch.randn(n, generator=g).to(dtype)
        y.backward(dy.to(DEV))
        assert torch.equal(lx.grad.cpu(), torch.where(keep, dy.float() * scale, torch.zeros(())).to(dtype))
        if n > 10 ** 5:
            assert abs(keep.double().mean().item() - (1 - p)) < 6 * (p * (1 - p) / n) ** 0.5


@gpu
def test_dropout_counters_beyond_32_bits_of_words_and_offsets():
    # 2^32 + 40 elements of bfloat16: element indexes pass 32 bits; the tail is compared with the generator at those counters
    n = (1 << 32) + 40
    if torch.cuda.mem_get_info(0)[0] < 40 << 30:
        pytest.skip("needs 20 GB")
    x = torch.ones(n, dtype=torch.bfloat16, device=DEV)
    y = wf.dropout(x, 0.5, 99)
    tail = y[-40:].cpu()
    c = np.arange((n - 40) // 4, n // 4, dtype=np.uint64)
    k, lo, s = [99, 0], np.uint64(0xFFFFFFFF), np.uint64(32)
    w = [c & lo, c >> s, np.zeros(10, np.uint64), np.zeros(10, np.uint64)]
    for _ in range(7):
        a, b = w[0] * np.uint64(0xD2511F53), w[2] * np.uint64(0xCD9E8D57)
        w = [(b >> s) ^ w[1] ^ np.uint64(k[0]), b & lo, (a >> s) ^ w[3] ^ np.uint64(k[1]), a & lo]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    keep = torch.from_numpy(np.stack(w, 1).reshape(-1) >= np.uint64(1 << 31))
    assert torch.equal(tail, torch.where(keep, 2.0, 0.0).to(torch.bfloat16))


@gpu
def test_dropout_edges_strides_and_seed_tensors():
    x = torch.randn(6, 7, 33, device=DEV)
    x[0, 0, 0] = float("inf")
    x[1, 1, 1] = float("nan")
    assert torch.equal(wf.dropout(x, 0.0, 5).nan_to_num(9), x.nan_to_num(9))
    assert not wf.dropout(x, 1.0, 5).any()                          # exactly zero, infinities and NaN included
    y = wf.dropout(x, 0.6, 77)
    keep = torch.from_numpy(philox7(x.numel(), 77) >= np.uint64(int(0.6 * 2.0 ** 32))).reshape(x.shape)
    assert not y.cpu()[~keep].any()
    s = x.transpose(0, 2)
    assert torch.equal(wf.dropout(s, 0.6, 77).nan_to_num(9), wf.dropout(s.contiguous(), 0.6, 77).nan_to_num(9))
    t = torch.tensor([77], device=DEV)
    assert torch.equal(wf.dropout(x, 0.6, t).nan_to_num(9), y.nan_to_num(9))
    lx = torch.randn(64, device=DEV).requires_grad_()
    wf.dropout(lx, 0.25, t).sum().backward()                        # an expanded gradient, the seed read again
    assert torch.equal(lx.grad, wf.dropout(torch.ones(64, device=DEV), 0.25, 77))


@gpu
def test_row_operators_in_a_graph_take_the_seed_of_the_replay():
    x = torch.randn(50, 130, device=DEV)
    w, b = torch.randn(130, device=DEV), torch.randn(130, device=DEV)
    dy = torch.randn(50, 130, device=DEV)
    seed = torch.tensor([1], device=DEV)

    def step(leaves):
        y = wf.dropout(wf.layer_norm(*leaves), 0.3, seed)
        return (y,) + torch.autograd.grad(y, leaves, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        leaves = [t.clone().requires_grad_() for t in (x, w, b)]
        step(leaves)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(leaves)
    for k in range(4):
        seed.fill_(k * 1000 + 7)
        with torch.no_grad():
            leaves[0].copy_(x * (k + 1))
        graph.replay()
        torch.cuda.synchronize()
        want = step([t.detach().clone().requires_grad_() for t in leaves])
        for a, c in zip(out, want):
            assert torch.equal(a, c), k


def test_row_operators_refuse_what_they_cannot_do():
    x = torch.zeros(2, 8)
    with pytest.raises(_lib.WfError, match="GPU"):
        wf.layer_norm(x)
    with pytest.raises(_lib.WfError, match="GPU"):
        wf.dropout(x, 0.1, 1)
    with pytest.raises(TypeError):
        wf.layer_norm(x.double())
    with pytest.raises(TypeError):
        wf.dropout([1.0], 0.1, 1)
    lib = _lib.lib()       # the C entry points check sizes and types before anything is launched
    assert lib.wf_layer_norm(None, 8, 2, 8, 0, None, None, 0, 1e-5, None, None, None) == -1
    assert lib.wf_layer_norm(1, 8, 2, 40000, 0, None, None, 0, 1e-5, 1, None, None) == -5
    assert lib.wf_layer_norm(1, 8, 2, 0, 0, None, None, 0, 1e-5, 1, None, None) == -1
    assert lib.wf_layer_norm(1, 8, 2, 8, 7, None, None, 0, 1e-5, 1, None, None) == -1
    assert lib.wf_layer_norm(None, 8, 0, 8, 0, None, None, 0, 1e-5, None, None, None) == 0
    assert lib.wf_layer_norm_backward(1, 8, 1, 8, 2, 8, 0, None, 0, 1, 1, 1, 1, None, 0, None) == -2
    assert lib.wf_dropout(None, 8, 0, 0.5, 1, None, None, None) == -1
    assert lib.wf_dropout(1, 8, 0, 1.5, 1, None, 1, None) == -1
    assert lib.wf_dropout(1, 8, 0, float("nan"), 1, None, 1, None) == -1
    assert lib.wf_dropout(None, 0, 0, 0.5, 1, None, None, None) == 0


@gpu
def test_row_operators_refuse_mismatches():
    x = torch.zeros(2, 8, device=DEV)
    for bad in (dict(weight=torch.zeros(7, device=DEV)), dict(bias=torch.zeros(2, 8, device=DEV))):
        with pytest.raises(ValueError):
            wf.layer_norm(x, **bad)
    with pytest.raises(_lib.WfError):
        wf.layer_norm(x, torch.ones(8))
    with pytest.raises(TypeError):
        wf.layer_norm(x, torch.ones(8, device=DEV), torch.ones(8, device=DEV, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        wf.layer_norm(torch.zeros(1, 32769, device=DEV))
    with pytest.raises(ValueError):
        wf.layer_norm(torch.zeros(3, 0, device=DEV))
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError):
            wf.dropout(x, p, 1)
    with pytest.raises(TypeError):
        wf.dropout(x, 0.5, torch.zeros(2, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError):
        wf.dropout(x, 0.5, torch.zeros(1, dtype=torch.int64))
