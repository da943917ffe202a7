"""The output head's operators at the edges of what they promise.  Bounds as in test_head_linear.py: they count roundings.

float16 gradients of logits are stored relative to a power of two: what `Case.products` takes as its last argument.  Log-probabilities:
with B the largest of max |G| and |sum(G)| over the rows, B is 2^13 to 2^14 of it, so it is at most 2^-13 B.  Cross entropy without
label smoothing: the largest incoming gradient is 2^14 of it."""
import ctypes as C

import pytest
import torch

import waterfall_amd as wf
from waterfall_amd import _lib
from tests import util
from tests.test_head_linear import Case, check_grads, dz_of_entropy, dz_of_log_softmax, DEV, TYPES
from tests.test_head_rows import norm64, U, within

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", [(40, 64, 50), (40, 64, 130), (5, 33, 1000), (3, 64, 5001), (40, 64, 20000), (300, 1031, 6007), (700, 80, 17000), (257, 96, 40)])
def test_rows_whose_every_output_is_masked_have_no_gradient(N, D, V, dtype):
    c = Case(N, D, V, dtype)
    G = torch.randn(N, V, generator=c.g).to(DEV)
    gone = torch.full((V,), float("-inf"), device=DEV, dtype=dtype)
    a = [v.detach().requires_grad_() for v in (c.x, c.w, gone)]
    lp = wf.linear_log_softmax(*a)
    assert (lp == float("-inf")).all()
    ce = wf.linear_cross_entropy(a[0], a[1], c.t, a[2], reduction="none")
    for got in (torch.autograd.grad(lp, a, G), torch.autograd.grad(ce, a, G[:, 0].contiguous())):
        for g, what in zip(got, ("dx", "dweight", "dbias")):
            assert not g.any(), what
    # one output left, the last: probability 1, and every other output's gradient is what comes in
    gone[-1] = 0
    a = [v.detach().requires_grad_() for v in (c.x, c.w, gone)]
    got = torch.autograd.grad(wf.linear_log_softmax(*a), a, G)
    with torch.no_grad():
        dz = G.double()
        s, size = dz.sum(1), dz.abs().sum(1, keepdim=True)
        dz[:, -1] -= s
        check_grads(got, c.products(dz, (V / 256 + 20) * 2.0 ** -24 * size * torch.nn.functional.one_hot(torch.tensor(V - 1, device=DEV), V) + 3 * 2.0 ** -24 * dz.abs(),
                                    2 * size.max().item()), (N, D, V))


@gpu
@pytest.mark.parametrize("N,D", [(4, 64), (300, 64)])
def test_half_precision_gradients_of_a_confident_row_and_a_gradient_that_sums_up(N, D):
    V = 262144
    c = Case(N, D, V, torch.float16)
    with torch.no_grad():
        c.b[7] = 40.0
    a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    G = torch.full((N, V), 1.0 / V, device=DEV)
    got = torch.autograd.grad(wf.linear_log_softmax(*a), a, G)
    with torch.no_grad():
        check_grads(got, c.products(*dz_of_log_softmax(c, G), 2.0 ** -13), (N, D, V))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", [(40, 64, 59), (40, 64, 700), (300, 1031, 6007)])
@pytest.mark.parametrize("eps", [0.5, 0.9, 0.996, 0.999, 0.99999, 1 - 2.0 ** -24])
def test_label_smoothing_just_under_one(N, D, V, eps, dtype):
    c = Case(N, D, V, dtype)
    with torch.no_grad():
        c.b[3] = 30.0                                       # probabilities near 1
    a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    up = torch.randn(N, generator=c.g).to(DEV)
    got = torch.autograd.grad(wf.linear_cross_entropy(a[0], a[1], c.t, a[2], label_smoothing=eps, reduction="none"), a, up)
    with torch.no_grad():
        check_grads(got, c.products(*dz_of_entropy(c, up, eps), 2 * up.abs().max().item()), (N, D, V, eps))


@gpu
@pytest.mark.parametrize("N,D,V", [(40, 64, 59), (40, 64, 700), (300, 1031, 6007), (700, 640, 5001)])
def test_half_precision_rows_of_unlike_weight(N, D, V):
    c = Case(N, D, V, torch.float16)
    up = (10.0 ** -(torch.arange(N) % 7).float()).to(DEV)
    a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    got = torch.autograd.grad(wf.linear_cross_entropy(a[0], a[1], c.t, a[2], reduction="none"), a, up)
    with torch.no_grad():
        check_grads(got, c.products(*dz_of_entropy(c, up, 0.0), 2.0 ** -14), (N, D, V))
        G = torch.randn(N, V, generator=c.g).to(DEV) * up[:, None]
        most = torch.maximum(G.abs().amax(1), G.sum(1).abs()).max().item()
    got = torch.autograd.grad(wf.linear_log_softmax(*a), a, G)
    with torch.no_grad():
        check_grads(got, c.products(*dz_of_log_softmax(c, G), most * 2.0 ** -13), (N, D, V))


@gpu
@pytest.mark.parametrize("N,D,V", [(40, 64, 59), (40, 64, 700), (3000, 257, 4099)])
def test_half_precision_rows_beside_one_whose_gradient_is_not_finite(N, D, V):
    c = Case(N, D, V, torch.float16)
    up = torch.full((N,), 1e-6, device=DEV)
    up[2] = float("inf")
    up[5] = float("nan")
    rows = torch.ones(N, dtype=torch.bool, device=DEV)
    rows[[2, 5]] = False
    a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    few = Case(N, D, V, torch.float16)
    few.x, few.t = c.x[rows], c.t[rows]
    dx, = torch.autograd.grad(wf.linear_cross_entropy(a[0], a[1], c.t, a[2], reduction="none"), a[:1], up)
    with torch.no_grad():
        check_grads((dx[rows],), few.products(*dz_of_entropy(few, up[rows], 0.0), 1e-6 * 2.0 ** -14), (N, D, V))
        G = torch.randn(N, V, generator=c.g).to(DEV) * up[:, None]
        most = torch.maximum(G[rows].abs().amax(1), G[rows].sum(1).abs()).max().item()
    dx, = torch.autograd.grad(wf.linear_log_softmax(*a), a[:1], G)
    with torch.no_grad():
        check_grads((dx[rows],), few.products(*dz_of_log_softmax(few, G[rows]), most * 2.0 ** -13), (N, D, V))


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [63, 512, 1500, 3000, 5000, 8200, 20000])
def test_layer_norm_rows_without_a_gradient_may_hold_anything(D, dtype):
    g = torch.Generator().manual_seed(D)
    x, dy = torch.randn(37, D, generator=g).to(dtype).to(DEV), torch.randn(37, D, generator=g).to(dtype).to(DEV)
    w, b = torch.randn(D, generator=g).to(DEV), torch.randn(D, generator=g).to(DEV)
    dead = [0, 5, 6, 7, 20, 36]
    y = x.clone()
    y[dead] = float("nan")
    y[5] = float("inf")
    y[20] = x[20]
    y[20, D // 2] = float("-inf")
    dy[dead] = 0
    got = [torch.autograd.grad(wf.layer_norm(*a), a, dy) for a in ([t.detach().requires_grad_() for t in (v, w, b)] for v in (y, x))]
    for p, q, what in zip(*got, ("dx", "dweight", "dbias")):
        assert torch.equal(p, q), what                      # as if those rows were ordinary ones
    assert not got[0][0][dead].any()
    # one element of such a row that has a gradient: the row takes part, and nothing about it is hidden
    dy[5, D - 1] = 1
    a = [t.detach().requires_grad_() for t in (y, w, b)]
    dx, dw, _ = torch.autograd.grad(wf.layer_norm(*a), a, dy)
    assert torch.isnan(dx[5]).all() and torch.isnan(dw[D - 1])


@gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_frames_behind_the_end_may_hold_anything_on_the_way_through_the_head(dtype):
    torch.manual_seed(4)
    head = wf.OutputHead(96, 58, dropout=0.2, device=DEV)
    x = torch.randn(4, 30, 96, device=DEV).to(dtype)
    length = torch.tensor([30, 21, 17, 5], device=DEV)
    there = torch.arange(30, device=DEV) < length[:, None]
    t = torch.where(there, torch.randint(0, 58, (4, 30), device=DEV), -1)
    G = torch.randn(4, 30, 58, device=DEV) * there[..., None]
    params = list(head.parameters())
    got = []
    for v in (x, torch.where(there[..., None], x, float("nan"))):
        leaf = v.clone().requires_grad_()
        torch.manual_seed(9)
        lp = head(leaf)
        a = torch.autograd.grad(lp, [leaf] + params, G)
        torch.manual_seed(9)
        got.append(a + torch.autograd.grad(head.cross_entropy(leaf, t), [leaf] + params))
    for p, q in zip(*got):
        assert torch.equal(p, q)


@gpu
def test_saved_tensors_that_come_back_in_another_shape():
    """As many elements in other rows: an error on the host before anything is launched, whichever saved tensor it is."""
    x, w, b = torch.randn(2, 4, 64, device=DEV, requires_grad=True), torch.randn(50, 64, device=DEV, requires_grad=True), torch.randn(50, device=DEV, requires_grad=True)
    t, g = torch.randint(0, 50, (2, 4), device=DEV), torch.ones(64, device=DEV, requires_grad=True)
    calls = ((3, lambda: wf.layer_norm(x, g)), (4, lambda: wf.linear_log_softmax(x, w, b)), (5, lambda: wf.linear_cross_entropy(x, w, t, b)),
             (5, lambda: wf.linear_cross_entropy(x, w, t, b, reduction="none")))
    shapes = (lambda v: v.reshape(-1), lambda v: v.reshape(-1, 1), lambda v: v.transpose(0, -1), lambda v: v.reshape(2, -1), lambda v: v.reshape((-1,) + v.shape[2:]),
              lambda v: v[None])
    for saved, call in calls:
        for k in range(saved):
            for other in shapes:
                seen = []

                def unpack(v):
                    seen.append(v)
                    return other(v) if len(seen) == k + 1 else v

                with torch.autograd.graph.saved_tensors_hooks(lambda v: v, unpack):
                    y = call()
                changed = False
                try:
                    y.sum().backward()
                except RuntimeError as e:
                    assert "came back" in str(e), e
                    changed = True
                assert len(seen) == saved and changed == (other(seen[k]).shape != seen[k].shape), (saved, k)
    seed = torch.tensor([3], device=DEV)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v, lambda v: v.reshape(())):       # one element in any shape
        y = wf.dropout(x, 0.5, seed)
    assert torch.equal(torch.autograd.grad(y.sum(), x)[0], wf.dropout(torch.ones_like(x), 0.5, 3))


def test_sizes_that_no_launch_takes_are_refused():
    lib, n = _lib.lib(), C.c_size_t(0)
    for what, N, D, V, t, rc in ((1, 63 << 22, 8, 3, 1, 0), (1, (63 << 22) + 1, 8, 3, 1, -5), (0, 1 << 28, 8, 3, 0, -5), (2, 1 << 20, 64, 1 << 17, 1, 0),
                                 (2, 1 << 22, 64, 1 << 20, 1, -5), (3, 1 << 22, 64, 1 << 20, 1, 0), (3, 1 << 27, 1 << 20, 300, 1, -5)):
        assert lib.wf_linear_workspace_bytes(what, N, D, V, t, C.byref(n)) == rc, (what, N, D, V, t)


@gpu
def test_gradients_of_more_rows_than_one_launch_takes():
    N, D, V = (1 << 26) + 70, 2, 3                          # a wave a row: more than 2^32 threads
    if torch.cuda.mem_get_info(0)[0] < 100 << 30:
        pytest.skip("needs 70 GB")
    c = Case(2, D, V, torch.bfloat16)
    c.N = N
    g = torch.Generator(device=DEV).manual_seed(3)
    c.x = torch.randn(N, D, generator=g, device=DEV).bfloat16()
    G = torch.randn(N, V, generator=g, device=DEV)
    G[torch.rand(N, generator=g, device=DEV) < 0.3] = 0
    a = [v.detach().requires_grad_() for v in (c.x, c.w, c.b)]
    got = torch.autograd.grad(wf.linear_log_softmax(*a), a, G)
    with torch.no_grad():
        check_grads(got, c.products(*dz_of_log_softmax(c, G)), (N, D, V))


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_capture_while_an_eager_graph_of_the_same_leaves_is_alive_is_refused(dtype):
    head = wf.OutputHead(64, 200, device=DEV)
    x, t = torch.randn(40, 64, device=DEV).to(dtype), torch.randint(0, 200, (40,), device=DEV)
    params = list(head.parameters())

    def step():
        return torch.autograd.grad(head.cross_entropy(x, t), params)

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

    alive = head.cross_entropy(x, t)                        # made on the default stream, as the leaves' accumulators are
    with pytest.raises(RuntimeError, match="eager graph of the same leaves"):
        capture()
    want = torch.autograd.grad(alive, params)               # everything else goes on
    del alive
    graph, out = capture()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        for p, q, r in zip(out, want, step()):
            assert torch.equal(p, q) and torch.equal(p, r)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 1025), (37, 1280), (300, 1536), (2, 2047), (9, 2048), (1, 4099), (270, 6001), (3, 8191), (5, 12007), (2, 30001)])
def test_layer_norm_of_wide_rows(shape, dtype):
    """Every way of sharing a row that test_head_rows.py has no length of: the last piece whole, of one element, of all but one."""
    g = torch.Generator().manual_seed(shape[1])
    D = shape[-1]
    x = (torch.randn(shape, generator=g) * 1.5 + 0.7).to(dtype)
    w, b = (torch.randn(D, generator=g) + 1).to(dtype), torch.randn(D, generator=g).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    leaves = [v.to(DEV).requires_grad_() for v in (x, w, b)]
    y = wf.layer_norm(*leaves)
    got = torch.autograd.grad(y, leaves, dy.to(DEV))
    want, dx, dw, db, adw, adb, r, gw, h = norm64(x, w, b, 1e-5, dy)
    u, f = U[dtype], 32 * U[torch.float32]                  # (bounds of test_head_rows.py: sums of 32 elements a lane are as deep)
    big = x.double().abs().amax(-1, keepdim=True)
    within(y.detach(), want, u * want.abs() + f * ((big * r + h.abs()) * w.double().abs() + want.abs()) + 1e-30, "y")
    size = r * (gw.abs() + gw.abs().mean(-1, keepdim=True) + (h.abs() + big * r) * (1 + (gw * h).abs().mean(-1, keepdim=True) + gw.abs().amax(-1, keepdim=True)))
    within(got[0], dx, u * dx.abs() + f * size, "dx")
    within(got[1], dw, u * dw.abs() + f * (1 + shape[0] / 4096) * (adw + (dy.double().abs() * big * r).sum(0)), "dweight")
    within(got[2], db, u * db.abs() + f * (1 + shape[0] / 4096) * adb, "dbias")


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_graph_loss_through_the_head_on_a_batch_padded_with_anything(dtype):
    c = util.random_case(77, "ctc", B=4, T=30, L=5, P=58)
    B, T, V = c["lp"].shape
    torch.manual_seed(3)
    head = wf.OutputHead(96, V, dropout=0.2, device=DEV)
    segs = torch.from_numpy(c["segs"])
    there = torch.arange(T, device=DEV)[None, :] < segs[:, 2].to(DEV)[:, None]
    assert not there.all()
    enc = torch.randn(B, T, 96, device=DEV).to(dtype)
    got = []
    for v in (enc, torch.where(there[..., None], enc, float("nan"))):
        x = v.clone().requires_grad_()
        torch.manual_seed(5)
        loss = wf.graphloss(c["fsa"], wf.DenseFsaVec(head(x), segs), reduction="sum")
        got.append((loss.detach(),) + torch.autograd.grad(loss, [x] + list(head.parameters())))
    for p, q in zip(*got):
        assert torch.equal(p, q) and torch.isfinite(p).all()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_row_without_leading_dimensions(dtype):
    x, w = torch.randn(64, device=DEV).to(dtype).requires_grad_(), torch.randn(40, 64, device=DEV).to(dtype).requires_grad_()
    b, t = torch.randn(40, device=DEV, requires_grad=True), torch.tensor(7, device=DEV)
    for reduction in ("mean", "sum", "none"):
        loss = wf.linear_cross_entropy(x, w, t, b, reduction=reduction)
        assert loss.shape == ()
        rows = wf.linear_cross_entropy(x[None], w, t[None], b, reduction=reduction).sum()
        for p, q in zip(torch.autograd.grad(loss, (x, w, b)), torch.autograd.grad(rows, (x, w, b))):
            assert torch.equal(p, q)
    lp = wf.linear_log_softmax(x, w, b)
    assert lp.shape == (40,) and torch.equal(lp, wf.linear_log_softmax(x[None], w, b)[0])
    assert torch.equal(wf.layer_norm(x), wf.layer_norm(x[None])[0])
    assert torch.autograd.grad(wf.layer_norm(x).sum() + lp.sum() + wf.dropout(x, 0.5, 3).sum(), x)[0].shape == (64,)


@gpu
def test_the_head_under_checkpointing_and_in_inference_mode():
    from torch.utils.checkpoint import checkpoint
    head = wf.OutputHead(64, 40, dropout=0.3, device=DEV)
    x = torch.randn(4, 64, device=DEV, requires_grad=True)
    torch.manual_seed(1)
    want = torch.autograd.grad(head(x).square().sum(), x)[0]
    for reentrant in (False, True):
        torch.manual_seed(1)
        checkpoint(head, x, use_reentrant=reentrant).square().sum().backward()
        assert torch.equal(x.grad, want)
        x.grad = None
    head.eval()
    lp = head(x).detach()
    with torch.inference_mode():
        assert torch.equal(head(x), lp)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", [(40, 64, 59), (300, 257, 700), (2100, 641, 5003), (5000, 64, 131)])
def test_leaves_of_which_only_one_wants_a_gradient(N, D, V, dtype):
    c = Case(N, D, V, dtype)
    c.t[::5] = -1
    G = torch.randn(N, V, generator=c.g).to(DEV)
    G[3::7] = 0
    calls = (lambda x, w, b: torch.autograd.grad(wf.linear_log_softmax(x, w, b), [v for v in (x, w, b) if v.requires_grad], G),
             lambda x, w, b: torch.autograd.grad(wf.linear_cross_entropy(x, w, c.t, b, label_smoothing=0.1), [v for v in (x, w, b) if v.requires_grad]))
    for call in calls:
        whole = call(*[v.detach().requires_grad_() for v in (c.x, c.w, c.b)])
        for wants in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
            got = call(*[v.detach().requires_grad_(k in wants) for k, v in enumerate((c.x, c.w, c.b))])
            for k, g in zip(wants, got):
                assert torch.equal(g, whole[k]), (wants, k)
    # the row operators: one of x, weight, bias
    y = [torch.randn(37, 300, generator=c.g).to(dtype).to(DEV), torch.randn(300, device=DEV), torch.randn(300, device=DEV)]
    dy = torch.randn(37, 300, generator=c.g).to(dtype).to(DEV)
    a = [v.clone().requires_grad_() for v in y]
    whole = torch.autograd.grad(wf.layer_norm(*a), a, dy)
    for k in range(3):
        a = [v.clone().requires_grad_(i == k) for i, v in enumerate(y)]
        assert torch.equal(torch.autograd.grad(wf.layer_norm(*a), a[k], dy)[0], whole[k]), k


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", [64, 1500, 3000, 9000])
def test_layer_norm_rows_without_a_gradient_at_the_ends_of_the_type(D, dtype):
    g = torch.Generator().manual_seed(D)
    x, dy = torch.randn(9, D, generator=g).to(dtype).to(DEV), torch.randn(9, D, generator=g).to(dtype).to(DEV)
    w, b = torch.randn(D, generator=g).to(DEV), torch.randn(D, generator=g).to(DEV)
    dead = [1, 4]
    dy[dead] = 0
    y = x.clone()
    most = torch.finfo(dtype).max                           # the mean is finite, and the first element's distance from it is not
    y[dead] = 0
    y[dead[0], :3] = y[dead[1], :3] = torch.tensor([-most, most, 0.99 * most], device=DEV).to(dtype)
    got = [torch.autograd.grad(wf.layer_norm(*a), a, dy) for a in ([t.detach().requires_grad_() for t in (v, w, b)] for v in (y, x))]
    for p, q in zip(*got):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,D,V", [(40, 64, 59), (300, 257, 700), (2100, 641, 5003)])
def test_rows_of_cross_entropy_without_an_incoming_gradient_may_hold_anything(N, D, V, dtype):
    c = Case(N, D, V, dtype)
    c.t[1::6] = -1
    c.t[3] = V + 5                                          # no output: a loss of NaN, no gradient
    up = torch.randn(N, generator=c.g).to(DEV)
    dead = torch.zeros(N, dtype=torch.bool, device=DEV)
    dead[2::5] = True
    dead[3] = True
    up[dead] = 0
    x = c.x.clone()
    x[dead] = float("nan")
    a = [v.detach().requires_grad_() for v in (x, c.w, c.b)]
    got = torch.autograd.grad(wf.linear_cross_entropy(a[0], a[1], c.t, a[2], label_smoothing=0.1, reduction="none"), a, up)
    assert not got[0][dead].any()
    with torch.no_grad():
        check_grads(got, c.products(*dz_of_entropy(c, up, 0.1), 2 * up.abs().max().item()), (N, D, V))
