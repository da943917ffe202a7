"""The output head's operators at the edges of what they promise.  Bounds as in test_head_linear.py: they count roundings."""
import pytest
import torch

import waterfall_amd as wf
from tests.test_head_linear import Case, check_grads, DEV, TYPES

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
