"""Calls of the optimizer that earlier tests did not make: states over steps that overflow, parameters
without a gradient in some steps, several groups, states from elsewhere, refused steps.  Tolerances are
those of test_optim.py."""
import pytest
import torch

from ganet_amd import _lib, optim
from test_optim import BLOCK, HYPER, U, check32, gpu


@gpu
@pytest.mark.parametrize("dtype,master", [(torch.float32, False), (torch.bfloat16, True),
                                          (torch.bfloat16, False)])
def test_a_square_past_the_largest_float_stops_its_weight_only(dtype, master):
    """A finite gradient whose square is not: as with float32 moments, its second moment stays
    infinite, so its weight stands still from then on (and does not become NaN in the next step);
    the other values of its block get the bits that they get without it.  The block's largest values
    are elsewhere, so that the scales have to be equal too."""
    n, at = 600, [100, 300, 599]
    runs = []
    for spoilt in (True, False):
        p = torch.ones(n, device="cuda", dtype=dtype)
        w = [p.float()] if master else None
        st = optim.state_8bit(p)
        m32, v32 = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
        q, seen = p.float().clone(), []
        for t in range(1, 7):
            g = torch.full((n,), 1e-3, device="cuda")
            g[::128] = 4e-3
            g[at] = 0.0
            if spoilt:
                g[at] = torch.tensor([1e20, -3e38, 2e19] if t == 2 else [1e-3, -1e-3, 0.0], device="cuda")
            g = g.to(dtype)
            kw = dict(lr=1e-2, weight_decay=0.0)
            optim.adamw_step_8bit([p], [g], [st[0]], [st[1]], [st[2]], [st[3]], t, seed=5, masters=w, **kw)
            if spoilt:
                before = q.clone()
                optim.adamw_step([q], [g.float()], [m32], [v32], t, **kw)
                if t >= 2:
                    assert torch.equal(q[at], before[at])          # what float32 moments do
            seen.append([x.clone() for x in (p, *(w or []), *(s.view(torch.uint8) for s in st[:2]), *st[2:])])
        runs.append(seen)
    rest = torch.ones(n, dtype=torch.bool, device="cuda")
    rest[at] = False
    for t, (one, two) in enumerate(zip(*runs)):
        for a, b in zip(one, two):
            if a.numel() == n:
                a, b = a[rest], b[rest]
            assert torch.equal(a, b), t
        if t >= 1:                                                 # from the second step on
            assert torch.equal(one[0][at], runs[0][0][0][at]) and torch.isfinite(one[0]).all()
