"""Calls of layer norm that earlier tests did not make: rows of equal values that float32 sums do not
hold exactly, the widest maps, evaluation.  Tolerances are those of test_norm.py."""
import pytest
import torch

from ganet_amd import norm
from test_norm import DTYPES, U, as_rows, both, chain, check_backward, check_forward, gpu, make


def test_statistics_only_for_a_backward(monkeypatch):
    """Mean and rstd are written where a backward pass can follow, not in evaluation."""
    asked = []

    def forward(input, weight, bias, eps, channel_dim, stats):
        asked.append(bool(stats))
        one = torch.zeros(1) if stats else None
        return input * 1, one, one

    monkeypatch.setattr(norm, "_forward", forward)
    m, x = norm.LayerNorm(8), torch.zeros(2, 8)
    m(x)
    with torch.no_grad():
        assert not m(x).requires_grad
    with torch.inference_mode():
        m(x)
    m.requires_grad_(False)
    assert not m(x).requires_grad
    m(x.clone().requires_grad_())
    assert asked == [True, False, False, False, True]
    with torch.autograd.forward_ad.dual_level():                    # no derivative is lost in silence
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises((RuntimeError, NotImplementedError), match="jvp"):
            m(dual)


@gpu
def test_evaluation_gives_the_same_values():
    m, x = norm.LayerNorm2d(24).cuda(), torch.randn(2, 24, 5, 9, device="cuda")
    y = m(x)
    with torch.no_grad():
        z = m(x)
    with torch.inference_mode():
        i = m(x)
    assert y.requires_grad and not z.requires_grad and not i.requires_grad
    assert torch.equal(y, z) and torch.equal(y, i)
    m.requires_grad_(False)
    assert not m(x).requires_grad and torch.equal(m(x), y)
