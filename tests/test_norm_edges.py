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


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape", [(1, 8193, 3, 5), (2, 16384, 2, 3), (1, 16384, 1, 2)])
def test_widest_maps(shape, dtype):
    """All channels that are accepted: two float32 sums a channel take 128 KiB of LDS."""
    both(*make(shape, 1, dtype, torch.float32, offset=40.0), 1)
    both(*make(shape, 1, dtype, dtype, offset=0.5), 1)


@gpu
@pytest.mark.parametrize("shape", [(1, 1100, 3, 9), (1, 16384, 3, 5), (2, 64, 1, 3)])
def test_sums_over_many_channels(shape):
    """Terms whose sum is rounded the same way again and again: from 2048 on a term of
    1 + 2^-13 - 2^-23 loses 2^-13 each time it is added by itself.  A lane that adds C / 4 terms in order is off by
    some 1000 u of the mean, past the bound of chain(C)."""
    term = 1 + 2.0 ** -13 - 2.0 ** -23
    g = torch.full(shape, term, device="cuda")
    x = torch.randn(shape, device="cuda")
    w = torch.ones(shape[1], device="cuda")
    for v in (x, g):
        y, mean, rstd = norm.layer_norm_forward(v, w, w, channel_dim=1)
        check_forward(v, w, w, 1e-5, 1, y, mean, rstd)
    y, mean, rstd = norm.layer_norm_forward(x, w, w, channel_dim=1)
    check_backward(x, w, g, mean, rstd, 1, *norm.layer_norm_backward(x, w, g, mean, rstd, 1))


EQUAL = [0.1, 15538.596, -1.0 / 3, 1e6 / 7, -3e-20]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("shape,dim", [((5, 96), -1), ((3, 777), -1), ((600, 64), -1), ((2, 3001), -1),
                                       ((2, 9001), -1), ((2, 16383), -1), ((2, 12, 3, 3), 1),
                                       ((1, 256, 10, 25), 1), ((1, 1000, 4, 33), 1), ((1, 1100, 3, 9), 1),
                                       ((2, 9001, 1, 3), 1)])
def test_equal_values_have_no_variance(shape, dim, dtype):
    """y is the bias and the mean the value itself, whatever the value: the sum of equal float32
    values is rounded, their mean is not.  The variance is the difference of two numbers below
    e^2, e = (chain + 4) u |x| the error of a first mean, each off by relative (chain + 4) u or twice
    that, so it is (3 chain + 12) u e^2 at most."""
    C = shape[dim]
    wide = [1] * len(shape)
    wide[dim] = C
    w, b = torch.rand(C, device="cuda") + 0.5, torch.randn(C, device="cuda")
    for value in EQUAL:
        x = torch.full(shape, value, device="cuda").to(dtype)
        if not torch.isfinite(x).all():                             # past float16
            continue
        y, mean, rstd = norm.layer_norm_forward(x, w, b, channel_dim=dim)
        exact = x.flatten()[0].float()
        assert (mean == exact).all(), value
        assert torch.equal(y, b.to(dtype).reshape(wide).expand(shape)), value
        k = chain(C)
        var = (3 * k + 12) * U * ((k + 4) * U * float(exact)) ** 2
        assert ((rstd.double() / 1e-5 ** -0.5 - 1).abs() <= 4 * U + var / 1e-5).all(), value


@gpu
@pytest.mark.parametrize("shape,dim", [((40, 320), -1), ((9, 5000), -1), ((3, 40, 9, 7), 1),
                                       ((1, 1100, 3, 9), 1)])
def test_mean_of_values_far_from_zero(shape, dim):
    """Values around 3e5 that differ by about one: the mean is off by a rounding, not by one a term."""
    x, w, b, _ = make(shape, dim, torch.float32, torch.float32, offset=3e5)
    y, mean, rstd = norm.layer_norm_forward(x, w, b, channel_dim=dim)
    check_forward(x, w, b, 1e-5, dim, y, mean, rstd)
    X = as_rows(x, dim)
    off = (mean.double() - X.mean(1)).abs()
    assert (off <= 2 * U * X.abs().amax(1)).all()


@gpu
def test_mean_of_values_around_zero():
    """A sum of C independent values of deviation 1 goes through some 16 levels of partial sums; the C / n sums
    of n values of a level are each off by a rounding of sqrt(n), u sqrt(n) at most and independent, so a level
    adds u sqrt(C) to the deviation of the sum: the mean's is u sqrt(16 / C) at most."""
    C = 4096
    x = make((2000, C), -1, torch.float32, torch.float32, offset=0.0)[0] / 1.3
    mean = norm.layer_norm_forward(x)[1]
    assert float((mean.double() - x.double().mean(1)).abs().mean()) <= U * (16 / C) ** 0.5


@gpu
@pytest.mark.parametrize("shape,dim", [((5, 96), -1), ((2, 3001), -1), ((2, 12, 3, 3), 1),
                                       ((1, 1100, 3, 9), 1)])
def test_values_whose_squares_overflow(shape, dim):
    """A deviation past the largest root counts as infinite, and y is the bias: also where the rounding of
    a mean is such a deviation."""
    C = shape[dim]
    wide = [1] * len(shape)
    wide[dim] = C
    w, b = torch.rand(C, device="cuda") + 0.5, torch.randn(C, device="cuda")
    for x in (torch.full(shape, 1.1e30, device="cuda"), torch.full(shape, 1.3e34, device="cuda"),
              torch.randn(shape, device="cuda") * 1e25, torch.randn(shape, device="cuda") * 1e25 + 1e32):
        y = norm.layer_norm_forward(x, w, b, channel_dim=dim)[0]
        assert torch.equal(y, b.reshape(wide).expand(shape))
