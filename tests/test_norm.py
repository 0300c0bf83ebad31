"""Layer norm over channels (ganet_amd.norm) against its formula in 64 bits.

Tolerances, element by element, with u = 2^-24 (a float32 rounding) and h = half a step of the
output's type.  A float32 sum of n terms, added as the kernels do (a lane's own terms in order, at
most ceil(n / 64) of them, then a tree), is off by at most k u times the sum of its terms'
magnitudes, k = ceil(n / 64) + 12.  Forward: the mean is off by k u max|x|, the variance by
relative k u and less, so y = xh w + b by (k + 16) u (|w| rstd max|x| + |xh w| + |b|), and h |y| for its
rounding.  Backward with mean and rstd given: xh is off by e = 2 u ((|x| + |mean|) rstd + |xh|); with
a = w dy, grad_x = rstd (a - mean(a) - xh mean(a xh)) follows by adding each part's error."""
import ctypes

import pytest
import torch

from ganet_amd import _lib, norm

U = 2.0 ** -24
HALF = {t: torch.finfo(t).eps / 2 for t in (torch.float32, torch.bfloat16, torch.float16)}
gpu = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def chain(n):
    return -(-n // 64) + 12


def as_rows(t, dim):
    """[positions, C] in 64 bits; positions in row-major order of the other dimensions."""
    t = t.detach().double().movedim(dim, -1)
    return t.reshape(-1, t.shape[-1])


def check_forward(x, w, b, eps, dim, y, mean, rstd):
    X, Y = as_rows(x, dim), as_rows(y, dim)
    C = X.shape[1]
    W = w.double() if w is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    Bv = b.double() if b is not None else torch.zeros_like(W)
    mu = X.mean(1, keepdim=True)
    var = ((X - mu) ** 2).mean(1, keepdim=True)
    rs = 1 / torch.sqrt(var + eps)
    xh = (X - mu) * rs
    ref = xh * W + Bv
    k, top = chain(C), X.abs().amax(1, keepdim=True)
    tol = HALF[y.dtype] * ref.abs() + (k + 16) * U * (W.abs() * rs * top + (xh * W).abs() + Bv.abs())
    tiny = torch.finfo(y.dtype).smallest_normal * torch.finfo(y.dtype).eps
    assert y.dtype == x.dtype and y.shape == x.shape
    assert ((Y - ref).abs() <= tol + tiny).all(), float(((Y - ref).abs() / (tol + tiny)).max())
    assert ((mean.double() - mu[:, 0]).abs() <= k * U * top[:, 0]).all()
    # the variance also takes up the square of the mean's error
    rel = (k + 8) * U + (k * U * top * rs) ** 2
    assert ((rstd.double() / rs[:, 0] - 1).abs() <= rel[:, 0]).all()


def check_backward(x, w, g, mean, rstd, dim, gx, gw, gb):
    X, G = as_rows(x, dim), as_rows(g, dim)
    N, C = X.shape
    W = w.double() if w is not None else torch.ones(C, dtype=torch.float64, device=x.device)
    mu, rs = mean.double()[:, None], rstd.double()[:, None]
    xh = (X - mu) * rs
    e = 2 * U * ((X.abs() + mu.abs()) * rs + xh.abs())
    a = G * W
    ref = rs * (a - a.mean(1, keepdim=True) - xh * (a * xh).mean(1, keepdim=True))
    if gx is not None:
        k = chain(C) + 8
        ax = (a * xh).abs().mean(1, keepdim=True)
        tol = rs * (k * U * (a.abs() + a.abs().mean(1, keepdim=True) + xh.abs() * ax)
                    + e * ax + xh.abs() * (a.abs() * e).mean(1, keepdim=True))
        tol = tol + HALF[gx.dtype] * ref.abs()
        tiny = torch.finfo(gx.dtype).smallest_normal * torch.finfo(gx.dtype).eps
        err = (as_rows(gx, dim) - ref).abs()
        assert gx.dtype == x.dtype and gx.shape == x.shape
        assert (err <= tol + tiny).all(), float((err / (tol + tiny)).max())
    k = chain(N) + 64
    for got, terms, more in ((gw, G * xh, (G.abs() * e).sum(0)), (gb, G, 0.0)):
        if got is None:
            continue
        ref = terms.sum(0)
        tol = HALF[got.dtype] * ref.abs() + k * U * terms.abs().sum(0) + more
        tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
        assert got.shape == (C,)
        assert ((got.double() - ref).abs() <= tol + tiny).all()


def make(shape, dim, dtype, wdtype, seed=0, offset=0.5):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(s):
        return torch.randn(s, generator=gen, device="cuda")

    C = shape[dim]
    x = (normal(shape) * 1.3 + offset).to(dtype)
    return (x, (normal((C,)) * 0.3 + 1).to(wdtype), (normal((C,)) * 0.3).to(wdtype),
            normal(shape).to(dtype))


def both(x, w, b, g, dim, eps=1e-5):
    y, mean, rstd = norm.layer_norm_forward(x, w, b, eps, dim)
    check_forward(x, w, b, eps, dim, y, mean, rstd)
    gx, gw, gb = norm.layer_norm_backward(x, w, g, mean, rstd, dim)
    check_backward(x, w, g, mean, rstd, dim, gx, gw, gb)
    return y, gx, gw, gb


# ------------------------------------------------------------------------------- without a GPU
def test_refusals_without_gpu():
    with pytest.raises(NotImplementedError):
        norm.layer_norm(torch.zeros(2, 8))
    with pytest.raises(NotImplementedError):
        norm.LayerNorm2d(8)(torch.zeros(2, 8, 3, 3))
    with pytest.raises(ValueError):
        norm.LayerNorm2d(8)(torch.zeros(2, 9, 3, 3))
    with pytest.raises(IndexError):
        norm.layer_norm(torch.zeros(2, 8), channel_dim=2)
    with pytest.raises(ValueError):
        norm.layer_norm(torch.zeros(2, 0))


def test_c_abi_refusals_without_gpu():
    L = _lib.lib()
    fake = ctypes.c_void_p(256)

    def params(**kw):
        p = _lib.LayerNormParams(outer=4, inner=1, x_stride=8, y_stride=8, g_stride=8, C=8, dtype=0,
                                 weight_dtype=0, eps=1e-5)
        for k, v in kw.items():
            setattr(p, k, v)
        return p

    def fwd(p, x=fake, y=fake, mean=fake, rstd=fake):
        return L.ganet_layer_norm_forward(x, fake, fake, y, mean, rstd, ctypes.byref(p), None)

    def bwd(p, ws=fake, nbytes=1 << 30, outs=(fake, fake, fake)):
        return L.ganet_layer_norm_backward(fake, fake, fake, fake, fake, *outs, ctypes.byref(p), ws,
                                           nbytes, None)

    for kw, code in [(dict(C=0), _lib.GANET_ERR_BAD_SHAPE), (dict(outer=-1), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(inner=0), _lib.GANET_ERR_BAD_SHAPE), (dict(dtype=3), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(weight_dtype=-1), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(eps=-1.0), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(eps=float("nan")), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(x_stride=7), _lib.GANET_ERR_BAD_SHAPE), (dict(y_stride=7), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(inner=3), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(outer=1 << 62), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(inner=1 << 62), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(x_stride=1 << 62), _lib.GANET_ERR_BAD_SHAPE),
                     (dict(C=_lib.GANET_LAYER_NORM_MAX_C + 1), _lib.GANET_ERR_UNSUPPORTED)]:
        assert fwd(params(**kw)) == code, kw
        assert bwd(params(**kw)) == code, kw
        assert L.ganet_layer_norm_backward_workspace_bytes(ctypes.byref(params(**kw))) == 0
    assert bwd(params(g_stride=7)) == _lib.GANET_ERR_BAD_SHAPE
    assert fwd(params(), x=None) == _lib.GANET_ERR_NULL
    assert fwd(params(), mean=None) == _lib.GANET_ERR_NULL
    assert fwd(params(outer=0), x=None, y=None) == _lib.GANET_OK
    assert bwd(params(), ws=None) == _lib.GANET_ERR_NULL
    assert bwd(params(), nbytes=16) == _lib.GANET_ERR_WORKSPACE
    assert bwd(params(), outs=(None, None, None)) == _lib.GANET_ERR_NULL


def test_rows_stride():
    t = torch.zeros(6, 5, 16)
    assert norm._rows_stride(t) == 16
    assert norm._rows_stride(t[:, :, :10]) == 16
    assert norm._rows_stride(t[:, 2]) == 80
    assert norm._rows_stride(t[:, :3]) is None          # rows not evenly spaced
    assert norm._rows_stride(t[..., ::2]) is None
    assert norm._rows_stride(torch.zeros(1, 16).expand(4, 16)) is None
    assert norm._rows_stride(torch.zeros(16)) == 16


# ------------------------------------------------------------------------------- on the GPU
ROWS = [(1, 1), (3, 1), (1, 7), (5, 3), (70, 8), (33, 64), (9, 100), (250, 256), (17, 257),
        (65, 511), (4, 1000), (777, 1001), (6, 2048), (3, 2049), (5, 4096), (2, 5000), (2, 8192),
        (3, 16384)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("n,c", ROWS)
def test_rows(n, c, dtype):
    both(*make((n, c), -1, dtype, dtype), -1)
    both(*make((n, c), -1, dtype, torch.float32, seed=1), -1)


MAPS = [(1, 1, 3, 5), (2, 3, 1, 1), (1, 64, 5, 7), (3, 5, 8, 25), (2, 256, 10, 25), (1, 33, 40, 100),
        (2, 129, 9, 13), (1, 512, 7, 11), (1, 600, 4, 33), (1, 1100, 3, 9), (1, 2048, 2, 5)]


@gpu
@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("channels_last", [False, True])
@pytest.mark.parametrize("shape", MAPS)
def test_maps(shape, channels_last, dtype):
    x, w, b, g = make(shape, 1, dtype, torch.float32)
    if channels_last:
        x = x.contiguous(memory_format=torch.channels_last)
    y, gx, _, _ = both(x, w, b, g, 1)
    for t in (y, gx):
        assert t.is_contiguous(memory_format=torch.channels_last) or not channels_last
        assert t.is_contiguous() or channels_last


@gpu
@pytest.mark.parametrize("c", [1, 7, 64, 100, 257, 511, 1001, 2048, 2049, 4096, 5000, 8192, 16384])
def test_more_rows(c):
    """Every width with enough rows for sums in the workspace."""
    for n in (512, 513, 1025):
        both(*make((n, c), -1, torch.float32, torch.float32), -1)
        both(*make((n, c), -1, torch.bfloat16, torch.float32), -1)


@gpu
@pytest.mark.parametrize("c", [1, 16, 33, 64, 129, 256, 257, 512, 600, 1024])
def test_more_positions(c):
    for shape in ((2, c, 97, 101), (8, c, 32, 64), (3, c, 9, 13)):      # past, at and below the limit
        if c * shape[0] * shape[2] * shape[3] < 6e6:
            both(*make(shape, 1, torch.float32, torch.float32), 1)
            both(*make(shape, 1, torch.float16, torch.float32), 1)


@gpu
@pytest.mark.parametrize("layout", ["rows", "nchw"])
def test_many_positions(layout):
    """More rows and tiles than the backward has workgroups."""
    if layout == "rows":
        both(*make((70001, 40), -1, torch.bfloat16, torch.bfloat16), -1)
    else:
        both(*make((9, 24, 97, 101), 1, torch.float16, torch.float32), 1)


@gpu
def test_other_strides_and_orders():
    dev = "cuda"
    wide = torch.randn(40, 300, device=dev)
    x, g = wide[:, 7:207], torch.randn(200, 40, device=dev).t()     # rows apart; transposed gradient
    w, b = torch.rand(400, device=dev)[::2], torch.rand(200, device=dev)
    both(x, w, b, g, -1)
    big = torch.randn(4, 30, 6, 7, device=dev)
    both(big[:, 3:23], w[:20], b[:20], torch.randn(4, 20, 6, 7, device=dev), 1)   # images apart
    both(big[1:3, ::2], w[:15], b[:15], torch.randn(2, 15, 6, 7, device=dev), 1)  # copied
    both(torch.randn(3, 5, 11, device=dev).expand(3, 5, 11), w[:5], b[:5],
         torch.ones(1, 1, 1, device=dev).expand(3, 5, 11), 1)                     # broadcast gradient
    both(torch.randn(6, 9, 2, 3, device=dev), w[:6], b[:6], torch.randn(6, 9, 2, 3, device=dev), 0)
    both(torch.randn(5, 33, device=dev), None, None, torch.randn(5, 33, device=dev), -1)
    flat = torch.randn(1 + 50 * 37, device=dev).bfloat16()
    both(flat[1:].view(50, 37), w[:37].bfloat16(), b[:37].bfloat16(), flat[:-1].view(50, 37), -1)


@gpu
def test_large_mean_and_constant_rows():
    x, w, b, g = make((40, 320), -1, torch.float32, torch.float32, offset=1000.0)
    both(x, w, b, g, -1)
    both(*make((3, 40, 9, 7), 1, torch.float32, torch.float32, offset=1000.0), 1)
    x = torch.full((7, 96), 3.25, device="cuda")                    # no variance: y is the bias
    y, mean, rstd = norm.layer_norm_forward(x, w[:96], b[:96])
    assert torch.equal(y, b[:96].expand(7, 96)) and (mean == 3.25).all()
    x = torch.full((2, 12, 3, 3), 3.25, device="cuda")
    y, mean, rstd = norm.layer_norm_forward(x, w[:12], b[:12], channel_dim=1)
    assert torch.equal(y, b[:12].reshape(1, 12, 1, 1).expand(2, 12, 3, 3))


@gpu
def test_non_finite_values_stay_in_their_position():
    for dim, shape in ((-1, (6, 50)), (1, (2, 50, 3, 1))):
        x, w, b, g = make(shape, dim, torch.float32, torch.float32)
        clean = norm.layer_norm_forward(x, w, b, channel_dim=dim)[0]
        bad = x.clone()
        bad[(2, 7) if dim == -1 else (0, 7, 2, 0)] = float("inf" if dim == -1 else "nan")
        y = as_rows(norm.layer_norm_forward(bad, w, b, channel_dim=dim)[0], dim)
        assert not torch.isfinite(y[2]).any()
        keep = [0, 1, 3, 4, 5]
        assert torch.equal(y[keep], as_rows(clean, dim)[keep])


@gpu
def test_nothing_in_it():
    w, b = torch.ones(8, device="cuda"), torch.zeros(8, device="cuda")
    for shape, dim in (((0, 8), -1), ((3, 8, 0, 4), 1), ((0, 8, 3, 4), 1)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        wp = w.clone().requires_grad_()
        y = norm.layer_norm(x, wp, b, channel_dim=dim)
        assert y.shape == shape
        y.sum().backward()
        assert (wp.grad == 0).all() and x.grad.shape == shape


@gpu
@pytest.mark.parametrize("need", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 0), (0, 1, 1)])
@pytest.mark.parametrize("shape,dim", [((37, 96), -1), ((2, 24, 5, 9), 1), ((3, 5000), -1),
                                       ((1, 1500, 3, 3), 1)])
def test_only_what_is_needed(shape, dim, need):
    x, w, b, g = make(shape, dim, torch.float32, torch.float32)
    _, mean, rstd = norm.layer_norm_forward(x, w, b, channel_dim=dim)
    outs = norm.layer_norm_backward(x, w, g, mean, rstd, dim, *map(bool, need))
    assert [o is not None for o in outs] == [bool(n) for n in need]
    check_backward(x, w, g, mean, rstd, dim, *outs)


@gpu
@pytest.mark.parametrize("shape,dim", [((3, 9), -1), ((2, 6, 2, 3), 1)])
def test_gradient_against_differences(shape, dim):
    """Central differences of the formula in 64 bits; the step is 2^-10, so the differences
    themselves are off by step^2 times a third derivative (values and weights near 1, C small)."""
    x, w, b, g = make(shape, dim, torch.float32, torch.float32)
    _, mean, rstd = norm.layer_norm_forward(x, w, b, channel_dim=dim)
    gx, gw, gb = norm.layer_norm_backward(x, w, g, mean, rstd, dim)
    C = shape[dim]
    wide = [1] * len(shape)
    wide[dim] = C

    def loss(x, w, b):
        mu = x.mean(dim, keepdim=True)
        xh = (x - mu) / torch.sqrt(((x - mu) ** 2).mean(dim, keepdim=True) + 1e-5)
        return float(((xh * w.reshape(wide) + b.reshape(wide)) * g.double().cpu()).sum())

    args = [t.double().cpu() for t in (x, w, b)]
    h = 2.0 ** -10
    for n, got in enumerate((gx, gw, gb)):
        flat = args[n].reshape(-1)
        for i in range(flat.numel()):
            keep = float(flat[i])
            flat[i] = keep + h
            up = loss(*args)
            flat[i] = keep - h
            down = loss(*args)
            flat[i] = keep
            assert abs((up - down) / (2 * h) - float(got.reshape(-1)[i])) <= 2e-4


@gpu
def test_autograd_and_module():
    m = norm.LayerNorm2d(24).cuda()
    with torch.no_grad():
        m.weight.uniform_(0.5, 1.5)
        m.bias.uniform_(-1, 1)
    x, _, _, g = make((2, 24, 5, 9), 1, torch.float32, torch.float32)
    x.requires_grad_()
    y = m(x)
    y.backward(g)
    _, mean, rstd = norm.layer_norm_forward(x.detach(), m.weight.detach(), m.bias.detach(), channel_dim=1)
    check_backward(x, m.weight.detach(), g, mean, rstd, 1, x.grad, m.weight.grad, m.bias.grad)
    t = torch.nn.LayerNorm(24).cuda()
    t.load_state_dict(norm.LayerNorm(24).state_dict())
    frozen = norm.LayerNorm(24, affine=False).cuda()
    assert torch.equal(frozen(x.detach().permute(0, 2, 3, 1)),
                       norm.layer_norm_forward(x.detach().permute(0, 2, 3, 1).contiguous())[0])
    with pytest.raises(RuntimeError):                # no second derivative: refused, not wrong
        gx, = torch.autograd.grad(m(x).square().sum(), x, create_graph=True)
        gx.sum().backward()


@gpu
def test_a_bias_alone_keeps_its_precision():
    """257 gradients of one and one of 2^-7 a channel: float32 holds their sum, bfloat16 does not."""
    x = torch.randn(258, 33, device="cuda").bfloat16()
    b = torch.zeros(33, device="cuda", requires_grad=True)
    g = torch.ones(258, 33, device="cuda").bfloat16()
    g[0] = 2.0 ** -7
    norm.layer_norm(x, None, b).backward(g)
    assert b.grad.dtype == torch.float32 and bool((b.grad == 257 + 2.0 ** -7).all())


@gpu
def test_refusals():
    x = torch.zeros(4, 8, device="cuda")
    with pytest.raises(TypeError):
        norm.layer_norm(x.double())
    with pytest.raises(TypeError):
        norm.layer_norm(x, torch.ones(8, device="cuda"), torch.ones(8, device="cuda").half())
    with pytest.raises(ValueError):
        norm.layer_norm(x, torch.ones(7, device="cuda"))
    with pytest.raises(ValueError):
        norm.layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError):
        norm.layer_norm(x, eps=-1.0)
    with pytest.raises(_lib.GanetError):
        norm.layer_norm(torch.zeros(1, _lib.GANET_LAYER_NORM_MAX_C + 1, device="cuda"))
    y, mean, rstd = norm.layer_norm_forward(x)
    with pytest.raises(ValueError):
        norm.layer_norm_backward(x, None, x[:3], mean, rstd)
    with pytest.raises(ValueError):
        norm.layer_norm_backward(x, None, x, mean[:3], rstd)
    with pytest.raises(ValueError):
        norm.layer_norm_backward(x, None, x, mean.cpu(), rstd)


@gpu
@pytest.mark.parametrize("shape,dim", [((3001, 72), -1), ((3, 64, 33, 41), 1), ((9, 5000), -1)])
def test_same_bits_again_and_in_a_graph(shape, dim):
    x, w, b, g = make(shape, dim, torch.bfloat16, torch.float32)

    def work():
        y, mean, rstd = norm.layer_norm_forward(x, w, b, channel_dim=dim)
        return (y,) + norm.layer_norm_backward(x, w, g, mean, rstd, dim)

    first = [t.clone() for t in work()]
    for a, c in zip(first, work()):
        assert torch.equal(a, c)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work()
    other = make(shape, dim, torch.bfloat16, torch.float32, seed=5)
    for turn in range(4):
        if turn == 2:                                # other inputs in the captured tensors
            for t, n in zip((x, w, b, g), other):
                t.copy_(n)
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in outs]
        for a, c in zip(kept, work()):               # eager, between the replays
            assert torch.equal(a, c), turn


@gpu
def test_another_stream():
    x, w, b, g = make((513, 200), -1, torch.float32, torch.float32)
    ref = both(x, w, b, g, -1)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y, mean, rstd = norm.layer_norm_forward(x, w, b)
        out = (y,) + norm.layer_norm_backward(x, w, g, mean, rstd)
    side.synchronize()
    for a, c in zip(ref, out):
        assert torch.equal(a, c)


@gpu
def test_offsets_past_32_bits():
    """2^31 + values: the last rows and the last image are right."""
    n, c = (1 << 31) // 4096 + 9, 4096
    x = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
    tail = make((5, c), -1, torch.bfloat16, torch.bfloat16)
    x[-5:] = tail[0]
    y, mean, rstd = norm.layer_norm_forward(x, tail[1], tail[2])
    check_forward(tail[0], tail[1], tail[2], 1e-5, -1, y[-5:], mean[-5:], rstd[-5:])
    del y
    g = torch.zeros_like(x)
    g[-5:] = tail[3]
    gx, gw, gb = norm.layer_norm_backward(x, tail[1], g, mean, rstd)
    check_backward(tail[0], tail[1], tail[3], mean[-5:], rstd[-5:], -1, gx[-5:], None, None)
    # rows of zeros add nothing
    check_backward(tail[0], tail[1], tail[3], mean[-5:], rstd[-5:], -1, None, gw, gb)
    del gx, g, x
    planes = torch.zeros(2, 600, 1800000, dtype=torch.bfloat16, device="cuda")
    part = make((600, 70), 0, torch.bfloat16, torch.bfloat16)
    planes[1, :, -70:] = part[0]
    y, mean, rstd = norm.layer_norm_forward(planes, part[1], part[2], channel_dim=1)
    check_forward(part[0], part[1], part[2], 1e-5, 0, y[1, :, -70:], mean[-70:], rstd[-70:])


@gpu
def test_more_rows_than_a_launch_takes():
    """One channel, 2^31 + rows: every output is its bias."""
    n = (1 << 31) + 70001
    x = torch.ones(n, 1, dtype=torch.bfloat16, device="cuda")
    b = torch.full((1,), 0.75, dtype=torch.bfloat16, device="cuda")
    y = norm.layer_norm(x, None, b)
    assert float(y.min()) == float(y.max()) == 0.75


@gpu
@pytest.mark.parametrize("layout", ["rows", "nchw", "nhwc"])
def test_captured_training_step(layout):
    """Forward, backward and the optimizer's step in one captured graph, replayed with new inputs,
    against the same steps taken eagerly."""
    from ganet_amd import optim
    dim, shape = (-1, (130, 48)) if layout == "rows" else (1, (2, 48, 5, 13))
    x, _, _, g = make(shape, dim, torch.float32, torch.float32)
    if layout == "nhwc":
        x, g = (t.contiguous(memory_format=torch.channels_last) for t in (x, g))

    def build():
        m = norm.LayerNorm(48, channel_dim=dim).cuda()
        return m, optim.AdamW(m.parameters(), lr=1e-2, capturable=True, max_grad_norm=1.0)

    def step(m, o):
        for p in m.parameters():
            p.grad = None
        m(x).backward(g)
        o.step()

    (m, o), (twin, e) = build(), build()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                    # states and first launches, outside the graph
        step(m, o)
    torch.cuda.current_stream().wait_stream(side)
    step(twin, e)
    torch.cuda.synchronize()
    for p in m.parameters():
        p.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        m(x).backward(g)
        o.step()
    for turn in range(4):
        fresh = make(shape, dim, torch.float32, torch.float32, seed=turn + 1)
        x.copy_(fresh[0])
        g.copy_(fresh[3])
        torch.cuda.synchronize()
        graph.replay()
        step(twin, e)
        torch.cuda.synchronize()
        for p, q in zip(m.parameters(), twin.parameters()):
            assert torch.equal(p, q), turn
