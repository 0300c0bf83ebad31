"""The AdamW step (states in 32 and 8 bits) and the norm of all gradients (ganet_amd.optim) against
their formulas in 64 bits.

Tolerances, with u = 2^-24: m = b1 m0 + (1 - b1) g takes at most four roundings a term (the two
coefficients, the products, the sum, the gradient's factor): 6 u (|b1 m0| + |(1 - b1) g|), v alike.
The update lr' m / (sqrt(v) c + eps) adds fewer than eight relative roundings to m's, so the
parameter is off by 16 u (|p| + lr' / denominator (|b1 m0| + |(1 - b1) g|)), and half a step of its
type for its rounding.  The norm is summed in float64 and rounded once: 2^-23 relative.
A value held in 8 bits is one of the two e4m3 values around it, each with the probability that keeps
the mean; which one is a function of the random word, tested against that word's own definition."""
import copy
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

from ganet_amd import _lib, optim

gpu = pytest.mark.gpu
U = 2.0 ** -24
BLOCK = 256
SIZES = [1, 2, 7, 255, 256, 257, 0, 2048, 4095, 4096, 4097, 33001]
PAIRS = [(torch.float32, torch.float32, False), (torch.bfloat16, torch.bfloat16, False),
         (torch.float16, torch.float16, True), (torch.bfloat16, torch.float32, True),
         (torch.float16, torch.float32, False), (torch.float32, torch.bfloat16, False),
         (torch.bfloat16, torch.bfloat16, True)]
HYPER = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.02)


def half(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def make(sizes, pdtype, gdtype, master, seed=0, fresh=False, views=False):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def normal(n, std, dtype):
        t = torch.randn(n + 3, generator=gen, device="cuda") * std
        return t.to(dtype)[3:] if views else t.to(dtype)[:n].clone()     # views: odd addresses

    d = dict(params=[normal(n, 0.05, pdtype) for n in sizes],
             grads=[normal(n, 10.0 ** (i % 5 - 3), gdtype) for i, n in enumerate(sizes)])
    d["m"] = [normal(n, 0.0 if fresh else 0.3 * 10.0 ** (i % 5 - 3), torch.float32)
              for i, n in enumerate(sizes)]
    d["v"] = [normal(n, 0.0 if fresh else 10.0 ** (i % 5 - 3), torch.float32).square()
              for i, n in enumerate(sizes)]
    d["masters"] = [(p.float() + 1e-6) for p in d["params"]] if master else None
    return d


def moved(old, m_terms, m, v, step, hyper):
    """The new parameter in 64 bits, and how far float32 may be from it."""
    b1, b2 = hyper["betas"]
    denom = (v / (1 - b2 ** step)).sqrt() + hyper["eps"]
    rate = hyper["lr"] / (1 - b1 ** step)
    new = old - hyper["lr"] * hyper["weight_decay"] * old - rate * m / denom
    return new, 16 * U * (old.abs() + rate / denom * m_terms)


def check32(before, after, step, hyper, factor=1.0):
    b1, b2 = hyper["betas"]
    for i in range(len(before["params"])):
        g = before["grads"][i].double() * factor
        m0, v0 = before["m"][i].double(), before["v"][i].double()
        m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
        terms = (b1 * m0).abs() + ((1 - b1) * g).abs()
        assert ((after["m"][i].double() - m).abs() <= 6 * U * terms + 1e-44).all()
        assert ((after["v"][i].double() - v).abs() <= 6 * U * v + 1e-44).all()
        old = (before["masters"] or before["params"])[i].double()
        new, tol = moved(old, terms, m, v, step, hyper)
        p = after["params"][i]
        if before["masters"]:
            w = after["masters"][i]
            assert ((w.double() - new).abs() <= tol).all()
            assert torch.equal(p, w.to(p.dtype))
        else:
            tol = tol + half(p.dtype) * new.abs() * (1 + 2 ** -7) + tiny(p.dtype)
            assert ((p.double() - new).abs() <= tol).all()


def clone(d):
    return {k: ([t.clone() for t in v] if v is not None else None) for k, v in d.items()}


def step32(d, step, **kw):
    optim.adamw_step(d["params"], d["grads"], d["m"], d["v"], step, masters=d["masters"], **kw)


# ---- the 8-bit state's definition -----------------------------------------------------------
def words(seed, step, tensor, n):
    """The random word of each of a tensor's n values."""
    def mix(x):
        x = x ^ (x >> np.uint32(16))
        x = x * np.uint32(0xBB67AE85)
        x = x ^ (x >> np.uint32(15))
        x = x * np.uint32(0x6A09E667)
        return x ^ (x >> np.uint32(16))
    i = np.arange(n, dtype=np.uint64)
    one = np.array([(seed + step * 0x9E3779B1 + tensor * 0x85EBCA6B) & 0xFFFFFFFF], np.uint32)
    block = ((i // BLOCK) & 0xFFFFFFFF).astype(np.uint32)
    h = mix(mix(one) + block * np.uint32(0xC2B2AE35))
    h = h + (i % BLOCK).astype(np.uint32) * np.uint32(0x9E3779B1)
    h = h ^ (h >> np.uint32(16))
    h = h * np.uint32(0xBB67AE85)
    return h ^ (h >> np.uint32(15))


def around(y):
    """The e4m3 values at or below and above y (0 <= y <= 448), as (lower, spacing)."""
    step = 2.0 ** (np.floor(np.log2(np.maximum(y, 2.0 ** -6))) - 3)
    return np.floor(y / step) * step, step


def spread(scale, n):
    return np.repeat(scale.cpu().double().numpy(), BLOCK)[:n]


def check8(before, after, step, hyper, seed, factor=1.0):
    b1, b2 = hyper["betas"]
    flips, total = 0, 0.0
    for i in range(len(before["params"])):
        n = before["params"][i].numel()
        g = before["grads"][i].double() * factor
        m0 = before["m"][i].double() * torch.from_numpy(spread(before["ms"][i], n)).cuda()
        r0 = before["r"][i].double() * torch.from_numpy(spread(before["rs"][i], n)).cuda()
        m, v = b1 * m0 + (1 - b1) * g, b2 * r0 ** 2 + (1 - b2) * g * g
        terms = (b1 * m0).abs() + ((1 - b1) * g).abs()
        old = (before["masters"] or before["params"])[i].double()
        new, tol = moved(old, terms, m, v, step, hyper)
        p = after["params"][i]
        if before["masters"]:
            assert ((after["masters"][i].double() - new).abs() <= tol).all()
            assert torch.equal(p, after["masters"][i].to(p.dtype))
        else:
            tol = tol + half(p.dtype) * new.abs() * (1 + 2 ** -7) + tiny(p.dtype)
            assert ((p.double() - new).abs() <= tol).all()
        if n == 0:
            continue
        h = words(seed, step, i, n)
        for key, x, bits in (("m", m, h & np.uint32(0xFFFF)), ("r", v.sqrt(), h >> np.uint32(16))):
            off = (6 * U * terms if key == "m" else 8 * U * x).cpu().numpy()    # of x in float32
            x, s = x.cpu().numpy(), spread(after[key + "s"][i], n)
            starts = np.arange(0, n, BLOCK)
            top, top_off = (np.maximum.reduceat(t, starts) for t in (np.abs(x), off))
            scale = after[key + "s"][i].double().cpu().numpy()
            assert (np.abs(scale * 448 - top) <= top_off + 4 * U * top).all()
            y = np.abs(x) / np.maximum(s, 1e-300)
            slack = off / np.maximum(s, 1e-300) + 8 * U * y                     # of y
            lower, grid = around(np.minimum(y, 448.0))
            got = np.abs(after[key][i].double().cpu().numpy())
            # one of the two neighbours; one further where y is that near to a value of the grid
            assert (got >= lower - (y - lower <= slack) * grid).all()
            assert (got <= lower + grid + (lower + grid - y <= slack) * grid).all()
            want = np.minimum(np.floor(y / grid + (bits + 0.5) / 65536) * grid, 448.0)
            if key == "r":
                want = np.where((x > 0) & (want == 0), 2.0 ** -9, want)
                assert (got[x > 0] > 0).all()
            else:
                signs = np.sign(after[key][i].double().cpu().numpy())
                assert (signs[got > 0] == np.sign(x)[got > 0]).all()
            flips += int((got != want).sum())
            total += float(np.minimum(1.0, 2 * slack / grid).sum())
    # an error below `slack` turns a rounding with probability 2 slack / grid at most
    assert flips <= 3 + 4 * total


def make8(sizes, pdtype, gdtype, master, **kw):
    d = make(sizes, pdtype, gdtype, master, **kw)
    for key, xs in (("m", d["m"]), ("r", [v.sqrt() for v in d["v"]])):
        codes, scales = [], []
        for x in xs:
            n = x.numel()
            pad = torch.nn.functional.pad(x, (0, -n % BLOCK)).reshape(-1, BLOCK)
            top = pad.abs().amax(1) if n else pad.new_zeros(0)
            scales.append(top / 448)
            y = torch.where(top[:, None] > 0, pad / (top / 448)[:, None], torch.zeros_like(pad))
            codes.append(y.clamp(-448, 448).reshape(-1)[:n].to(torch.float8_e4m3fn))
        d[key], d[key + "s"] = codes, scales
    del d["v"]
    return d


def step8(d, step, seed, **kw):
    optim.adamw_step_8bit(d["params"], d["grads"], d["m"], d["r"], d["ms"], d["rs"], step, seed=seed,
                          masters=d["masters"], **kw)


# ------------------------------------------------------------------------------- without a GPU
def test_refusals_without_gpu():
    t = [torch.zeros(4)]
    with pytest.raises(NotImplementedError):
        optim.adamw_step(t, t, t, t, 1)
    with pytest.raises(NotImplementedError):
        optim.grad_norm(t)
    with pytest.raises(ValueError):
        optim.grad_norm([])
    with pytest.raises(ValueError):
        optim.adamw_step(t, t + t, t, t, 1)
    p = [torch.nn.Parameter(torch.zeros(4))]
    for kw in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1e-8), dict(weight_decay=-1.0),
               dict(state_bits=16), dict(max_grad_norm=-1.0), dict(lr=math.nan), dict(eps=math.inf)):
        with pytest.raises(ValueError):
            optim.AdamW(p, **kw)
    o = optim.AdamW(p)
    o.step()                                     # no gradients: nothing to do
    p[0].grad = torch.zeros(4)
    with pytest.raises(NotImplementedError):
        o.step()


def test_c_abi_refusals_without_gpu():
    L = _lib.lib()

    def step(count=1, table=True, tensor=None, **kw):
        t = _lib.StepTensor(param=256, grad=256, exp_avg=256, second=256, exp_avg_scale=256,
                            second_scale=256, master=None, n=16)
        for k, v in (tensor or {}).items():
            setattr(t, k, v)
        p = _lib.AdamwParams(param_dtype=0, grad_dtype=0, state_bits=32, step=1, lr=1e-3, beta1=0.9,
                             beta2=0.999, eps=1e-8, weight_decay=0.0)
        for k, v in kw.items():
            setattr(p, k, v)
        return L.ganet_adamw_step(ctypes.byref(t) if table else None, count, ctypes.byref(p), None)

    bad = _lib.GANET_ERR_BAD_SHAPE
    for kw in (dict(count=-1), dict(param_dtype=3), dict(grad_dtype=-1), dict(state_bits=16),
               dict(reserved=1), dict(lr=-1.0), dict(lr=math.inf), dict(lr=math.nan), dict(beta1=1.0),
               dict(beta2=-0.1), dict(eps=-1.0), dict(eps=math.nan), dict(weight_decay=-0.1), dict(step=0),
               dict(tensor=dict(n=-1)), dict(tensor=dict(n=1 << 62)), dict(tensor=dict(master=256))):
        assert step(**kw) == bad, kw
    for kw in (dict(table=False), dict(tensor=dict(param=None)), dict(tensor=dict(grad=None)),
               dict(tensor=dict(exp_avg=None)), dict(state_bits=8, tensor=dict(second_scale=None))):
        assert step(**kw) == _lib.GANET_ERR_NULL, kw
    assert L.ganet_adamw_step(None, 0, None, None) == _lib.GANET_ERR_NULL
    assert step(count=0, table=False) == _lib.GANET_OK          # nothing to do: no launch
    assert step(tensor=dict(n=0, param=None)) == _lib.GANET_OK

    ptr, num, typ = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(100), (ctypes.c_int32 * 1)(0)

    def gnorm(ptrs=ptr, numel=num, dtypes=typ, count=1, top=1.0, inv=1.0, out=256, ws=256, n=4096):
        return L.ganet_grad_norm(ptrs, numel, dtypes, count, top, inv, out, ws, n, None)

    assert gnorm(count=-1) == bad and gnorm(top=-1.0) == bad and gnorm(top=math.nan) == bad
    assert gnorm(inv=math.inf) == bad and gnorm(numel=(ctypes.c_int64 * 1)(-1)) == bad
    assert gnorm(dtypes=(ctypes.c_int32 * 1)(9)) == bad
    assert gnorm(out=None) == _lib.GANET_ERR_NULL and gnorm(ws=None) == _lib.GANET_ERR_NULL
    assert gnorm(ptrs=(ctypes.c_void_p * 1)(None)) == _lib.GANET_ERR_NULL
    assert gnorm(n=8) == _lib.GANET_ERR_WORKSPACE
    assert L.ganet_grad_norm_workspace_bytes((ctypes.c_int64 * 1)(-5), 1) == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_too_large_a_tensor_is_refused_before_any_step(bits):
    """At the end of a list that takes two launches: nothing is launched (that would be an error of
    another kind without a GPU)."""
    n = 200
    ts = (_lib.StepTensor * n)(*[
        _lib.StepTensor(param=256, grad=256, exp_avg=256, second=256, exp_avg_scale=256,
                        second_scale=256, master=None, n=16) for _ in range(n)])
    ts[n - 1].n = (1 << 33) + 1
    p = _lib.AdamwParams(param_dtype=0, grad_dtype=0, state_bits=bits, step=1, lr=1e-3, beta1=0.9,
                         beta2=0.999, eps=1e-8, weight_decay=0.0)
    rc = _lib.lib().ganet_adamw_step(ts, n, ctypes.byref(p), None)
    assert rc == _lib.GANET_ERR_UNSUPPORTED


def test_dense_and_order():
    t = torch.zeros(4, 3, 5, 7)
    cl = t.contiguous(memory_format=torch.channels_last)
    assert optim._dense(t) and optim._dense(cl) and optim._dense(t.permute(3, 1, 0, 2))
    assert not optim._dense(t[:, :2]) and not optim._dense(t[:, :1].expand(4, 3, 5, 7))
    assert optim._same_order(t, torch.ones_like(t)) and not optim._same_order(t, cl)
    assert optim._same_order(cl, torch.empty_like(cl)) and not optim._same_order(t, t[0])


def test_random_words_are_spread():
    """Means, and the correlation of the two halves and of neighbours, within 6 sigma."""
    n = 1 << 18
    for seed, step, tensor in ((0, 1, 0), (7, 1000, 3), (1, 2, 0)):
        h = words(seed, step, tensor, n)
        lo, hi = (h & 0xFFFF) / 65536.0 - 0.5, (h >> 16) / 65536.0 - 0.5
        sigma = 1 / math.sqrt(12 * n)
        for x in (lo, hi):
            assert abs(x.mean()) < 6 * sigma
            for lag in (1, 2, 8, BLOCK):
                assert abs((x[lag:] * x[:-lag]).mean()) < 6 / 12 / math.sqrt(n)
        assert abs((lo * hi).mean()) < 6 / 12 / math.sqrt(n)
    a, b = words(3, 5, 0, n) / 2.0 ** 32 - 0.5, words(3, 6, 0, n) / 2.0 ** 32 - 0.5
    assert abs((a * b).mean()) < 6 / 12 / math.sqrt(n)


# ------------------------------------------------------------------------------- on the GPU
@gpu
@pytest.mark.parametrize("pdtype,gdtype,master", PAIRS, ids=str)
@pytest.mark.parametrize("views", [False, True])
def test_step32(pdtype, gdtype, master, views):
    d = make(SIZES, pdtype, gdtype, master, views=views)
    before = clone(d)
    step32(d, 17, **HYPER)
    check32(before, d, 17, HYPER)
    for a, b in zip(before["grads"], d["grads"]):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("pdtype,gdtype,master", PAIRS, ids=str)
@pytest.mark.parametrize("views", [False, True])
def test_step8(pdtype, gdtype, master, views):
    d = make8(SIZES, pdtype, gdtype, master, views=views)
    if views:
        for key in ("m", "r"):
            d[key] = [torch.cat([t.view(torch.uint8).new_zeros(1), t.view(torch.uint8)])[1:].view(
                torch.float8_e4m3fn) for t in d[key]]
    before = clone(d)
    step8(d, 17, 5, **HYPER)
    check8(before, d, 17, HYPER, 5)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_first_steps_and_many_tensors(bits):
    """More tensors than a launch takes, states of zeros, three steps."""
    sizes = [(i * 37) % 900 for i in range(150)]
    if bits == 32:
        d = make(sizes, torch.float32, torch.float32, False, fresh=True)
        for t in (1, 2, 3):
            before = clone(d)
            step32(d, t, **HYPER)
            check32(before, d, t, HYPER)
    else:
        d = make8(sizes, torch.float32, torch.float32, False, fresh=True)
        for t in (1, 2, 3):
            before = clone(d)
            step8(d, t, 9, **HYPER)
            check8(before, d, t, HYPER, 9)


@gpu
@pytest.mark.parametrize("hyper", [dict(HYPER, betas=(0.0, 0.0)), dict(HYPER, lr=0.0),
                                   dict(HYPER, weight_decay=0.0, eps=1e-3)], ids=str)
def test_other_hyper_parameters(hyper):
    d = make(SIZES, torch.float32, torch.float32, False)
    before = clone(d)
    step32(d, 4, **hyper)
    check32(before, d, 4, hyper)
    d = make8(SIZES, torch.float32, torch.float32, False)
    before = clone(d)
    step8(d, 4, 1, **hyper)
    check8(before, d, 4, hyper, 1)


@gpu
def test_rounding_keeps_the_mean():
    """A constant gradient: r follows its average, which nearest rounding would stop far below.
    The rounding keeps the mean of r, so v = r^2 gains each rounding's variance: at most the share
    (change of r / r) * (grid / r) = 1 / (2 t) * 1 / 8 of v in step t, which adds up to 1 / 16 of the
    final v = g^2 (1 - b2^t).  Noise: v's relative grid is at most 1 / 4, a rounding's deviation half
    of it, the steps' words independent: 6 sigma = 6 sqrt(steps) / 8 / sqrt(n)."""
    n, steps, g = 1 << 20, 200, 1e-3
    p, grad = [torch.zeros(n, device="cuda")], [torch.full((n,), g, device="cuda")]
    grad[0][::BLOCK] = 50 * g                     # the blocks' scales
    st = optim.state_8bit(p[0])
    for t in range(1, steps + 1):
        optim.adamw_step_8bit(p, grad, [st[0]], [st[1]], [st[2]], [st[3]], t, seed=3, lr=0.0)
    v = (st[1].float().reshape(-1, BLOCK) * st[3][:, None]).double().square()[:, 1:]
    want = g * g * (1 - 0.999 ** steps)
    noise = 6 * math.sqrt(steps) / 8 / math.sqrt(n)
    assert -noise <= float(v.mean()) / want - 1 <= 1 / 16 + noise
    m = (st[0].float().reshape(-1, BLOCK) * st[2][:, None]).double()[:, 1:]
    assert abs(float(m.mean()) / g - 1) <= noise + 0.9 ** steps


@gpu
def test_determinism_and_seeds():
    d = [make8([70000, 300], torch.float32, torch.float32, False) for _ in range(3)]
    for x, seed in zip(d, (1, 1, 2)):
        step8(x, 8, seed, **HYPER)
    for key in ("params", "m", "r", "ms", "rs"):
        for a, b, c in zip(*(x[key] for x in d)):
            view = (lambda t: t.view(torch.uint8)) if key in "mr" else (lambda t: t)
            assert torch.equal(view(a), view(b))
            if key in "mr":
                assert not torch.equal(view(a), view(c))
            else:
                assert torch.equal(view(a), view(c))


@gpu
def test_norm_and_clipping():
    gen = torch.Generator(device="cuda")
    gen.manual_seed(2)
    for sizes in ([1], [0, 5, 0], SIZES, [(i * 53) % 3000 for i in range(300)], [3000001, 12, 70000]):
        grads = [torch.randn(n, generator=gen, device="cuda").to(
            [torch.float32, torch.bfloat16, torch.float16][i % 3]) for i, n in enumerate(sizes)]
        want = math.sqrt(sum(float(g.double().square().sum()) for g in grads))
        for top, inv in ((None, 1.0), (0.5, 1.0), (1e9, 0.25), (0.0, 1.0), (1.0, -2.0)):
            s = optim.grad_norm(grads, top, inv)
            again = optim.grad_norm(grads, top, inv)
            assert torch.equal(s, again)
            s = s.double().tolist()
            norm = want * abs(inv)
            coef = inv * min(1.0, math.inf if top is None else top / (norm + 1e-6))
            assert abs(s[0] - norm) <= 2 ** -23 * norm and abs(s[1] - coef) <= 2 ** -22 * abs(coef)
            assert s[2:] == [0.0, 0.0]
    odd = torch.randn(1001, generator=gen, device="cuda").half()[1:]
    assert abs(float(optim.grad_norm([odd])[0]) / float(odd.double().norm()) - 1) < 2 ** -22
    strided = torch.randn(30, 40, generator=gen, device="cuda")[:, ::2]
    assert abs(float(optim.grad_norm([strided])[0]) / float(strided.double().norm()) - 1) < 2 ** -22
    huge = torch.full((9000,), 1e30, device="cuda")              # squares past float32
    assert abs(float(optim.grad_norm([huge])[0]) / (1e30 * math.sqrt(9000)) - 1) < 1e-6
    for v in (math.inf, -math.inf, math.nan):
        for g in (torch.randn(5000, device="cuda"), torch.randn(5000, device="cuda").bfloat16()):
            g[4321] = v
            s = optim.grad_norm([g, g], 1.0).tolist()
            assert not math.isfinite(s[0]) and s[1:] == [0.0, 1.0, 0.0]
    assert optim.grad_norm([], 1.0, out=torch.ones(4, device="cuda")).tolist() == [0.0, 1.0, 0.0, 0.0]


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_clipped_and_skipped_steps(bits):
    builder, take, check = ((make, step32, check32) if bits == 32 else
                            (make8, lambda d, t, **kw: step8(d, t, 3, **kw),
                             lambda b, a, t, h, f=1.0: check8(b, a, t, h, 3, f)))
    d = builder(SIZES, torch.float32, torch.float32, False)
    stats = optim.grad_norm(d["grads"], 0.25)
    before = clone(d)
    take(d, 5, grad_stats=stats, **HYPER)
    check(before, d, 5, HYPER, float(stats[1]))
    d["grads"][4][3] = math.inf
    stats = optim.grad_norm(d["grads"], 0.25)
    before = clone(d)
    take(d, 6, grad_stats=stats, **HYPER)
    for key, ts in d.items():
        for a, b in zip(ts or [], before[key] or []):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), key


@gpu
def test_non_finite_gradients_stay_in_their_place():
    for v in (math.inf, -math.inf, math.nan):
        d = make([600], torch.float32, torch.float32, False)
        d8 = make8([600], torch.float32, torch.float32, False)
        clean = make8([600], torch.float32, torch.float32, False)
        for x in (d, d8):
            x["grads"][0][300] = v
        clean["grads"][0][300] = 0.0
        step32(d, 3, **HYPER)
        step8(d8, 3, 1, **HYPER)
        step8(clean, 3, 1, **HYPER)
        keep = torch.arange(600, device="cuda") != 300
        assert torch.isfinite(d["params"][0][keep]).all() and not torch.isfinite(d["params"][0][300])
        assert torch.equal(d8["params"][0][keep], clean["params"][0][keep])
        for key in ("m", "r"):
            s = d8[key + "s"][0]
            assert torch.isfinite(s).all() and (s > 0).all()
            assert torch.isfinite(d8[key][0].float()[keep]).all() and d8[key][0].float()[300].isnan()


def states_in_float32(m, r, ms, rs, g, factor, seed, step, tensor, hyper):
    """Codes and scales after a step, every operation rounded to float32 by itself (numpy)."""
    f = np.float32
    b1, b2 = hyper["betas"]
    n = g.size
    at = np.arange(n) // BLOCK
    g = g * f(factor)
    m = m * ms[at] * f(b1) + g * f(1 - b1)
    r = r * rs[at]
    r = np.sqrt(r * r * f(b2) + g * g * f(1 - b2))
    h = words(seed, step, tensor, n)
    out = []
    for x, bits in ((m, h & np.uint32(0xFFFF)), (r, h >> np.uint32(16))):
        top = np.maximum.reduceat(np.abs(x), np.arange(0, n, BLOCK))
        y = np.minimum(np.abs(x) * (f(448) * (f(1) / top))[at], f(448)).astype(np.float64)
        lower, grid = around(y)
        code = np.minimum(np.floor(y / grid + (bits + 0.5) / 65536) * grid, 448.0)
        if x is r:
            code = np.where((x > 0) & (code == 0), 2.0 ** -9, code)
        out += [(code * np.sign(x)).astype(f), top * (f(1) / f(448))]
    return out


@gpu
def test_states_bit_for_bit():
    """Codes and scales are those of the formula in float32, a step after the other."""
    n, seed, factor = 300 * BLOCK + 77, 41, 0.3
    d = make8([5, n], torch.float32, torch.float32, False)
    stats = torch.tensor([1.0, factor, 0.0, 0.0], device="cuda")

    def host():
        return [d[k][1].float().cpu().numpy() for k in ("m", "r", "ms", "rs")]

    for t in range(7, 11):
        want = states_in_float32(*host(), d["grads"][1].cpu().numpy(), factor, seed, t, 1, HYPER)
        step8(d, t, seed, grad_stats=stats, **HYPER)
        got = host()
        for g, w in zip(got, (want[0], want[2], want[1], want[3])):
            assert np.array_equal(g, w), t
        d["grads"][1].mul_(-0.7)


@gpu
def test_squares_past_the_largest_float():
    """A finite gradient whose square is not: its weight does not move, its neighbours do not notice."""
    p = torch.ones(512, device="cuda")
    g = torch.full((512,), 1e-3, device="cuda")
    g[100] = 1e20
    st = optim.state_8bit(p)
    optim.adamw_step_8bit([p], [g], [st[0]], [st[1]], [st[2]], [st[3]], 1, lr=1e-2, weight_decay=0.0)
    assert float(p[100]) == 1.0
    rest = torch.arange(512, device="cuda") != 100
    # m / (1 - b1) over sqrt(v / (1 - b2)) + eps is 1 - 1e-5; a few roundings of 2^-24
    assert ((1 - p[rest]) - 1e-2 * (1 - 1e-5)).abs().max() <= 16 * U
    assert torch.isfinite(st[0].float()[rest]).all() and torch.isfinite(st[2]).all()


@gpu
def test_tiny_gradients_without_eps():
    """Second moments below float32's normal range in 8 bits: nothing becomes infinite, and a step
    is at most some times lr."""
    n = 512
    p = torch.ones(n, device="cuda")
    g = torch.randn(n, device="cuda") * 1e-19
    g[:256] = 0.0
    st = optim.state_8bit(p)
    for t in range(1, 6):
        old = p.clone()
        optim.adamw_step_8bit([p], [g], [st[0]], [st[1]], [st[2]], [st[3]], t, lr=1e-3, eps=0.0,
                              weight_decay=0.0)
        assert ((p - old).abs() <= 0.1).all()
    assert (p[:256] == 1.0).all()


@gpu
def test_two_threads_at_once():
    """Two host threads, each with its own stream and tensors: each gets what one alone gets."""
    jobs = [(make(SIZES, torch.float32, torch.float32, False, seed=i), 3 + i) for i in range(2)]
    alone = []
    for d, t in jobs:
        a = clone(d)
        for k in range(20):
            step32(a, t + k, grad_stats=optim.grad_norm(a["grads"], 0.5), **HYPER)
        alone.append(a)
    torch.cuda.synchronize()
    errors = []

    def work(d, t):
        try:
            side = torch.cuda.Stream()
            with torch.cuda.stream(side):
                for k in range(20):
                    step32(d, t + k, grad_stats=optim.grad_norm(d["grads"], 0.5), **HYPER)
            side.synchronize()
        except Exception as e:                               # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for th in threads:
        th.start()
    for th in threads:
        th.join()
    assert not errors
    for (d, _), a in zip(jobs, alone):
        for key in ("params", "m", "v"):
            for x, y in zip(d[key], a[key]):
                assert torch.equal(x, y)


@gpu
def test_device_step_and_lr():
    for t in (1, 2, 1000, 70000):
        d, e = (make(SIZES, torch.float32, torch.float32, False) for _ in range(2))
        before = clone(d)
        lr = torch.tensor(HYPER["lr"], device="cuda")
        step32(e, torch.tensor(t, device="cuda"), **dict(HYPER, lr=lr))
        check32(before, e, t, HYPER)
        d8 = make8(SIZES, torch.float32, torch.float32, False)
        before = clone(d8)
        step8(d8, torch.tensor(t, device="cuda"), 4, **dict(HYPER, lr=lr))
        check8(before, d8, t, HYPER, 4)


@gpu
def test_orders_and_refusals():
    w = torch.randn(16, 8, 3, 3, device="cuda").contiguous(memory_format=torch.channels_last)
    g = torch.randn(16, 8, 3, 3, device="cuda")                # another order: copied
    m, v = torch.zeros_like(w), torch.zeros_like(w)
    keep = w.clone()
    optim.adamw_step([w], [g], [m], [v], 1, **HYPER)
    d = dict(params=[keep], grads=[g], m=[torch.zeros_like(w)], v=[torch.zeros_like(w)], masters=None)
    check32(d, dict(params=[w], m=[m], v=[v]), 1, HYPER)
    f = torch.zeros(64, device="cuda")

    def call(p=f, g=f, m=None, v=None, **kw):
        m = torch.zeros_like(f) if m is None else m
        v = torch.zeros_like(f) if v is None else v
        optim.adamw_step([p], [g], [m], [v], kw.pop("step", 1), **kw)

    for error, kw in ((ValueError, dict(g=f[:32])), (ValueError, dict(m=f[:32])),
                      (ValueError, dict(m=f)),                          # the parameter itself
                      (ValueError, dict(p=torch.zeros(128, device="cuda")[::2])),
                      (TypeError, dict(m=f.half())), (TypeError, dict(p=f.double())),
                      (TypeError, dict(masters=[f])),
                      (ValueError, dict(grad_stats=torch.zeros(3, device="cuda"))),
                      (ValueError, dict(step=torch.tensor(1))),
                      (ValueError, dict(lr=torch.zeros(2, device="cuda"))),
                      (_lib.GanetError, dict(step=0)), (_lib.GanetError, dict(lr=-1.0))):
        with pytest.raises(error):
            call(**kw)
    with pytest.raises(ValueError):
        s = torch.zeros(4, 64, device="cuda")
        optim.adamw_step([f, f], [f, f], [s[0], s[1]], [s[2], s[3]], 1)
    with pytest.raises(ValueError):
        c = optim.state_8bit(f)
        optim.adamw_step_8bit([f], [f], [c[0]], [c[1]], [c[2]], [torch.zeros(3, device="cuda")], 1)
    with pytest.raises(TypeError):
        optim.grad_norm([f.double()])
    with pytest.raises(ValueError):
        optim.grad_norm([f], math.nan)


def small_model(dtype=torch.float32):
    torch.manual_seed(0)
    return torch.nn.Sequential(torch.nn.Linear(40, 200), torch.nn.ReLU(),
                               torch.nn.Linear(200, 30)).cuda().to(dtype)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_optimizer_matches_the_raw_calls_and_reloads(bits, master):
    dtype = torch.bfloat16 if master else torch.float32
    model = small_model(dtype)
    kw = dict(lr=1e-2, weight_decay=0.1, state_bits=bits, master_weights=master, max_grad_norm=0.5,
              min_8bit_size=100, seed=11)
    o = optim.AdamW(model.parameters(), **kw)
    x = torch.randn(64, 40, device="cuda").to(dtype)

    def backward(model):
        for p in model.parameters():
            p.grad = None
        model(x).float().square().mean().backward()

    for t in (1, 2, 3):
        backward(model)
        ps = list(model.parameters())
        stats = optim.grad_norm([p.grad for p in ps], 0.5)
        small = [p for p in ps if bits == 32 or p.numel() < 100]
        state = {p: {k: v.clone() if torch.is_tensor(v) else v for k, v in o.state[p].items()}
                 for p in small} if t > 1 else None
        old = [p.detach().clone() for p in small]
        o.step()
        assert torch.equal(o.grad_stats, stats)
        if state is not None and small:
            before = dict(params=old, grads=[p.grad for p in small],
                          m=[state[p]["exp_avg"] for p in small],
                          v=[state[p]["exp_avg_sq"] for p in small],
                          masters=[state[p]["master"] for p in small] if master else None)
            after = dict(params=[p.detach() for p in small], m=[o.state[p]["exp_avg"] for p in small],
                         v=[o.state[p]["exp_avg_sq"] for p in small],
                         masters=[o.state[p]["master"] for p in small] if master else None)
            check32(before, after, t, dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1),
                    float(stats[1]))
    # a copy goes on from the saved state with the same bits
    twin = small_model(dtype)
    twin.load_state_dict(model.state_dict())
    o2 = optim.AdamW(twin.parameters(), **kw)
    o2.load_state_dict(o.state_dict())
    for p, q in zip(model.parameters(), twin.parameters()):
        for name, value in o.state[p].items():
            if torch.is_tensor(value):
                assert o2.state[q][name].dtype == value.dtype
                assert o2.state[q][name].data_ptr() != value.data_ptr()
    copied = copy.deepcopy(o2)                       # options and states go along
    assert (copied.state_bits, copied.max_grad_norm, copied.seed) == (bits, 0.5, 11)
    for _ in range(2):
        for m, opt in ((model, o), (twin, o2)):
            backward(m)
            opt.step()
    for p in copied.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    copied.step()
    for p, q in zip(model.parameters(), twin.parameters()):
        assert torch.equal(p, q)


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_captured_step_counts_on(bits):
    """A captured step (capturable) replayed equals the same steps taken eagerly; eager work and
    waits stand between the replays."""
    model, twin = small_model(), small_model()
    kw = dict(lr=1e-2, state_bits=bits, min_8bit_size=100, max_grad_norm=1.0)
    o = optim.AdamW(model.parameters(), capturable=True, **kw)
    e = optim.AdamW(twin.parameters(), capturable=True, **kw)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(1)

    def fill():
        for p, q in zip(model.parameters(), twin.parameters()):
            g = torch.randn(p.shape, generator=gen, device="cuda")
            for t in (p, q):
                if t.grad is None:
                    t.grad = torch.empty_like(t)
                t.grad.copy_(g)

    fill()
    plain = optim.AdamW(model.parameters(), **kw)
    for opt in (o, plain):                           # no state yet; a number that would not count on
        with pytest.raises(RuntimeError):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
    o.step()
    e.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o.step()
    for _ in range(4):
        fill()
        torch.cuda.synchronize()
        graph.replay()
        e.step()
        torch.cuda.synchronize()
        for p, q in zip(model.parameters(), twin.parameters()):
            assert torch.equal(p, q)


@gpu
def test_another_stream():
    d = make(SIZES, torch.float32, torch.float32, False)
    before = clone(d)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        stats = optim.grad_norm(d["grads"], 0.25)
        step32(d, 5, grad_stats=stats, **HYPER)
    side.synchronize()
    check32(before, d, 5, HYPER, float(stats[1]))


@gpu
@pytest.mark.parametrize("order", [torch.contiguous_format, torch.channels_last])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_is_a_change_in_place(bits, order):
    """A backward pass that saved the weights of before the step is refused, as after torch's."""
    p = torch.ones(2, 3, 40, 50, device="cuda").contiguous(memory_format=order).bfloat16()
    p.requires_grad_()
    opt = optim.AdamW([p], state_bits=bits, master_weights=True)
    for _ in range(2):                       # a fresh state, a kept one
        loss = (p.float() * p.float()).sum() + (p * p).sum()
        p.grad = torch.ones_like(p)
        before = p._version, opt.state[p]["master"]._version if p in opt.state else 0
        opt.step()
        assert p._version > before[0] and opt.state[p]["master"]._version > before[1]
        with pytest.raises(RuntimeError, match="inplace"):
            loss.backward()
    with torch.inference_mode():             # tensors without versions
        q = [torch.ones(9, device="cuda") for _ in range(4)]
        optim.adamw_step(q[:1], q[1:2], q[2:3], q[3:], 1)
        assert float(q[0][0]) < 1


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_offsets_past_32_bits(bits):
    n, last = (1 << 31) + 1001, 777
    p = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    g[-last:] = torch.randn(last, device="cuda").bfloat16()
    p[-last:] = torch.randn(last, device="cuda").bfloat16()
    assert abs(float(optim.grad_norm([g])[0]) / float(g[-last:].double().norm()) - 1) < 2 ** -22
    before = dict(params=[p[-last:].clone()], grads=[g[-last:]], masters=None)
    if bits == 32:
        m, v = (torch.zeros(n, device="cuda") for _ in range(2))
        before["m"], before["v"] = [m[-last:].clone()], [v[-last:].clone()]
        optim.adamw_step([p], [g], [m], [v], 1, **HYPER)
        check32(before, dict(params=[p[-last:]], m=[m[-last:]], v=[v[-last:]]), 1, HYPER)
    else:
        st = optim.state_8bit(p)
        optim.adamw_step_8bit([p], [g], [st[0]], [st[1]], [st[2]], [st[3]], 1, **HYPER)
        x = g[-last:].double()
        new, tol = moved(before["params"][0].double(), 0.1 * x.abs(), 0.1 * x, 0.001 * x * x, 1, HYPER)
        tol = tol + half(p.dtype) * new.abs() * (1 + 2 ** -7)
        assert ((p[-last:].double() - new).abs() <= tol).all()
        scale = st[2][-5:].double().repeat_interleave(BLOCK)
        at = n - (n - 1) // BLOCK * BLOCK                       # values of the last block
        got = st[0][-at:].double() * float(st[2][-1])
        assert ((got - 0.1 * g[-at:].double()).abs() <= float(st[2][-1]) * 32 + 1e-30).all()
        assert scale.numel() and float(st[0][:1 << 31].view(torch.uint8)[::4099].max()) == 0


@gpu
def test_training_chain():
    """DeformConv1D -> LayerNorm2d -> loss, backward, clipping, AdamW: what a user trains.  Every
    step is checked from the gradients that the backward left."""
    from ganet_amd import dcn, norm

    class Block(torch.nn.Module):
        def __init__(self):
            super(Block, self).__init__()
            self.conv = dcn.DeformConv1D(64, 32, 7, 1, 3)
            self.norm = norm.LayerNorm2d(32)

        def forward(self, x, offset):
            return torch.relu(self.norm(self.conv(x, offset)))

    torch.manual_seed(3)
    block = Block().cuda()
    x = torch.randn(2, 64, 9, 13, device="cuda")
    off = torch.randn(2, 14, 9, 13, device="cuda")
    target = torch.rand(2, 32, 9, 13, device="cuda")
    o = optim.AdamW(block.parameters(), lr=5e-3, max_grad_norm=0.1)
    ps = list(block.parameters())
    for t in (1, 2, 3):
        o.zero_grad()
        (block(x, off) - target).square().mean().backward()
        # the norm's gradients against autograd of the plain formula on the same activations
        with torch.no_grad():
            h = block.conv(x, off)
        w, b = (q.detach().double().requires_grad_() for q in (block.norm.weight, block.norm.bias))
        hd = h.double()
        xh = (hd - hd.mean(1, keepdim=True)) / (hd.var(1, keepdim=True, correction=0) + 1e-5).sqrt()
        y = xh * w.reshape(1, -1, 1, 1) + b.reshape(1, -1, 1, 1)
        (torch.relu(y) - target).square().mean().backward()
        for q, ref in ((block.norm.weight, w), (block.norm.bias, b)):
            # a sum of 234 float32 terms, and elements of relu within rounding of zero
            assert (q.grad - ref.grad).abs().max() <= 1e-4 * ref.grad.abs().max()
        before = dict(params=[p.detach().clone() for p in ps], grads=[p.grad.clone() for p in ps],
                      masters=None)
        state = [o.state[p] if p in o.state else {} for p in ps]
        before["m"] = [s["exp_avg"].clone() if s else torch.zeros_like(p) for s, p in zip(state, ps)]
        before["v"] = [s["exp_avg_sq"].clone() if s else torch.zeros_like(p) for s, p in zip(state, ps)]
        o.step()
        total = math.sqrt(sum(float(g.double().square().sum()) for g in before["grads"]))
        assert abs(float(o.grad_stats[0]) / total - 1) <= 2 ** -22
        check32(before, dict(params=[p.detach() for p in ps], m=[o.state[p]["exp_avg"] for p in ps],
                             v=[o.state[p]["exp_avg_sq"] for p in ps]), t,
                dict(lr=5e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2), float(o.grad_stats[1]))
