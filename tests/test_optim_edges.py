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


def numbers(opt, ps):
    return [int(opt.state[p]["step"]) if p in opt.state else 0 for p in ps]


def sparse_steps(opt, ps, present, t_of, gen, bits=32):
    """One step in which only the parameters `present` have gradients, checked with a number of its
    own for each of them."""
    for i, p in enumerate(ps):
        p.grad = torch.randn(p.shape, generator=gen, device="cuda") if i in present else None
    some = [ps[i] for i in present]
    had = [p in opt.state for p in some]
    before = [dict(params=[p.detach().clone()], grads=[p.grad], masters=None,
                   m=[opt.state[p]["exp_avg"].clone() if h else torch.zeros_like(p)],
                   v=[opt.state[p]["exp_avg_sq"].clone() if h else torch.zeros_like(p)])
              for p, h in zip(some, had)] if bits == 32 else None
    opt.step()
    for i in present:
        t_of[i] += 1
    if before is not None:
        for i, p, b in zip(present, some, before):
            s = opt.state[p]
            check32(b, dict(params=[p.detach()], m=[s["exp_avg"]], v=[s["exp_avg_sq"]]), t_of[i], HYPER)
    assert numbers(opt, ps) == t_of


@gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("capturable", [False, True])
def test_a_parameter_without_a_gradient_is_not_counted(capturable, bits):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(4)
    ps = [torch.nn.Parameter(torch.randn(n, generator=gen, device="cuda")) for n in (300, 70, 513)]
    opt = optim.AdamW(ps, capturable=capturable, state_bits=bits, min_8bit_size=1, **HYPER)
    t_of = [0, 0, 0]
    for present in ((0, 1), (0, 2), (0, 1, 2), (0, 2), (2,), (0, 1, 2), (1,)):      # the third comes later
        sparse_steps(opt, ps, present, t_of, gen, bits)
    twin = optim.AdamW(ps, capturable=capturable, state_bits=bits, min_8bit_size=1, **HYPER)
    twin.load_state_dict(opt.state_dict())
    assert numbers(twin, ps) == t_of == [5, 4, 5]
    for present in ((0, 1, 2), (0,), (1, 2)):
        sparse_steps(twin, ps, present, t_of, gen, bits)


@gpu
def test_captured_steps_and_missing_gradients():
    """What a captured step shares a number with has to have a gradient too, before and after."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(5)

    def fresh():
        ps = [torch.nn.Parameter(torch.randn(n, generator=gen, device="cuda")) for n in (300, 70)]
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen, device="cuda")
        opt = optim.AdamW(ps, capturable=True, **HYPER)
        opt.step()
        torch.cuda.synchronize()
        return ps, opt

    ps, opt = fresh()
    keep, ps[1].grad = ps[1].grad, None
    with pytest.raises(RuntimeError, match="gradient"):      # would count ps[1] on every replay
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
    opt.step()                                               # the same outside: has numbers of its own
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
    assert numbers(opt, ps) == [5, 1]
    ps[1].grad = keep
    opt.step()
    assert numbers(opt, ps) == [6, 2]

    ps, opt = fresh()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    graph.replay()
    torch.cuda.synchronize()
    ps[1].grad = None
    with pytest.raises(RuntimeError, match="captured"):      # the graph counts both with one number
        opt.step()
    assert numbers(opt, ps) == [2, 2]


def codes(opt, p):
    return [opt.state[p][k].view(torch.uint8) for k in ("exp_avg", "exp_rms")]


@gpu
@pytest.mark.parametrize("capturable", [False, True])
def test_groups_round_with_words_of_their_own(capturable):
    """Equal weights with equal gradients in two groups: equal moments, unlike roundings; the words
    are those of one list of all tensors."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(6)
    value, grad = (torch.randn(5000, generator=gen, device="cuda") for _ in range(2))
    ps = [torch.nn.Parameter(value.clone()) for _ in range(4)]
    opt = optim.AdamW([dict(params=ps[:2], weight_decay=0.0), dict(params=ps[2:], weight_decay=0.1)],
                      state_bits=8, seed=21, capturable=capturable)
    st = [optim.state_8bit(p.detach()) for p in ps]
    raw = [value.clone() for _ in ps]
    for t in (1, 2):
        for p in ps:
            p.grad = grad.clone()
        opt.step()
        # the moments do not depend on the weights: one raw call over all four
        optim.adamw_step_8bit(raw, [grad] * 4, *([s[k] for s in st] for k in range(4)), t, seed=21)
        for p, s in zip(ps, st):
            for a, b in zip(codes(opt, p), s[:2]):
                assert torch.equal(a, b.view(torch.uint8))
    for i in range(4):
        for j in range(i):
            for a, b in zip(codes(opt, ps[i]), codes(opt, ps[j])):
                assert not torch.equal(a, b), (i, j)


@gpu
def test_groups_alike_are_stepped_in_one_call(monkeypatch):
    """One group a parameter, as a config with settings by name makes them."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(7)
    values = [torch.randn(500 + i, generator=gen, device="cuda") for i in range(6)]
    grads = [torch.randn(500 + i, generator=gen, device="cuda") for i in range(6)]
    done = []
    for split in (True, False):
        ps = [torch.nn.Parameter(v.clone()) for v in values]
        opt = optim.AdamW([dict(params=[p], betas=[0.9, 0.99]) for p in ps] if split else ps, lr=1e-2,
                          betas=(0.9, 0.99), state_bits=8, min_8bit_size=503, seed=3)
        calls = []
        for name in ("adamw_step", "adamw_step_8bit"):
            monkeypatch.setattr(optim, name, lambda *a, _f=getattr(optim, name), **kw: (
                calls.append(len(a[0])), _f(*a, **kw))[1])
        for _ in range(2):
            for p, g in zip(ps, grads):
                p.grad = g.clone()
            opt.step()
        monkeypatch.undo()
        assert sorted(calls) == [3, 3, 3, 3]
        done.append([p.detach() for p in ps] + [c for p in ps[3:] for c in codes(opt, p)])
    for a, b in zip(*done):
        assert torch.equal(a, b)


@gpu
def test_states_of_another_memory_order():
    """Scales belong to 256 values in memory order: states saved from a channels_last weight and loaded
    into a contiguous one are divided into other blocks.  A value keeps its sign and is off by half
    of e4m3's spacing in its new scale, 2^-4 of itself or 2^-10 of the scale; a root above zero
    stays above zero (2^-9 of the scale at least)."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(8)
    shape = (16, 40, 3, 3)
    w = torch.randn(shape, generator=gen, device="cuda")
    size = torch.exp(torch.randn(shape, generator=gen, device="cuda") * 2)
    p = torch.nn.Parameter(w.contiguous(memory_format=torch.channels_last))
    q = torch.nn.Parameter(w.clone())
    a, b, same = (optim.AdamW([x], state_bits=8, seed=2) for x in (p, q, torch.nn.Parameter(p.detach())))
    for _ in range(3):
        p.grad = (torch.randn(shape, generator=gen, device="cuda") * size).contiguous(
            memory_format=torch.channels_last)
        a.step()

    def values(opt, p, key, scale):
        """The state in the weight's shape, and the scale of each of its values."""
        s = opt.state[p]
        spread = s[scale].repeat_interleave(BLOCK)[:p.numel()]
        per = torch.empty_like(p, requires_grad=False)
        per.as_strided((p.numel(),), (1,)).copy_(spread)
        assert s[key].stride() == p.stride()
        return s[key].float() * per, per

    b.load_state_dict(a.state_dict())
    for key, scale in (("exp_avg", "avg_scale"), ("exp_rms", "rms_scale")):
        old, _ = values(a, p, key, scale)
        new, per = values(b, q, key, scale)
        least = 2.0 ** -9 if key == "exp_rms" else 2.0 ** -10
        tol = torch.maximum(old.abs() * 2.0 ** -4, per * least) * (1 + 8 * U)
        assert ((new - old).abs() <= tol).all()
        assert ((new > 0) == (old > 0)).all() or key == "exp_avg"
        assert (new * old >= 0).all()
    q.grad = p.grad.contiguous()
    b.step()
    assert torch.isfinite(q).all()
    # in the same order nothing changes
    same.load_state_dict(a.state_dict())
    r = same.param_groups[0]["params"][0]
    for k in ("exp_avg", "exp_rms", "avg_scale", "rms_scale"):
        one, two = a.state[p][k], same.state[r][k]
        assert torch.equal(one.view(torch.uint8), two.view(torch.uint8)) and one.stride() == two.stride()


@gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("master", [False, True])
def test_states_of_torch_are_taken_over(dtype, master):
    """torch.optim.AdamW keeps 16-bit moments for 16-bit weights, and no masters."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(9)
    ps = [torch.nn.Parameter(torch.randn(n, generator=gen, device="cuda").to(dtype)) for n in (77, 400)]
    theirs = torch.optim.AdamW(ps, lr=HYPER["lr"], weight_decay=HYPER["weight_decay"])

    def gradients():
        for p in ps:
            p.grad = torch.randn(p.shape, generator=gen, device="cuda").to(dtype)

    for _ in range(3):
        gradients()
        theirs.step()
    ours = optim.AdamW(ps, master_weights=master, **HYPER)
    ours.load_state_dict(theirs.state_dict())
    masters = master and dtype != torch.float32
    before = dict(params=[p.detach().clone() for p in ps], grads=None,
                  m=[theirs.state[p]["exp_avg"].float() for p in ps],
                  v=[theirs.state[p]["exp_avg_sq"].float() for p in ps],
                  masters=[p.detach().float() for p in ps] if masters else None)
    gradients()
    before["grads"] = [p.grad for p in ps]
    ours.step()
    st = [ours.state[p] for p in ps]
    assert all(("master" in s) == masters for s in st)
    check32(before, dict(params=[p.detach() for p in ps], m=[s["exp_avg"] for s in st],
                         v=[s["exp_avg_sq"] for s in st],
                         masters=[s["master"] for s in st] if masters else None), 4, HYPER)


@gpu
def test_a_refused_step_counts_nothing():
    """A parameter that was not stepped keeps its number and gets no half-made state."""
    def parameter(*shape):
        return torch.nn.Parameter(torch.ones(*shape, device="cuda"))

    good, gaps, late = parameter(60), torch.nn.Parameter(torch.ones(8, 6, device="cuda")[:, ::2]), parameter(9)
    opt = optim.AdamW([good, gaps], **HYPER)
    for p in (good, gaps):
        p.grad = torch.ones_like(p)
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(good, torch.ones_like(good)) and numbers(opt, [good]) == [0]
    gaps.grad = None
    opt.step()
    assert numbers(opt, [good]) == [1] and gaps not in opt.state
    check = torch.ones(60, device="cuda")
    optim.adamw_step([check], [good.grad], [torch.zeros_like(check)], [torch.zeros_like(check)], 1, **HYPER)
    assert torch.equal(check, good)

    for capturable in (False, True):
        good, late = parameter(60), parameter(9)
        opt = optim.AdamW([dict(params=[good]), dict(params=[late], lr=1e-4)], capturable=capturable)
        for p in (good, late):
            p.grad = torch.ones_like(p)
        opt.param_groups[1]["lr"] = -1.0
        with pytest.raises((ValueError, _lib.GanetError)):
            opt.step()
        assert torch.equal(late, torch.ones_like(late))
        # whatever was stepped has been counted, and what was not has not
        assert numbers(opt, [good, late]) == [int(not torch.equal(good, torch.ones_like(good))), 0]

        before = numbers(opt, [good, late])
        opt.param_groups[1]["lr"] = torch.tensor(1e-4)              # on the host: not taken
        for _ in range(2):
            opt.param_groups[0]["lr"] = torch.tensor(1e-3)
            with pytest.raises(ValueError):
                opt.step()
        assert numbers(opt, [good, late]) == before


def test_overlaps():
    inside = optim._overlap
    assert not inside([]) and not inside([(100, 4)]) and not inside([(100, 4), (104, 4), (0, 100)])
    assert inside([(100, 4), (100, 4)]) and inside([(100, 8), (104, 4)]) and inside([(104, 4), (96, 9)])
    assert inside([(0, 1000), (10, 4), (500, 4)])
    assert not inside([(100, 0), (100, 4)]) and not inside([(0, 0), (0, 0)])      # nothing in them


@gpu
def test_tensors_that_share_memory_are_refused():
    """Views of one buffer that share some values: which step they would get is a matter of luck."""
    flat = torch.zeros(4096, device="cuda")

    def call(a, b, ma=None, mb=None):
        zeros = [torch.zeros_like(a) for _ in range(6)]
        optim.adamw_step([a, b], zeros[:2], [zeros[2] if ma is None else ma, zeros[3] if mb is None else mb],
                         zeros[4:], 1)

    call(flat[:100], flat[100:200])                                  # neighbours
    with pytest.raises(ValueError, match="memory"):
        call(flat[:100], flat[99:199])
    with pytest.raises(ValueError, match="memory"):
        call(flat[:100], flat[100:200], flat[150:250])
    with pytest.raises(ValueError, match="memory"):
        call(flat[:100].view(10, 10).t(), flat[50:150].view(10, 10).t())
    call(flat[:100].view(10, 10).t(), flat[100:200].view(10, 10).t())
    p = [flat[:512], flat[600:1112]]
    st = [optim.state_8bit(t) for t in p]
    scales = torch.zeros(3, device="cuda")
    with pytest.raises(ValueError, match="memory"):
        optim.adamw_step_8bit(p, [torch.zeros(512, device="cuda")] * 2, *([s[k] for s in st] for k in (0, 1)),
                              [scales[:2], scales[1:]], [s[3] for s in st], 1)
    assert not flat.any()


@gpu
def test_out_of_memory_keeps_its_type():
    """Programs catch torch.OutOfMemoryError to try again with less."""
    from ganet_amd import norm
    g = torch.zeros(1 << 20, device="cuda")
    x = torch.zeros(1 << 22, 64, device="cuda", dtype=torch.bfloat16)
    y, mean, rstd = norm.layer_norm_forward(x[:64])
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    total = torch.cuda.get_device_properties(0).total_memory
    torch.cuda.set_per_process_memory_fraction((torch.cuda.memory_reserved() + (1 << 25)) / total)
    try:
        with pytest.raises(torch.OutOfMemoryError):
            norm.layer_norm_forward(x)
        with pytest.raises(torch.OutOfMemoryError):
            norm.layer_norm(x)
    finally:
        torch.cuda.set_per_process_memory_fraction(1.0)
    assert float(optim.grad_norm([g])[0]) == 0.0 and torch.equal(norm.layer_norm(x)[0], x[0])


@gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_states_of_another_shape_are_refused(bits):
    """A state of one value would have been spread over all."""
    one, many = (torch.nn.Parameter(torch.ones(n, 5, device="cuda")) for n in (1, 9))
    a, b = (optim.AdamW([p], state_bits=bits, min_8bit_size=1) for p in (one, many))
    one.grad = torch.ones_like(one)
    a.step()
    with pytest.raises(ValueError):
        b.load_state_dict(a.state_dict())
