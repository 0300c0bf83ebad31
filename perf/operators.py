"""The training operators beside the deformable convolutions: layer norm over channels
(forward, backward), the AdamW step over many tensors (states in 32 or in 8 bits) and the norm of
all gradients with its clipping coefficient.  `run` computes them in plain torch operations, or
(`own`) by the calls of ganet_amd.norm and ganet_amd.optim."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256                       # values that share a scale in the 8-bit states
E4M3_MAX = 448.0
EPS_LN = 1e-5
HYPER = dict(lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01)
M32 = 0xFFFFFFFF


# ---------------------------------------------------------------------------------- the cases
def listed():
    return [
        # the top pyramid level of one 800x320 frame (10x25 positions) as tokens: latency
        dict(name="ln_fwd_tokens_f32", op="ln_fwd", layout="rows", dtype="f32", wdtype="f32",
             n=250, c=256),
        # the map that a deformable convolution leaves, NCHW, batch 32
        dict(name="ln_fwd_nchw_bf16", op="ln_fwd", layout="nchw", dtype="bf16", wdtype="f32",
             b=32, c=256, h=40, w=100),
        # channels_last map of the full head, batch 128: the aggregator's 64 output channels
        dict(name="ln_fwd_nhwc_c64_bf16", op="ln_fwd", layout="nhwc", dtype="bf16", wdtype="bf16",
             b=128, c=64, h=40, w=100),
        # odd width, rows that start at any alignment, training backward of a small batch
        dict(name="ln_bwd_odd_f16", op="ln_bwd", layout="rows", dtype="f16", wdtype="f32",
             n=777, c=1001),
        # backward over an NCHW float32 map, batch 32
        dict(name="ln_bwd_nchw_f32", op="ln_bwd", layout="nchw", dtype="f32", wdtype="f32",
             b=32, c=256, h=40, w=100),
        # long bf16 rows, generic token training
        dict(name="ln_bwd_rows_bf16", op="ln_bwd", layout="rows", dtype="bf16", wdtype="bf16",
             n=16384, c=4096),
        # the aggregator's own weight [64, 256, 1, 7]: the smallest step, latency
        dict(name="adamw32_lfa_f32", op="adamw32", pdtype="f32", gdtype="f32", master=False,
             tensors=1, values=64 * 256 * 7, step=1),
        # a large model's parameters, float32 throughout
        dict(name="adamw32_large_f32", op="adamw32", pdtype="f32", gdtype="f32", master=False,
             tensors=150, values=100_000_003, step=1000),
        # bf16 weights and gradients on float32 masters, states in 8 bits, a detector's worth
        dict(name="adamw8_master_bf16", op="adamw8", pdtype="bf16", gdtype="bf16", master=True,
             tensors=62, values=24_000_011, step=37),
        # float32 weights, states in 8 bits, a large model
        dict(name="adamw8_large_f32", op="adamw8", pdtype="f32", gdtype="f32", master=False,
             tensors=150, values=100_000_003, step=1000),
        # the norm over a detector's many small gradients: latency and ragged sizes
        dict(name="grad_norm_many_f32", op="grad_norm", gdtype="f32", tensors=62,
             values=11_000_017),
        # the norm over a large model's bf16 gradients
        dict(name="grad_norm_large_bf16", op="grad_norm", gdtype="bf16", tensors=300,
             values=400_000_013),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "ln_fwd", "ln_bwd", "adamw32", "adamw8", "grad_norm"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op in ("ln_fwd", "ln_bwd"):
        c = _log(rng, 16, 8192)
        wdtype = rng.choice([dtype, "f32"])
        layout = rng.choice(["rows", "nchw", "nhwc"])
        if layout == "rows":
            n = _log(rng, 16, max(17, min(200_000, 30_000_000 // c)))
            return dict(op=op, layout=layout, dtype=dtype, wdtype=wdtype, n=n, c=c)
        c = min(c, 1024)
        h, w = rng.randint(5, 80), rng.randint(7, 200)
        b = _log(rng, 1, max(2, min(128, 30_000_000 // (c * h * w))))
        return dict(op=op, layout=layout, dtype=dtype, wdtype=wdtype, b=b, c=c, h=h, w=w)
    tensors = _log(rng, 1, 200)
    values = _log(rng, max(100_000, 300 * tensors), 50_000_000)
    if op == "grad_norm":
        return dict(op=op, gdtype=dtype, tensors=tensors, values=values)
    master = dtype != "f32" and rng.random() < 0.5
    return dict(op=op, pdtype=dtype, gdtype=rng.choice([dtype, "f32"]), master=master,
                tensors=tensors, values=values, step=_log(rng, 1, 100_000))


def _sizes(case):
    """Sizes of a model's tensors: spread over their logarithm, the rest in the largest."""
    rng = random.Random(case["tensors"] * 1_000_003 + case["values"])
    mean = case["values"] // case["tensors"]
    sizes = [max(1, min(2 * mean, _log(rng, 32, 8 * mean + 64))) for _ in range(case["tensors"])]
    over = sum(sizes) - case["values"]
    scale = case["values"] / sum(sizes) if over > 0 else 1.0
    sizes = [max(1, int(s * scale)) for s in sizes]
    sizes[-1] += max(0, case["values"] - sum(sizes))
    return sizes


# ---------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))

    def normal(shape, dtype, std=1.0, mean=0.0):
        return (torch.randn(shape, generator=gen, device="cuda") * std + mean).to(dtype)

    s = {"case": case}
    if case["op"] in ("ln_fwd", "ln_bwd"):
        dt, wt, c = DTYPES[case["dtype"]], DTYPES[case["wdtype"]], case["c"]
        if case["layout"] == "rows":
            shape, wide, s["dim"] = (case["n"], c), (1, c), -1
        else:
            shape, wide, s["dim"] = (case["b"], c, case["h"], case["w"]), (1, c, 1, 1), 1
        scale = normal(wide, torch.float32).abs() + 0.3        # channels of unlike size
        x = (normal(shape, torch.float32) * scale + normal(wide, torch.float32, 0.5)).to(dt)
        grad = normal(shape, dt)
        if case["layout"] == "nhwc":
            x = x.contiguous(memory_format=torch.channels_last)
            grad = grad.contiguous(memory_format=torch.channels_last)
        s.update(x=x, weight=normal((c,), wt, 0.2, 1.0), bias=normal((c,), wt, 0.2), wide=wide)
        if case["op"] == "ln_bwd":
            var, mean = torch.var_mean(x.double() if x.numel() < 1 << 27 else x.float(), s["dim"],
                                       correction=0)
            s.update(grad=grad, mean=mean.float().reshape(-1),
                     rstd=torch.rsqrt(var.double() + EPS_LN).float().reshape(-1))
        return s

    # every tensor starts at a block's border of one flat buffer, as an allocator would align it;
    # what lies between is zero and stays zero
    sizes = _sizes(case)
    blocks = [-(-n // BLOCK) for n in sizes]
    starts = [0]
    for b in blocks:
        starts.append(starts[-1] + b)
    total = starts[-1] * BLOCK
    s["spans"] = spans = [(a * BLOCK, n) for a, n in zip(starts, sizes)]
    real = torch.zeros(total, dtype=torch.bool, device="cuda")
    for a, n in spans:
        real[a:a + n] = True

    def views(flat):
        return [flat[a:a + n] for a, n in spans]

    gt = DTYPES[case["gdtype"]]
    size = torch.exp(torch.randn(starts[-1], generator=gen, device="cuda")) * 1e-3
    size = size.repeat_interleave(BLOCK) * real                 # gradients: unlike from block to block
    s["g"] = (torch.randn(total, generator=gen, device="cuda") * size).to(gt)
    s["grads"] = views(s["g"])
    if case["op"] == "grad_norm":
        return s
    weight = torch.randn(total, generator=gen, device="cuda") * 0.05 * real
    s["p"] = weight.to(DTYPES[case["pdtype"]])
    s["params"] = views(s["p"])
    if case["master"]:
        s["w32"] = s["p"].float()
        s["masters"] = views(s["w32"])
    s["stats"] = torch.tensor([2.0, 0.5, 0.0, 0.0], device="cuda")     # a clipped step
    fresh = case["step"] == 1
    m = torch.randn(total, generator=gen, device="cuda") * size * (0.0 if fresh else 0.3)
    r = (torch.rand(total, generator=gen, device="cuda") + 0.5) * size * (0.0 if fresh else 1.0)
    if case["op"] == "adamw32":
        s["m"], s["v"] = m, r * r
        s["exp_avgs"], s["exp_avg_sqs"] = views(s["m"]), views(s["v"])
    else:
        for key, x in (("m", m), ("r", r)):
            top = x.abs().reshape(-1, BLOCK).amax(1)
            s[key + "_scale"] = top / E4M3_MAX
            inv = torch.where(top > 0, E4M3_MAX / top, torch.zeros_like(top))
            s[key] = (x.reshape(-1, BLOCK) * inv[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(
                torch.float8_e4m3fn).reshape(-1)
            s[key + "_codes"] = views(s[key])
            s[key + "_scales"] = [s[key + "_scale"][a:b] for a, b in zip(starts, starts[1:])]
        # which tensor a block belongs to, and which of its blocks it is
        count = torch.tensor(blocks, device="cuda")
        s["tensor"] = torch.arange(len(sizes), device="cuda").repeat_interleave(count)
        s["block"] = (torch.arange(starts[-1], device="cuda")
                      - torch.tensor(starts[:-1], device="cuda")[s["tensor"]])
        s["seed"] = int(seed) & 0xFFFF
    return s


# ---------------------------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)[s["case"]["op"]](s)


def _ln_fwd(s):
    x = s["x"].float()
    mean = x.mean(s["dim"], keepdim=True)
    x = x - mean
    rstd = 1.0 / (x.square().mean(s["dim"], keepdim=True) + EPS_LN).sqrt()
    y = x * rstd * s["weight"].float().reshape(s["wide"]) + s["bias"].float().reshape(s["wide"])
    return {"y": y.to(s["x"].dtype), "mean": mean.reshape(-1), "rstd": rstd.reshape(-1)}


def _per_position(s, v):
    """mean or rstd, one value a position, against x."""
    shape = list(s["x"].shape)
    shape[s["dim"]] = 1
    return v.reshape(shape)


def _ln_bwd(s):
    dim, wt = s["dim"], s["weight"].dtype
    rest = [d for d in range(s["x"].dim()) if d != dim % s["x"].dim()]
    dy, rstd = s["grad"].float(), _per_position(s, s["rstd"])
    xh = (s["x"].float() - _per_position(s, s["mean"])) * rstd
    a = dy * s["weight"].float().reshape(s["wide"])
    dx = rstd * (a - a.mean(dim, keepdim=True) - xh * (a * xh).mean(dim, keepdim=True))
    return {"dx": dx.to(s["x"].dtype), "dw": (dy * xh).sum(rest).to(wt), "db": dy.sum(rest).to(wt)}


def _update(s, m, r):
    """The parameters' part of the step, from the new moments (r = sqrt of the second)."""
    b1, b2 = HYPER["betas"]
    t = s["case"]["step"]
    bc1, bc2 = -math.expm1(t * math.log(b1)), -math.expm1(t * math.log(b2))
    w = s["w32"] if "w32" in s else s["p"].float()
    w = (w * (1.0 - HYPER["lr"] * HYPER["weight_decay"])
         - (HYPER["lr"] / bc1) * m / (r * (1.0 / math.sqrt(bc2)) + HYPER["eps"]))
    if "w32" in s:
        s["w32"].copy_(w)
    s["p"].copy_(w)
    return {k: s[k] for k in ("p", "w32") if k in s}


def _adamw32(s):
    b1, b2 = HYPER["betas"]
    g = s["g"].float() * s["stats"][1]
    s["m"].mul_(b1).add_(g * (1.0 - b1))
    s["v"].mul_(b2).add_(g.square() * (1.0 - b2))
    out = _update(s, s["m"], s["v"].sqrt())
    return {**out, "m": s["m"], "v": s["v"]}


def _mix(x):
    x = x ^ (x >> 16)
    x = (x * 0xBB67AE85) & M32
    x = x ^ (x >> 15)
    x = (x * 0x6A09E667) & M32
    return x ^ (x >> 16)


def _random(s):
    """32 bits for every value: a hash of (seed, step, tensor, block, place in the block)."""
    key = _mix((s["seed"] + s["case"]["step"] * 0x9E3779B1 + s["tensor"] * 0x85EBCA6B) & M32)
    key = _mix((key + s["block"] * 0xC2B2AE35) & M32)
    h = (key[:, None] + torch.arange(BLOCK, device="cuda") * 0x9E3779B1) & M32
    h = h ^ (h >> 16)
    h = (h * 0xBB67AE85) & M32
    return (h ^ (h >> 15)).to(torch.int64)


def _to_e4m3(x, top, bits16, floor):
    """x [blocks, 256] over the blocks' scales top / 448, rounded up or down by 16 random bits;
    `floor`: what is above zero stays above zero."""
    inv = torch.where(top > 0, E4M3_MAX / top, torch.zeros_like(top))
    a = (x.abs() * inv[:, None]).clamp(max=E4M3_MAX)
    small = a < 2.0 ** -6                       # below: e4m3 is evenly spaced
    code = torch.where(small, a + 2.0 ** -6, a).view(torch.int32)
    code = ((code + (bits16 * 16 + 8).to(torch.int32)) >> 20) - torch.where(small, 968, 960).to(torch.int32)
    code = code.clamp(max=0x7E)
    if floor:
        code = torch.where((x > 0) & (code < 1), torch.ones_like(code), code)
    code = code | torch.where(x < 0, 0x80, 0).to(torch.int32)
    return code.to(torch.uint8).view(torch.float8_e4m3fn).reshape(-1)


def _adamw8(s):
    b1, b2 = HYPER["betas"]
    g = (s["g"].float() * s["stats"][1]).reshape(-1, BLOCK)
    m = s["m"].float().reshape(-1, BLOCK) * s["m_scale"][:, None] * b1 + g * (1.0 - b1)
    r = s["r"].float().reshape(-1, BLOCK) * s["r_scale"][:, None]
    r = (r.square() * b2 + g.square() * (1.0 - b2)).sqrt()
    out = _update(s, m.reshape(-1), r.reshape(-1))
    h = _random(s)
    for key, x, bits in (("m", m, h & 0xFFFF), ("r", r, h >> 16)):
        top = x.abs().amax(1)
        s[key].copy_(_to_e4m3(x, top, bits, key == "r"))
        s[key + "_scale"].copy_(top / E4M3_MAX)
        out[key], out[key + "_scale"] = s[key], s[key + "_scale"]
    return out


def _grad_norm(s):
    norm = s["g"].double().square().sum().sqrt()
    coef = (1.0 / (norm + 1e-6)).clamp(max=1.0)
    bad = (~torch.isfinite(norm)).double()
    return torch.stack([norm, coef, bad, torch.zeros_like(bad)]).float()


def _own_ln_fwd(s):
    from ganet_amd import norm
    y, mean, rstd = norm.layer_norm_forward(s["x"], s["weight"], s["bias"], eps=EPS_LN,
                                            channel_dim=s["dim"])
    return {"y": y, "mean": mean, "rstd": rstd}


def _own_ln_bwd(s):
    from ganet_amd import norm
    dx, dw, db = norm.layer_norm_backward(s["x"], s["weight"], s["grad"], s["mean"], s["rstd"],
                                          channel_dim=s["dim"])
    return {"dx": dx, "dw": dw, "db": db}


def _own_adamw32(s):
    from ganet_amd import optim
    optim.adamw_step(s["params"], s["grads"], s["exp_avgs"], s["exp_avg_sqs"],
                     step=s["case"]["step"], masters=s.get("masters"), grad_stats=s["stats"],
                     **HYPER)
    return {k: s[k] for k in ("p", "w32", "m", "v") if k in s}


def _own_adamw8(s):
    from ganet_amd import optim
    optim.adamw_step_8bit(s["params"], s["grads"], s["m_codes"], s["r_codes"], s["m_scales"],
                          s["r_scales"], step=s["case"]["step"], seed=s["seed"],
                          masters=s.get("masters"), grad_stats=s["stats"], **HYPER)
    return {k: s[k] for k in ("p", "w32", "m", "m_scale", "r", "r_scale") if k in s}


def _own_grad_norm(s):
    from ganet_amd import optim
    return optim.grad_norm(s["grads"], max_norm=1.0)


_plain = {"ln_fwd": _ln_fwd, "ln_bwd": _ln_bwd, "adamw32": _adamw32, "adamw8": _adamw8,
          "grad_norm": _grad_norm}
_own = {"ln_fwd": _own_ln_fwd, "ln_bwd": _own_ln_bwd, "adamw32": _own_adamw32,
        "adamw8": _own_adamw8, "grad_norm": _own_grad_norm}


# ---------------------------------------------------------------------------------- work
def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if case["op"] in ("ln_fwd", "ln_bwd"):
        n = case["n"] if case["layout"] == "rows" else case["b"] * case["h"] * case["w"]
        values, sx, sw = n * case["c"], size[case["dtype"]], size[case["wdtype"]]
        if case["op"] == "ln_fwd":
            return {"bytes": 2 * values * sx + 2 * case["c"] * sw + 8 * n, "flops": 8 * values}
        return {"bytes": 3 * values * sx + 3 * case["c"] * sw + 8 * n, "flops": 14 * values}
    values = sum(_sizes(case))
    gs = size[case["gdtype"]]
    if case["op"] == "grad_norm":
        return {"bytes": values * gs + 16, "flops": 2 * values}
    ps = size[case["pdtype"]]
    weights = 8 + ps if case["master"] else 2 * ps
    if case["op"] == "adamw32":
        return {"bytes": values * (weights + gs + 16), "flops": 15 * values}
    return {"bytes": values * (weights + gs + 4 + 16 / BLOCK), "flops": 40 * values}


# ---------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "grad_norm":
        total = torch.linalg.vector_norm(s["g"], dtype=torch.float64)
        coef = torch.minimum(torch.ones_like(total), 1.0 / (total + 1e-6))
        return torch.cat([total[None], coef[None], torch.zeros(2, dtype=torch.float64, device="cuda")])
    if case["op"] in ("ln_fwd", "ln_bwd"):
        if s["x"].numel() > 1 << 28:
            return None
        # positions as rows, channels last
        x = s["x"].double().movedim(s["dim"], -1)
        shape, c = x.shape, case["c"]
        x, w = x.reshape(-1, c), s["weight"].double()

        def back(v):
            return v.reshape(shape).movedim(-1, s["dim"])

        if case["op"] == "ln_fwd":
            mean = x.sum(1) / c
            var = (x * x).sum(1) / c - mean * mean
            rstd = (var + EPS_LN) ** -0.5
            y = ((x - mean[:, None]) * rstd[:, None]) * w + s["bias"].double()
            return {"y": back(y), "mean": mean, "rstd": rstd}
        dy = s["grad"].double().movedim(s["dim"], -1).reshape(-1, c)
        mean, rstd = s["mean"].double()[:, None], s["rstd"].double()[:, None]
        xh = (x - mean) * rstd
        both = dy * xh
        along = torch.mv(dy, w)[:, None] / c                     # mean of w dy
        across = torch.mv(both, w)[:, None] / c                  # mean of w dy xh
        ones = torch.ones(x.shape[0], dtype=torch.float64, device="cuda")
        return {"dx": back(rstd * (dy * w - along - xh * across)),
                "dw": torch.mv(both.t(), ones), "db": torch.mv(dy.t(), ones)}
    # the step, a value at a time in 64 bits
    (b1, b2), lr = HYPER["betas"], HYPER["lr"]
    t = case["step"]
    g = s["g"].double() * 0.5
    old = s["w32"].double() if case["master"] else s["p"].double()
    if case["op"] == "adamw32":
        m = s["m"].double() + (1 - b1) * (g - s["m"].double())
        v = s["v"].double() + (1 - b2) * (g * g - s["v"].double())
        out = {"m": m, "v": v}
    else:
        per = {k: s[k + "_scale"].double().repeat_interleave(BLOCK) for k in ("m", "r")}
        m0, r0 = s["m"].double() * per["m"], s["r"].double() * per["r"]
        m = m0 + (1 - b1) * (g - m0)
        v = r0 * r0 + (1 - b2) * (g * g - r0 * r0)
        out = {}
        h = _random(s).reshape(-1)
        for key, x, bits in (("m", m, h & 0xFFFF), ("r", v.sqrt(), h >> 16)):
            scale = x.abs().reshape(-1, BLOCK).max(1).values / E4M3_MAX
            y = x.abs() / scale.repeat_interleave(BLOCK).clamp(min=1e-300)
            step = 2.0 ** (torch.floor(torch.log2(y.clamp(min=2.0 ** -6))).clamp(min=-6) - 3)
            q = torch.floor(y / step + (bits.double() + 0.5) / 65536) * step
            if key == "r":
                q = torch.where(x > 0, q.clamp(min=2.0 ** -9), q)
            out[key], out[key + "_scale"] = (q.clamp(max=E4M3_MAX) * x.sign()), scale
    hat = m / (1 - b1 ** t) / ((v / (1 - b2 ** t)).sqrt() + HYPER["eps"])
    new = old - lr * (HYPER["weight_decay"] * old + hat)
    out["p"] = new
    if case["master"]:
        out["w32"] = new
    return out
