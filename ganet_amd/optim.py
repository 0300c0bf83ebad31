"""The AdamW step over many tensors at once, and the norm of all gradients, on the gfx950 C-ABI
(csrc/optim.hip).

    m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
    p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)

No counterpart in the reference, whose training loop takes its optimizer from torch
(mmdet/apis/train.py:83-168).

  AdamW             torch.optim.Optimizer; states in 32 or 8 bits, float32 masters of 16-bit
                    weights, clipping by the norm of all gradients without a pass or a wait of
                    its own; register_with_mmcv() offers it to an `optimizer` config
  adamw_step, adamw_step_8bit, grad_norm    the raw calls

Parameters and gradients are float32, bfloat16 or float16, dense in any order (channels_last
weights too).  CPU tensors raise NotImplementedError.
"""
import ctypes
import math
from array import array
from itertools import chain
from operator import attrgetter

import torch

from . import _lib
from .dcn import _DTYPES

BLOCK = _lib.GANET_STATE_BLOCK
_PLACE = 0x85EBCA6B           # a place further in the list adds this to the seed of the random words


_ptrs, _sizes, _gpus = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.get_device
_dtypes, _shapes, _plain = attrgetter("dtype"), attrgetter("shape"), torch.Tensor.is_contiguous


def _dense(t):
    """Whether t's values fill their memory without gaps or overlaps, in any order."""
    if t.is_contiguous():
        return True
    expect = 1
    for step, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if step != expect:
            return False
        expect *= size
    return True


def _same_order(a, b):
    """Whether two dense tensors of one shape lie alike in memory."""
    if a.shape != b.shape:
        return False
    if a.is_contiguous() and b.is_contiguous():
        return True
    return all(x == y for x, y, n in zip(a.stride(), b.stride(), a.shape) if n != 1)


def _overlap(spans):
    """Whether two of the (address, bytes) share a byte."""
    end = 0
    for begin, size in sorted(spans):
        if size:
            if begin < end:
                return True
            end = begin + size
    return False


def _one(tensors, what, index, dtype=None):
    """Checks that a list's tensors share one GPU and dtype; returns the dtype."""
    gpus = set(map(_gpus, tensors))
    if gpus != {index} or index < 0:
        if -1 in gpus:
            raise NotImplementedError
        raise ValueError("adamw: %s on GPUs %s, parameters on %d" % (what, sorted(gpus), index))
    found = set(map(_dtypes, tensors))
    if len(found) != 1 or (dtype is not None and dtype not in found):
        raise TypeError("adamw: %s of dtypes %s%s" % (
            what, ", ".join(map(str, found)), "" if dtype is None else ", expected %s" % dtype))
    return found.pop()


def _like_params(params, shapes, plain, tensors, what):
    """Checks that `tensors` have the parameters' shapes and memory order."""
    if list(map(_shapes, tensors)) == shapes and plain and all(map(_plain, tensors)):
        return
    for p, t in zip(params, tensors):
        if not _same_order(p, t):
            raise ValueError("adamw: %s of shape %s and strides %s for a parameter of shape %s and "
                             "strides %s" % (what, tuple(t.shape), t.stride(), tuple(p.shape),
                                             p.stride()))


def _table(params, grads, avgs, seconds, avg_scales, second_scales, masters, bits):
    """(GPU, parameters' dtype, gradients' dtype, rows of ganet_step_tensor, what they point into):
    any order of memory, and the errors of what cannot be stepped.  Plain lists (contiguous, nothing
    wrong) do not come here: _lib.host().step reads them."""
    n = len(params)
    for what, ts in (("gradients", grads), ("exp_avgs", avgs), ("second moments", seconds),
                     ("masters", masters), ("scales", avg_scales), ("scales", second_scales)):
        if ts is not None and len(ts) != n:
            raise ValueError("adamw: %d %s for %d parameters" % (len(ts), what, n))
    index = params[0].get_device()
    pdtype = _one(params, "parameters", index)
    gdtype = _one(grads, "gradients", index)
    for t in (pdtype, gdtype):
        if t not in _DTYPES:
            raise TypeError("adamw: unsupported dtype %s" % t)
    state = torch.float32 if bits == 32 else torch.float8_e4m3fn
    _one(avgs, "states", index, state)
    _one(seconds, "states", index, state)
    shapes, plain = list(map(_shapes, params)), all(map(_plain, params))
    if not plain:
        for p in params:
            if not _dense(p):
                raise ValueError("adamw: a parameter of shape %s and strides %s is not dense"
                                 % (tuple(p.shape), p.stride()))
    _like_params(params, shapes, plain, avgs, "a state")
    _like_params(params, shapes, plain, seconds, "a state")
    sizes = list(map(_sizes, params))
    none = [0] * n
    columns = [list(map(_ptrs, params)), None, list(map(_ptrs, avgs)), list(map(_ptrs, seconds)),
               none, none, none, sizes]
    written = list(chain(params, avgs, seconds))
    if masters is not None:
        if pdtype == torch.float32:
            raise TypeError("adamw: masters of float32 parameters")
        _one(masters, "masters", index, torch.float32)
        _like_params(params, shapes, plain, masters, "a master")
        columns[6] = list(map(_ptrs, masters))
        written += masters
    if bits == 8:
        blocks = [-(-k // BLOCK) for k in sizes]
        for at, ts in ((4, avg_scales), (5, second_scales)):
            _one(ts, "scales", index, torch.float32)
            if list(map(_sizes, ts)) != blocks or not all(map(_plain, ts)):
                raise ValueError("adamw: a dense scale for each %d values of a parameter is wanted"
                                 % BLOCK)
            columns[at] = list(map(_ptrs, ts))
        written += chain(avg_scales, second_scales)
    # gradients in their parameters' order
    if list(map(_shapes, grads)) != shapes:
        raise ValueError("adamw: a gradient's shape is not its parameter's")
    if not (plain and all(map(_plain, grads))):
        grads = [g if _same_order(p, g) else torch.empty_like(p, dtype=gdtype).copy_(g)
                 for p, g in zip(params, grads)]
    columns[1] = list(map(_ptrs, grads))
    if _overlap([(t.data_ptr(), t.nbytes) for t in written]):
        raise ValueError("adamw: tensors in the lists share memory, or one is there twice")
    rows = array("Q", chain.from_iterable(zip(*columns))).tobytes()
    return index, _DTYPES[pdtype], _DTYPES[gdtype], rows, grads


def _step(params, grads, avgs, seconds, avg_scales, second_scales, bits, step, lr, betas, eps,
          weight_decay, masters, grad_stats, skip_nonfinite, seed):
    n = len(params)
    lists = (params, grads, avgs, seconds, avg_scales, second_scales, masters)
    if n and type(step) is int and not torch.is_tensor(lr) and torch.is_tensor(params[0]):
        index = params[0].get_device()
        if index >= 0 and torch.cuda.current_device() == index:
            rc = _lib.host().adamw(_lib.address("ganet_adamw_step"), *lists, BLOCK, bits, step, lr,
                                   betas[0], betas[1], eps, weight_decay, grad_stats,
                                   skip_nonfinite, int(seed), index, _lib.raw_stream(index))
            if rc is not None:
                if rc:
                    _lib.check(rc, "ganet_adamw_step")
                return
    # a step or lr on the device, another order of memory, another GPU, or something wrong
    found = _lib.host().step(*lists, BLOCK)
    if found is not None and found[3] == bits:
        index, ptype, gtype, _, rows = found
    elif n or any(lists[1:]):
        if not n:
            raise ValueError("adamw: no parameters")
        index, ptype, gtype, rows, grads = _table(*lists, bits)
    else:
        return
    h = _lib.AdamwParams(ptype, gtype, bits, 1 if skip_nonfinite else 0, 0, int(seed) & 0xFFFFFFFF,
                         0, 0.0, betas[0], betas[1], eps, weight_decay)
    if torch.is_tensor(step):
        h.step_device = _scalar(step, torch.int64, index, "step")
    else:
        h.step = int(step)
    if torch.is_tensor(lr):
        h.lr_device = _scalar(lr, torch.float32, index, "lr")
    else:
        h.lr = lr
    if grad_stats is not None:
        if (grad_stats.dtype != torch.float32 or grad_stats.numel() != 4
                or grad_stats.get_device() != index or not grad_stats.is_contiguous()):
            raise ValueError("adamw: grad_stats is the float32 [4] tensor of grad_norm")
        h.grad_stats = grad_stats.data_ptr()
    rc = _lib.call(index, _lib.lib().ganet_adamw_step, rows, n, ctypes.byref(h))
    if rc:
        _lib.check(rc, "ganet_adamw_step")
    for ts in (params, masters):
        if ts is not None:
            _lib.host().written(list(ts))


def _scalar(t, dtype, index, what):
    if t.dtype != dtype or t.numel() != 1 or t.get_device() != index:
        raise ValueError("adamw: %s as a tensor is one %s on GPU %d" % (what, dtype, index))
    return t.data_ptr()


def adamw_step(params, grads, exp_avgs, exp_avg_sqs, step, lr=1e-3, betas=(0.9, 0.999), eps=1e-8,
               weight_decay=1e-2, masters=None, grad_stats=None, skip_nonfinite=True):
    """One step on all `params`, in place; exp_avgs and exp_avg_sqs are float32.

    step: t, 1 at the first step (or a one-element int64 tensor on the device, as a captured graph
    needs it; lr likewise as float32).  masters: float32 copies of 16-bit parameters: these are
    stepped and the parameters get them rounded; without masters 16-bit parameters are stepped in
    float32 and rounded to nearest, and updates below half a step of theirs are lost.
    grad_stats: what grad_norm returned: gradients are multiplied by its coefficient on the way,
    and with skip_nonfinite nothing changes where the norm is not finite.  Parameters in one call
    share one dtype, gradients another; a gradient in another memory order is copied first."""
    _step(params, grads, exp_avgs, exp_avg_sqs, None, None, 32, step, lr, betas, eps, weight_decay,
          masters, grad_stats, skip_nonfinite, 0)


def adamw_step_8bit(params, grads, exp_avgs, exp_rms, avg_scales, rms_scales, step, seed=0,
                    lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, masters=None,
                    grad_stats=None, skip_nonfinite=True):
    """adamw_step with states in 8 bits: exp_avgs (m) and exp_rms (the root of the second moment)
    are float8_e4m3fn of the parameter's shape, in units of avg_scales / rms_scales, one float32
    for each 256 values in memory order (state_8bit makes them).  States are rounded up or down at
    random, by a hash of (seed, step, the parameter's place in the list, the value's place in it):
    the same inputs give the same bits.  Several calls of one step need seeds of their own, or their
    i-th parameters are rounded alike (AdamW counts the places on over its calls).  Parameters move
    by the moments before that rounding."""
    _step(params, grads, exp_avgs, exp_rms, avg_scales, rms_scales, 8, step, lr, betas, eps,
          weight_decay, masters, grad_stats, skip_nonfinite, seed)


def state_8bit(param):
    """(exp_avg, exp_rms, avg_scale, rms_scale) of zeros for adamw_step_8bit."""
    codes = [torch.zeros_like(param, dtype=torch.uint8).view(torch.float8_e4m3fn)
             for _ in range(2)]
    scales = [torch.zeros(-(-param.numel() // BLOCK), dtype=torch.float32, device=param.device)
              for _ in range(2)]
    return tuple(codes + scales)


def grad_norm(grads, max_norm=None, inv_scale=1.0, out=None):
    """The 2-norm of all gradients together, as a float32 [4] tensor on their device:
    [norm, coefficient, 1 where the norm is not finite, 0].  norm is of inv_scale * gradients
    (inv_scale: one over a loss scale); coefficient = inv_scale * min(1, max_norm / (norm + 1e-6)),
    0 where the norm is not finite.  Nothing waits for the device; adamw_step and
    adamw_step_8bit take the tensor as grad_stats.  Gradients of several dtypes may be mixed."""
    grads = list(grads)
    n = len(grads)
    max_norm = math.inf if max_norm is None else float(max_norm)
    if not max_norm >= 0 or not math.isfinite(inv_scale):
        raise ValueError("grad_norm: max_norm %r, inv_scale %r" % (max_norm, inv_scale))
    if out is None and n and torch.is_tensor(grads[0]):
        index = grads[0].get_device()
        if index >= 0 and torch.cuda.current_device() == index:
            stats = _lib.host().grad_norm(_lib.address("ganet_grad_norm_workspace_bytes"),
                                          _lib.address("ganet_grad_norm"), grads, max_norm,
                                          inv_scale, index, _lib.raw_stream(index))
            if torch.is_tensor(stats):
                return stats
            if stats is not None:
                _lib.check(stats, "ganet_grad_norm")
    found = _lib.host().grads(grads)
    if found is not None:
        index, ptrs, numel, dtypes = found
    else:
        index, ptrs, numel, dtypes, grads = _read_grads(grads, out)
    L = _lib.lib()
    if out is None:
        out = torch.empty(4, dtype=torch.float32, device=grads[0].device)
    elif (out.dtype != torch.float32 or out.numel() != 4 or out.get_device() != index
          or not out.is_contiguous()):
        raise ValueError("grad_norm: out is a float32 [4] tensor on the gradients' device")
    nbytes = L.ganet_grad_norm_workspace_bytes(numel, n)
    ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=out.device)
    rc = _lib.call(index, L.ganet_grad_norm, ptrs, numel, dtypes, n, max_norm, inv_scale,
                   out.data_ptr(), ws.data_ptr(), nbytes)
    if rc:
        _lib.check(rc, "ganet_grad_norm")
    return out


def _read_grads(grads, out):
    """(GPU, addresses, sizes, dtypes, tensors) of gradients that are not all contiguous, and the
    errors of what is none."""
    if out is None and not grads:
        raise ValueError("grad_norm: no gradients")
    index = (grads[0] if grads else out).get_device()
    gpus = set(map(_gpus, grads)) or {index}
    if gpus != {index} or index < 0:
        if -1 in gpus:
            raise NotImplementedError
        raise ValueError("grad_norm: gradients on GPUs %s" % sorted(gpus))
    grads = [g if _dense(g) else g.contiguous() for g in grads]
    try:
        dtypes = array("i", [_DTYPES[t] for t in map(_dtypes, grads)])
    except KeyError as e:
        raise TypeError("grad_norm: unsupported dtype %s" % e.args[0])
    return (index, array("Q", map(_ptrs, grads)).tobytes(), array("q", map(_sizes, grads)).tobytes(),
            dtypes.tobytes(), grads)


def _check_settings(lr, betas, eps, weight_decay):
    if not torch.is_tensor(lr) and not 0 <= lr < math.inf:
        raise ValueError("AdamW: lr %r" % (lr,))
    if not all(0 <= b < 1 for b in betas):
        raise ValueError("AdamW: betas %r" % (betas,))
    if not 0 <= eps < math.inf or not 0 <= weight_decay < math.inf:
        raise ValueError("AdamW: eps %r, weight_decay %r" % (eps, weight_decay))


class AdamW(torch.optim.Optimizer):
    """AdamW over the parameters of a model, a few launches a step (parameters of equal settings and
    types share one, whatever groups they are in).

    state_bits=8: moments in 8 bits (parameters of fewer than min_8bit_size values keep 32).
    master_weights: 16-bit parameters get float32 masters, made from them at their first step.
    max_grad_norm: the gradients of ALL parameters are clipped to this norm, on the way.
    skip_nonfinite: with max_grad_norm (or grad_stats given to step) a step whose gradients' norm
    is not finite changes no weight and no moment; the step number goes on.
    capturable: step numbers live on the device, so that a step captured into a HIP graph counts
    on when replayed; make one step before the capture, with gradients for the same parameters.  lr
    may be a float32 tensor on the device.  Bias corrections are formed in float32 there, so such a
    step and one that the host counts may differ in a weight's last bit.
    `grad_stats` holds the last step's grad_norm tensor."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2,
                 state_bits=32, master_weights=False, max_grad_norm=None, skip_nonfinite=True,
                 seed=0, min_8bit_size=4096, capturable=False):
        _check_settings(lr, betas, eps, weight_decay)
        if state_bits not in (32, 8):
            raise ValueError("AdamW: states of %r bits" % (state_bits,))
        if max_grad_norm is not None and not max_grad_norm >= 0:
            raise ValueError("AdamW: max_grad_norm %r" % (max_grad_norm,))
        super(AdamW, self).__init__(params, dict(lr=lr, betas=betas, eps=eps,
                                                 weight_decay=weight_decay))
        self.state_bits, self.master_weights = state_bits, master_weights
        self.max_grad_norm, self.skip_nonfinite = max_grad_norm, skip_nonfinite
        self.seed, self.min_8bit_size, self.capturable = seed, min_8bit_size, capturable
        self.grad_stats = None
        self._captured = {}               # step numbers on the device that a graph counts, by id

    def __getstate__(self):
        """Copies and pickles keep the options too (torch's own state has the groups only)."""
        kept = super(AdamW, self).__getstate__()
        for name in ("state_bits", "master_weights", "max_grad_norm", "skip_nonfinite", "seed",
                     "min_8bit_size", "capturable"):
            kept[name] = getattr(self, name)
        kept["grad_stats"], kept["_captured"] = None, {}
        return kept

    def _init_state(self, p, fresh):
        """First step of a parameter.  `fresh`: the step counters made in this call, by device."""
        if not p.is_cuda:
            raise NotImplementedError
        if p.dtype not in _DTYPES:
            raise TypeError("AdamW: unsupported dtype %s" % p.dtype)
        if not _dense(p):
            raise ValueError("AdamW: a parameter of strides %s is not dense" % (p.stride(),))
        st = {}
        if self.capturable:
            if p.device not in fresh:
                fresh[p.device] = torch.zeros((), dtype=torch.int64, device=p.device)
            st["step"] = fresh[p.device]
        else:
            st["step"] = 0
        if self.state_bits == 8 and p.numel() >= self.min_8bit_size:
            st["exp_avg"], st["exp_rms"], st["avg_scale"], st["rms_scale"] = state_8bit(p.detach())
        else:
            st["exp_avg"] = torch.zeros_like(p, dtype=torch.float32)
            st["exp_avg_sq"] = torch.zeros_like(p, dtype=torch.float32)
        if self.master_weights and p.dtype != torch.float32:
            st["master"] = p.detach().float()
        self.state[p] = st                    # whole or not at all

    def _split_counters(self, stepped, capturing):
        """Parameters share their step number on the device with all that have been stepped as often;
        those that are stepped while others of theirs have no gradient get one of their own."""
        now, users = {}, {}
        for _, p, _ in stepped:
            st = self.state.get(p, ())
            if "step" in st:
                now.setdefault(id(st["step"]), []).append(st)
        if sum(map(len, now.values())) < len(self.state):
            for st in self.state.values():
                if "step" in st:
                    at = id(st["step"])
                    users[at] = users.get(at, 0) + 1
        parted = [sts for at, sts in now.items() if len(sts) < users.get(at, 0)]
        if parted and capturing:             # the copy of the number would be part of the graph
            raise RuntimeError("AdamW: a parameter without a gradient shares its step number with some "
                               "of a captured step: make one step with the same gradients before")
        if any(id(sts[0]["step"]) in self._captured for sts in parted):
            raise RuntimeError("AdamW: a captured step counts these parameters with one number: all of "
                               "them need gradients (load_state_dict(state_dict()) forgets the graph)")
        for sts in parted:
            number = sts[0]["step"].clone()
            for st in sts:
                st["step"] = number
        if capturing:
            self._captured.update((id(sts[0]["step"]), sts[0]["step"]) for sts in now.values())

    def _call(self, calls, grad_stats, counters):
        """The raw calls of a step.  What has been stepped is counted; its numbers on the device leave
        `counters`."""
        place = 0                                 # 8-bit tensors of the calls before
        for key, (group, ps, gs, st) in calls.items():
            common = dict(lr=group["lr"], betas=group["betas"], eps=group["eps"],
                          weight_decay=group["weight_decay"], grad_stats=grad_stats,
                          masters=[s["master"] for s in st] if key[5] else None,
                          skip_nonfinite=self.skip_nonfinite)
            number = st[0]["step"] if self.capturable else key[6] + 1
            if key[4]:
                adamw_step_8bit(ps, gs, [s["exp_avg"] for s in st], [s["exp_rms"] for s in st],
                                [s["avg_scale"] for s in st], [s["rms_scale"] for s in st],
                                number, seed=self.seed + place * _PLACE, **common)
                place += len(ps)
            else:
                adamw_step(ps, gs, [s["exp_avg"] for s in st], [s["exp_avg_sq"] for s in st],
                           number, **common)
            if self.capturable:
                counters.pop(key[6], None)
            else:
                for s in st:
                    s["step"] = number

    @torch.no_grad()
    def step(self, closure=None, grad_stats=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        # groups of equal settings are one
        every, alike = [], {}
        for group in self.param_groups:
            lr = group["lr"]
            values = (("lr", id(lr)) if torch.is_tensor(lr) else lr, tuple(group["betas"]),
                      group["eps"], group["weight_decay"])
            if values not in alike:
                _check_settings(lr, *values[1:])
            first = alike.setdefault(values, group)
            every += [(first, p, p.grad) for p in group["params"] if p.grad is not None]
        if not every:
            return loss
        grads = [g for _, _, g in every]
        if any(g.is_sparse for g in grads):
            raise RuntimeError("AdamW: sparse gradients")
        capturing = every[0][1].is_cuda and torch.cuda.is_current_stream_capturing()
        if capturing:
            # the number of the step would be part of the graph, a new state its memory
            if not self.capturable:
                raise RuntimeError("AdamW: a captured step needs capturable=True")
            if any("step" not in self.state.get(p, ()) for _, p, _ in every):
                raise RuntimeError("AdamW: make one step before the capture")
        if self.capturable:
            self._split_counters(every, capturing)
        if grad_stats is None and self.max_grad_norm is not None:
            grad_stats = grad_norm(grads, self.max_grad_norm)
        self.grad_stats = grad_stats
        # one call for the parameters that share a group, a GPU, their types and their step
        fresh, counters, calls, state = {}, {}, {}, self.state
        for group, p, g in every:
            st = state.get(p)
            if st is None or "step" not in st:
                self._init_state(p, fresh)
                st = state[p]
            at = st["step"]
            if self.capturable:
                at = id(at)
                counters[at] = st["step"]
            key = (id(group), p.get_device(), p.dtype, g.dtype, "avg_scale" in st, "master" in st,
                   at)
            call = calls.get(key)
            if call is None:
                call = calls[key] = (group, [], [], [])
            call[1].append(p)
            call[2].append(g)
            call[3].append(st)
        for t in counters.values():
            t.add_(1)
        try:
            self._call(calls, grad_stats, counters)
        except Exception:
            for t in counters.values():           # of what has not been stepped
                t.sub_(1)
            raise
        return loss

    def load_state_dict(self, state_dict):
        """States keep the types they were saved in (torch would cast them to the parameter's); 16-bit
        moments, as torch's AdamW keeps for 16-bit parameters, become float32, and with
        master_weights a state without a master gets one from the parameter."""
        super(AdamW, self).load_state_dict(state_dict)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        ps = [p for group in self.param_groups for p in group["params"]]
        counters = {}
        for i, p in zip(ids, ps):
            saved = state_dict["state"].get(i, {})
            for name, value in saved.items():
                if name == "step":
                    value = int(value)
                    if self.capturable:        # one counter for the parameters that share a number
                        key = (p.device, value)
                        if key not in counters:
                            counters[key] = torch.full((), value, dtype=torch.int64,
                                                       device=p.device)
                        value = counters[key]
                elif name in _SCALES.values():
                    continue                   # comes with its codes
                elif torch.is_tensor(value) and value.dtype == torch.float8_e4m3fn:
                    scale = _SCALES[name]
                    value, self.state[p][scale] = _codes_like(p, value.detach(), saved[scale].detach(),
                                                              name == "exp_rms")
                elif torch.is_tensor(value):
                    value = _values_like(p, value.float() if name in ("exp_avg", "exp_avg_sq") else value)
                self.state[p][name] = value
            if saved and self.master_weights and p.dtype != torch.float32 and "master" not in saved:
                self.state[p]["master"] = p.detach().float()


_SCALES = dict(exp_avg="avg_scale", exp_rms="rms_scale")      # of the states in 8 bits


def _values_like(p, value):
    """A copy of a state's values in the parameter's memory order."""
    if value.shape != p.shape:
        raise ValueError("AdamW: a saved state of shape %s for a parameter of shape %s"
                         % (tuple(value.shape), tuple(p.shape)))
    return torch.empty_like(p, dtype=value.dtype).copy_(value.detach())


def _codes_like(p, codes, scale, root):
    """Copies of a state's codes and scales in the parameter's memory order.  A scale belongs to 256
    values in memory order: where the state was saved from another one its values are divided into
    other blocks, each rounded to nearest in its new scale; a root above zero stays above zero."""
    codes = codes.to(p.device, copy=True)
    scale = scale.to(p.device, copy=True)
    if _same_order(p, codes):
        return codes, scale
    if codes.shape != p.shape or not _dense(codes) or not _dense(p):
        raise ValueError("AdamW: a saved state of shape %s and strides %s for a parameter of shape %s and "
                         "strides %s" % (tuple(codes.shape), codes.stride(), tuple(p.shape), p.stride()))
    n = p.numel()

    def flat(t):
        return t.as_strided((n,), (1,))

    saved = torch.empty_strided(codes.shape, codes.stride(), dtype=torch.float32, device=p.device)
    flat(saved).copy_(flat(codes.view(torch.uint8)).view(torch.float8_e4m3fn).float()
                      * scale.repeat_interleave(BLOCK)[:n])
    x = torch.nn.functional.pad(flat(_values_like(p, saved)), (0, -n % BLOCK)).reshape(-1, BLOCK)
    top = torch.where(x.isnan(), torch.zeros_like(x), x.abs()).amax(1)
    top = torch.where(top < 2.0 ** -110, torch.zeros_like(top), top)      # as the step holds such blocks
    y = (x * torch.where(top > 0, 448 / top, torch.zeros_like(top))[:, None]).clamp(-448, 448)
    if root:
        y = torch.where((x > 0) & (y < 2.0 ** -9), torch.full_like(y, 2.0 ** -9), y)
    kept = torch.empty_like(p, dtype=torch.uint8)
    flat(kept).copy_(y.reshape(-1)[:n].to(torch.float8_e4m3fn).view(torch.uint8))
    return kept.view(torch.float8_e4m3fn), top / 448


def register_with_mmcv(force=False):
    """Register AdamW as 'HipAdamW' in mmcv's OPTIMIZERS (optimizer=dict(type='HipAdamW', ...)).
    An explicit call, as in ganet_amd.dcn; False when mmcv is absent."""
    try:
        from mmcv.runner import OPTIMIZERS
    except Exception:
        return False
    OPTIMIZERS.register_module('HipAdamW', module=AdamW, force=force)
    return True
