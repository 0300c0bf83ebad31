"""Layer norm over channels, forward and backward, on the gfx950 C-ABI (csrc/layer_norm.hip).

    y = (x - mean) / sqrt(var + eps) * weight + bias

over the channels of every position of a map (NCHW or channels_last, the layouts of
ganet_amd.dcn) or over the last dimension of rows of tokens.  No counterpart in the reference,
whose models normalise with torch's and mmcv's layers (`norm_cfg` of the ConvModules,
mmdet/models/dense_heads/lanepoints_conv.py:77-126).

  layer_norm              differentiable function
  LayerNorm, LayerNorm2d  modules; register_with_mmcv() offers 'LN2d' to a `norm_cfg`
  layer_norm_forward, layer_norm_backward   the raw calls

float32, bfloat16 and float16 tensors; weight and bias of the tensor's type or of another of the
three.  Sums are float32, each output is rounded once.  The gradients of weight and bias are added
up in a fixed order: the same inputs give the same bits.  CPU tensors raise NotImplementedError.
"""
import ctypes

import torch
import torch.nn as nn
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .dcn import _DTYPES, _is_channels_last


def _rows_stride(t):
    """Values from one row (last dimension) to the next where all rows are evenly spaced and
    dense, else None."""
    c = t.shape[-1]
    if c > 1 and t.stride(-1) != 1:
        return None
    stride = None
    span = 1                                   # rows that the dimensions seen so far hold
    for size, step in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if stride is None:
            stride = step
        elif step != stride * span:
            return None
        span *= size
    if stride is None:
        return c
    return stride if stride >= c else None     # smaller: an expanded or overlapping view


class _Layout(object):
    """How a tensor's channels lie in memory, in the order that the tensor itself suggests:
    `outer` rows (inner = 1) or images of `inner` positions, `stride` values apart."""
    __slots__ = ("x", "dim", "C", "positions", "outer", "inner", "stride", "channels_last")

    def __init__(self, x, channel_dim):
        shape = x.shape
        dims = len(shape)
        dim = channel_dim + dims if channel_dim < 0 else channel_dim
        if not 0 <= dim < dims:
            raise IndexError("layer_norm: channel_dim %d of a %d-dimensional tensor"
                             % (channel_dim, dims))
        C = shape[dim]
        if C < 1:
            raise ValueError("layer_norm: no channels in %s" % (tuple(shape),))
        self.dim, self.C = dim, C
        self.positions = n = x.numel() // C
        self.channels_last = False
        inner = 1
        if dim != dims - 1 and n:
            for size in shape[dim + 1:]:
                inner *= size
            if dim == 1 and inner > 1 and _is_channels_last(x):
                self.channels_last, inner = True, 1
        self.inner, self.outer = inner, n // inner
        self.x, self.stride = self.fit(x)

    def fit(self, t):
        """(t in this order, values between its rows or images), copied where it is in another."""
        one = self.C * self.inner
        if self.channels_last:
            return (t if _is_channels_last(t)
                    else t.contiguous(memory_format=torch.channels_last)), one
        if t.is_contiguous():
            return t, one
        if self.dim == t.dim() - 1:
            stride = _rows_stride(t)
            if stride is not None:
                return t, stride
        elif self.dim == 1 and t.shape[0] > 0 and t[0].is_contiguous():
            if t.shape[0] == 1:
                return t, one
            if t.stride(0) >= one:
                return t, t.stride(0)
        return t.contiguous(), one

    def like(self, x):
        """An output of the input's memory format."""
        if self.channels_last:
            return torch.empty_like(x, memory_format=torch.channels_last)
        return torch.empty_like(x, memory_format=torch.contiguous_format)


def _weight_dtype(x, tensors, C):
    """The (one) dtype of weight and bias, the input's without them; checks them."""
    dtype = None
    for name, t in tensors:
        if t is None:
            continue
        if t.dtype not in _DTYPES:
            raise TypeError("layer_norm: unsupported dtype %s of the %s" % (t.dtype, name))
        if dtype is not None and t.dtype != dtype:
            raise TypeError("layer_norm: weight and bias of unlike dtypes")
        if t.get_device() != x.get_device():
            raise ValueError("layer_norm: %s on %s, input on %s" % (name, t.device, x.device))
        if t.dim() != 1 or t.numel() != C:
            raise ValueError("layer_norm: %s of shape %s for %d channels"
                             % (name, tuple(t.shape), C))
        dtype = t.dtype
    return dtype or x.dtype


def _check_input(x):
    if not x.is_cuda:
        raise NotImplementedError
    if x.dtype not in _DTYPES:
        raise TypeError("layer_norm: unsupported dtype %s" % x.dtype)


def _dense(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _forward(input, weight, bias, eps, channel_dim, stats):
    if not eps >= 0:
        raise ValueError("layer_norm: eps %r" % (eps,))
    index = input.get_device()
    if index >= 0 and torch.cuda.current_device() == index:
        out = _lib.host().layer_norm_forward(_lib.address("ganet_layer_norm_forward"), input, weight,
                                             bias, eps, channel_dim, stats, _lib.raw_stream(index))
        if type(out) is tuple:
            return out
        if out is not None:
            _lib.check(out, "ganet_layer_norm_forward")
    # another order of memory, nothing to do, or something wrong
    lay = _Layout(input, channel_dim)
    _check_input(input)
    wdtype = _weight_dtype(input, (("weight", weight), ("bias", bias)), lay.C)
    L = _lib.lib()
    x, weight, bias = lay.x, _dense(weight), _dense(bias)
    p = _lib.LayerNormParams(lay.outer, lay.inner, lay.stride, lay.C * lay.inner, 0, lay.C,
                             _DTYPES[x.dtype], _DTYPES[wdtype], eps)
    out = lay.like(x)
    mean = rstd = None
    if stats:
        mean = torch.empty(lay.positions, dtype=torch.float32, device=x.device)
        rstd = torch.empty_like(mean)
    rc = _lib.call(x.get_device(), L.ganet_layer_norm_forward, x.data_ptr(), _ptr(weight),
                   _ptr(bias), out.data_ptr(), _ptr(mean), _ptr(rstd), ctypes.byref(p))
    if rc:
        _lib.check(rc, "ganet_layer_norm_forward")
    return out, mean, rstd


def layer_norm_forward(input, weight=None, bias=None, eps=1e-5, channel_dim=-1):
    """Raw forward: (out, mean, rstd).  `input` of any shape; `channel_dim` is normalised
    (-1: rows of tokens, 1: the channels of a [B, C, H, W] map, contiguous or channels_last).
    `out` has the memory format of `input`; mean and rstd are float32, one value a position (the
    input's shape without channel_dim, flattened), for layer_norm_backward."""
    return _forward(input, weight, bias, eps, channel_dim, True)


def layer_norm_backward(input, weight, grad_output, mean, rstd, channel_dim=-1,
                        need_input=True, need_weight=True, need_bias=True):
    """Raw backward: (grad_input, grad_weight, grad_bias), None for what is not asked for.
    grad_input has the memory format of `input`; grad_weight and grad_bias are [C] of the weight's
    dtype (the input's without a weight)."""
    index = input.get_device()
    if index >= 0 and torch.cuda.current_device() == index:
        out = _lib.host().layer_norm_backward(
            _lib.address("ganet_layer_norm_backward_workspace_bytes"),
            _lib.address("ganet_layer_norm_backward"), input, weight, grad_output, mean, rstd,
            channel_dim, bool(need_input) + 2 * bool(need_weight) + 4 * bool(need_bias),
            _lib.raw_stream(index))
        if type(out) is tuple:
            return out
        if out is not None:
            _lib.check(out, "ganet_layer_norm_backward")
    lay = _Layout(input, channel_dim)
    if not grad_output.is_cuda:
        raise NotImplementedError
    _check_input(input)
    wdtype = _weight_dtype(input, (("weight", weight),), lay.C)
    if grad_output.shape != input.shape:
        raise ValueError("layer_norm: grad_output of shape %s for an input of shape %s"
                         % (tuple(grad_output.shape), tuple(input.shape)))
    for t in (grad_output, mean, rstd):
        if t.get_device() != index:
            raise ValueError("layer_norm: tensors on %s and %s" % (t.device, input.device))
    for t in (mean, rstd):
        if t.dtype != torch.float32 or t.numel() != lay.positions or not t.is_contiguous():
            raise ValueError("layer_norm: mean and rstd are dense float32, one value a position")
    if not (need_input or need_weight or need_bias):
        return None, None, None
    L = _lib.lib()
    x, weight = lay.x, _dense(weight)
    grad, g_stride = lay.fit(grad_output if grad_output.dtype == x.dtype
                             else grad_output.to(x.dtype))
    p = _lib.LayerNormParams(lay.outer, lay.inner, lay.stride, lay.C * lay.inner, g_stride, lay.C,
                             _DTYPES[x.dtype], _DTYPES[wdtype], 0.0)
    at = ctypes.byref(p)
    gx = gw = gb = ws = None
    nbytes = 0
    if need_input:
        gx = lay.like(x)
    if need_weight:
        gw = torch.empty(lay.C, dtype=wdtype, device=x.device)
    if need_bias:
        gb = torch.empty(lay.C, dtype=wdtype, device=x.device)
    if need_weight or need_bias:
        nbytes = L.ganet_layer_norm_backward_workspace_bytes(at)
        ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=x.device)
    rc = _lib.call(index, L.ganet_layer_norm_backward, x.data_ptr(), _ptr(weight),
                   grad.data_ptr(), mean.data_ptr(), rstd.data_ptr(), _ptr(gx), _ptr(gw),
                   _ptr(gb), at, _ptr(ws), nbytes)
    if rc:
        _lib.check(rc, "ganet_layer_norm_backward")
    return gx, gw, gb


class LayerNormFunction(Function):

    @staticmethod
    def forward(ctx, input, weight, bias, eps, channel_dim):
        ctx.channel_dim = channel_dim
        ctx.bias_dtype = bias.dtype if bias is not None else None
        out, mean, rstd = _forward(input, weight, bias, eps, channel_dim, True)
        ctx.save_for_backward(input, weight, mean, rstd)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        input, weight, mean, rstd = ctx.saved_tensors
        want = ctx.needs_input_grad
        if weight is None and want[2] and ctx.bias_dtype != input.dtype:
            # the sums of a bias alone are rounded to the weight's dtype: one of the bias's, of ones
            weight = torch.ones(input.shape[ctx.channel_dim], dtype=ctx.bias_dtype,
                                device=input.device)
        return layer_norm_backward(input, weight, grad_output, mean, rstd, ctx.channel_dim,
                                   *want[:3]) + (None, None)


def layer_norm(input, weight=None, bias=None, eps=1e-5, channel_dim=-1):
    """Layer norm over `channel_dim` with gradients; see layer_norm_forward.  Where no backward can
    follow (evaluation) mean and rstd are not written."""
    if ((torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                         for t in (input, weight, bias)))
            or forward_ad._current_level >= 0):           # has no forward derivative: autograd says so
        return LayerNormFunction.apply(input, weight, bias, eps, channel_dim)
    return _forward(input, weight, bias, eps, channel_dim, False)[0]


class LayerNorm(nn.Module):
    """Parameters `weight` and `bias` [num_channels], named and shaped like torch.nn.LayerNorm's
    of one dimension, so its state dict loads."""

    def __init__(self, num_channels, eps=1e-5, affine=True, channel_dim=-1):
        super(LayerNorm, self).__init__()
        self.num_channels, self.eps, self.channel_dim = num_channels, eps, channel_dim
        if affine:
            self.weight = nn.Parameter(torch.ones(num_channels))
            self.bias = nn.Parameter(torch.zeros(num_channels))
        else:
            self.register_parameter('weight', None)
            self.register_parameter('bias', None)

    def forward(self, x):
        if x.shape[self.channel_dim] != self.num_channels:
            raise ValueError("LayerNorm: %d channels at dimension %d of %s, expected %d"
                             % (x.shape[self.channel_dim], self.channel_dim, tuple(x.shape),
                                self.num_channels))
        return layer_norm(x, self.weight, self.bias, self.eps, self.channel_dim)

    def extra_repr(self):
        return '{num_channels}, eps={eps}, channel_dim={channel_dim}'.format(**self.__dict__)


class LayerNorm2d(LayerNorm):
    """Over the channels of [B, C, H, W] maps, as DeformConv writes them."""
    _abbr_ = 'ln'                                 # mmcv: the name of the norm in a ConvModule

    def __init__(self, num_channels, eps=1e-5, affine=True):
        super(LayerNorm2d, self).__init__(num_channels, eps, affine, channel_dim=1)


def register_with_mmcv(force=False):
    """Register LayerNorm2d as 'LN2d' in mmcv's NORM_LAYERS (norm_cfg=dict(type='LN2d')).  An
    explicit call, as in ganet_amd.dcn; False when mmcv is absent."""
    try:
        from mmcv.cnn import NORM_LAYERS
    except Exception:
        return False
    NORM_LAYERS.register_module('LN2d', module=LayerNorm2d, force=force)
    return True
