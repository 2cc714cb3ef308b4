"""Group normalisation with activation, and dropout from a counter-based generator (csrc/group_norm.hip, csrc/dropout.hip):
the operators of ops.py that take float32, bfloat16 and float16 activations.

Both work on channels-last memory like the rest of ops.py: a [N,C,...] tensor is brought to [N][pixels][C] order (zero-copy
when it is already there) and the result comes back in that order under the input's logical shape.
"""
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from . import _C
from ._opbase import _ws, to_nhwc

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # VSPW_F32 / VSPW_BF16 / VSPW_F16
_ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}

# These operators are called on small tensors too, where the host decides: addresses and streams go to ctypes as integers,
# and calls that need no gradient do not pass through autograd.
_raw_stream = torch._C._cuda_getCurrentRawStream
_current_device = torch._C._cuda_getDevice


def _addr(t):
    return None if t is None else t.data_ptr()


def _require_float(t, what, dtypes=_DTYPES):
    if not t.is_cuda:
        raise RuntimeError("%s: the VSPW hot path runs only through the HIP kernels on a GPU tensor (got device %s); "
                           "there is no CPU fallback" % (what, t.device))
    if t.dtype not in dtypes:
        raise RuntimeError("%s: %s tensors only (got %s)" % (what, " / ".join(str(d)[6:] for d in dtypes), t.dtype))


def _require_ints(what, *sizes):
    if max(sizes) >= 2 ** 31:
        raise RuntimeError("%s: sizes below 2^31 only, got %s" % (what, sizes))


def _same_device(what, first, *others):
    dev = first.device
    for t in others:
        if t is not None and t.device != dev:
            raise RuntimeError("%s: tensors on %s and %s" % (what, dev, t.device))


def _on_device(fn):
    """fn(t, ...) with t's device as the current one: kernels run on ITS device's current stream."""

    @functools.wraps(fn)
    def run(t, *args):
        if t.device.index == _current_device():
            return fn(t, *args)
        with torch.cuda.device(t.device):
            return fn(t, *args)

    return run


def _wants_grad(*ts):
    if not torch.is_grad_enabled():
        return False
    for t in ts:
        if t is not None and t.requires_grad:
            return True
    return False


def _rows(x):
    """[N,C,...] of any strides -> ([N][pixels][C] memory under the logical shape [N,C,P,1], its 4-D tensor)."""
    x4 = x if x.dim() == 4 else x.reshape(x.shape[0], x.shape[1], math.prod(x.shape[2:]), 1)
    if x4.is_contiguous(memory_format=torch.channels_last):
        return x4
    if x4.dtype == torch.float32 and x4.is_contiguous() and x4.numel():
        return to_nhwc(x4)
    return x4.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)


def _aligned(t):
    return t if t.data_ptr() % 16 == 0 else t.clone(memory_format=torch.preserve_format)


def _check_rng(what, p, rng):
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("%s: dropout probability %r is not in [0, 1]" % (what, p))
    if p > 0.0:
        if rng is None:
            raise ValueError("%s: dropout needs rng, an int64 tensor (seed, offset) on the GPU" % what)
        if rng.dtype != torch.int64 or rng.numel() != 2 or not rng.is_contiguous():
            raise RuntimeError("%s: rng must be two contiguous int64 values (seed, offset)" % what)
    return p


# ------------------------------------------------------------------------------------------------------------ dropout
@_on_device
def _dropout(x, p, rng, channelwise):
    shape = x.shape
    nd = len(shape)
    if nd >= 3:
        xr = _rows(x)
        n, c, h, w = xr.shape
        hw = h * w
    else:
        xr = x.contiguous()
        n, hw, c = (shape[0], 1, shape[1]) if channelwise else (1, xr.numel(), 1)
    y = torch.empty_like(xr)  # preserves the dense memory order
    if xr.numel():
        _C.call("vspw_dropout", xr.data_ptr(), y.data_ptr(), n, hw, c, _DTYPES[x.dtype], p, rng.data_ptr(),
                1 if channelwise else 0, _raw_stream(x.device.index))
    return y if nd == 4 else y.reshape(shape)


class DropoutFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, p, rng, channelwise):
        ctx.meta = (p, channelwise)
        ctx.save_for_backward(rng)
        return _dropout(x, p, rng, channelwise)

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        return _dropout(g, ctx.meta[0], ctx.saved_tensors[0], ctx.meta[1]), None, None, None


def dropout(x, p, rng=None, channelwise=False):
    """x * keep / (1 - p) with keep recomputed from rng = (seed, offset) in forward and backward, never stored.

    The word of element e of the generator decides (csrc/elem.h: Philox4x32-10): e counts elements in channels-last order for
    [N,C,...] inputs (row-major below three dimensions), or images and channels when `channelwise` (whole channels are
    dropped, nn.Dropout2d).  rng: int64 [2] on x's device, read by the kernel, so a replayed graph sees its current values;
    the caller leaves it unchanged until the backward pass has run."""
    _require_float(x, "dropout")
    p = _check_rng("dropout", p, rng)
    if p == 0.0:
        return x
    _same_device("dropout", x, rng)
    if channelwise and x.dim() < 2:
        raise RuntimeError("dropout: channelwise needs a [N,C,...] tensor, got %s" % (tuple(x.shape),))
    if channelwise or x.dim() > 2:
        _require_ints("dropout", x.shape[0], x.shape[1])
    if _wants_grad(x):
        return DropoutFn.apply(x, p, rng, bool(channelwise))
    return _dropout(x, p, rng, channelwise)


@_on_device
def _rng_next(state):
    used = torch.empty_like(state)
    _C.call("vspw_rng_next", state.data_ptr(), used.data_ptr(), _raw_stream(state.device.index))
    return used


def rng_next(state):
    """(seed, offset) for one training step of a dropout layer: a copy of `state` (int64 [2] on the GPU), whose offset then
    advances by one - on the stream, so every replay of a captured step draws a new mask."""
    if not state.is_cuda or state.dtype != torch.int64 or state.numel() != 2 or not state.is_contiguous():
        raise RuntimeError("rng_next: two contiguous int64 values (seed, offset) on the GPU expected")
    used = _rng_next(state)
    torch.autograd.graph.increment_version(state)  # written outside autograd's sight: a graph that saved it has to notice
    return used


# --------------------------------------------------------------------------------------------------------- group norm
@functools.lru_cache(maxsize=None)
def _norm_workspace(which, n, hw, c, groups, dt):
    return _C.query("vspw_group_norm_%s_workspace" % which, n, hw, c, groups, dt)


@_on_device
def _norm_fwd(x, weight, bias, groups, eps, act, p, rng, channelwise, train):
    """(y, rows of x, stats)"""
    xr = _aligned(_rows(x))
    n, c, h, w = xr.shape
    hw = h * w
    dt = _DTYPES[x.dtype]
    y = torch.empty_like(xr)
    stats = torch.empty((n, groups, 2), device=x.device, dtype=torch.float64) if train else None
    if xr.numel():
        nbytes = _norm_workspace("fwd", n, hw, c, groups, dt)
        ws = _ws(nbytes, x.device) if nbytes else None
        _C.call("vspw_group_norm_fwd", xr.data_ptr(), y.data_ptr(), n, hw, c, groups, dt, _addr(weight), _addr(bias), eps, act, p,
                _addr(rng), channelwise, _addr(stats), _addr(ws), nbytes, _raw_stream(x.device.index))
    return (y if x.dim() == 4 else y.reshape(x.shape)), xr, stats


@_on_device
def _norm_bwd(xr, g, weight, bias, rng, stats, meta, need):
    groups, act, p, channelwise, shape = meta
    n, c, h, w = xr.shape
    hw = h * w
    dt = _DTYPES[xr.dtype]
    gr = _aligned(_rows(g))
    dx = torch.empty_like(xr) if need[0] else None
    dw = torch.empty_like(weight) if need[1] else None
    db = torch.empty_like(bias) if need[2] else None
    if xr.numel():
        nbytes = _norm_workspace("bwd", n, hw, c, groups, dt)
        ws = _ws(nbytes, xr.device)
        _C.call("vspw_group_norm_bwd", xr.data_ptr(), gr.data_ptr(), _addr(dx), n, hw, c, groups, dt, _addr(weight), _addr(bias),
                act, p, _addr(rng), channelwise, stats.data_ptr(), _addr(dw), _addr(db), ws.data_ptr(), nbytes,
                _raw_stream(xr.device.index))
    else:
        for t in (dw, db):
            if t is not None:
                t.zero_()
    if dx is not None and len(shape) != 4:
        dx = dx.reshape(shape)
    return dx, dw, db


class GroupNormActFn(torch.autograd.Function):
    """y = dropout(act(group_norm(x))); the backward pass re-reads x and the fp64 statistics [N,groups,2].
    how: (groups, eps, act, p, channelwise)."""

    @staticmethod
    def forward(ctx, x, weight, bias, rng, how):
        groups, eps, act, p, channelwise = how
        y, xr, stats = _norm_fwd(x, weight, bias, groups, eps, act, p, rng, channelwise, True)
        ctx.meta = (groups, act, p, channelwise, x.shape)
        ctx.save_for_backward(xr, weight, bias, rng, stats)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        xr, weight, bias, rng, stats = ctx.saved_tensors
        return _norm_bwd(xr, g, weight, bias, rng, stats, ctx.meta, ctx.needs_input_grad) + (None, None)


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", p=0.0, rng=None, channelwise=False):
    """dropout(act(weight * (x - mean) / sqrt(var + eps) + bias)) for x [N,C,...] (float32 / bfloat16 / float16), mean and
    variance over the positions and the C / num_groups channels of a group.  act: "none", "relu", "silu" or "gelu" (erf);
    p, rng, channelwise: see dropout().  weight / bias [C] are used in float32, their gradients come back in their own type."""
    _require_float(x, "group_norm_act")
    if x.dim() < 2:
        raise RuntimeError("group_norm_act: a [N,C,...] tensor expected, got %s" % (tuple(x.shape),))
    c = x.shape[1]
    _require_ints("group_norm_act", x.shape[0], c)
    num_groups = int(num_groups)
    if num_groups <= 0 or c % num_groups or c == 0:
        raise ValueError("group_norm_act: %d channels do not divide into %d groups" % (c, num_groups))
    if act not in _ACTS:
        raise ValueError("group_norm_act: act must be one of %s, got %r" % (", ".join(_ACTS), act))
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("group_norm_act: eps must not be negative, got %r" % eps)
    p = _check_rng("group_norm_act", p, rng)
    if p == 0.0:
        rng = None
    _same_device("group_norm_act", x, weight, bias, rng)
    if weight is not None:
        if weight.dim() != 1 or weight.shape[0] != c:
            raise RuntimeError("group_norm_act: weight must be [%d], got %s" % (c, tuple(weight.shape)))
        weight = weight.float().contiguous()
    if bias is not None:
        if bias.dim() != 1 or bias.shape[0] != c:
            raise RuntimeError("group_norm_act: bias must be [%d], got %s" % (c, tuple(bias.shape)))
        bias = bias.float().contiguous()
    if _wants_grad(x, weight, bias):
        return GroupNormActFn.apply(x, weight, bias, rng, (num_groups, eps, _ACTS[act], p, 1 if channelwise else 0))
    return _norm_fwd(x, weight, bias, num_groups, eps, _ACTS[act], p, rng, 1 if channelwise else 0, False)[0]
