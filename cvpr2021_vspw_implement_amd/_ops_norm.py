"""Group normalisation with activation, and dropout from a counter-based generator (csrc/group_norm.hip, csrc/dropout.hip):
the operators of ops.py that take float32, bfloat16 and float16 activations.

Both work on channels-last memory like the rest of ops.py: a [N,C,...] tensor is brought to [N][pixels][C] order (zero-copy
when it is already there) and the result comes back in that order under the input's logical shape.
"""
import contextlib

import torch

from . import _C
from ._opbase import _p, _stream, _ws, is_nhwc, to_nhwc

_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}  # VSPW_F32 / VSPW_BF16 / VSPW_F16
_ACTS = {"none": 0, "relu": 1, "silu": 2, "gelu": 3}


def _require_float(t, what, dtypes=_DTYPES):
    if not t.is_cuda:
        raise RuntimeError("%s: the VSPW hot path runs only through the HIP kernels on a GPU tensor (got device %s); "
                           "there is no CPU fallback" % (what, t.device))
    if t.dtype not in dtypes:
        raise RuntimeError("%s: %s tensors only (got %s)" % (what, " / ".join(str(d)[6:] for d in dtypes), t.dtype))


def _same_device(what, first, *others):
    for t in others:
        if t is not None and t.device != first.device:
            raise RuntimeError("%s: tensors on %s and %s" % (what, first.device, t.device))


def _on(t):
    """The tensor's device as the current one: kernels run on ITS device's current stream."""
    if t.device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(t.device)


def _rows(x):
    """[N,C,...] of any strides -> ([N][pixels][C] memory under the logical shape [N,C,P,1], its 4-D tensor)."""
    n, c = x.shape[0], x.shape[1]
    x4 = x if x.dim() == 4 else x.reshape(n, c, -1, 1)
    if is_nhwc(x4):
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


def _drop(x, p, rng, channelwise, dims):
    y = torch.empty_like(x)  # preserves the dense memory order
    n, hw, c = dims
    if x.numel():
        _C.call("vspw_dropout", _p(x), _p(y), n, hw, c, _DTYPES[x.dtype], p, _p(rng), 1 if channelwise else 0, _stream())
    return y


class DropoutFn(torch.autograd.Function):
    @staticmethod
    def _launch(x, p, rng, channelwise):
        if x.dim() >= 3:
            xr = _rows(x)
            dims = (xr.shape[0], xr.shape[2] * xr.shape[3], xr.shape[1])
        else:
            xr = x.contiguous()
            dims = (x.shape[0], 1, x.shape[1]) if channelwise else (1, xr.numel(), 1)
        return _drop(xr, p, rng, channelwise, dims).reshape(x.shape)

    @staticmethod
    def forward(ctx, x, p, rng, channelwise):
        with _on(x):
            y = DropoutFn._launch(x, p, rng, channelwise)
        ctx.meta = (p, channelwise)
        ctx.save_for_backward(rng)
        return y

    @staticmethod
    def backward(ctx, g):
        (rng,) = ctx.saved_tensors
        with _on(g):
            return DropoutFn._launch(g, ctx.meta[0], rng, ctx.meta[1]), None, None, None


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
    return DropoutFn.apply(x, p, rng, bool(channelwise))


def rng_next(state):
    """(seed, offset) for one training step of a dropout layer: a copy of `state` (int64 [2] on the GPU), whose offset then
    advances by one - on the stream, so every replay of a captured step draws a new mask."""
    if not state.is_cuda or state.dtype != torch.int64 or state.numel() != 2 or not state.is_contiguous():
        raise RuntimeError("rng_next: two contiguous int64 values (seed, offset) on the GPU expected")
    used = torch.empty_like(state)
    with _on(state):
        _C.call("vspw_rng_next", _p(state), _p(used), _stream())
    return used


class GroupNormActFn(torch.autograd.Function):
    """y = dropout(act(group_norm(x))); the backward pass re-reads x and the fp64 statistics [N,groups,2]."""

    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act, p, rng, channelwise):
        xr = _aligned(_rows(x))
        n, c, h, w = xr.shape
        hw = h * w
        dt = _DTYPES[x.dtype]
        y = torch.empty_like(xr)
        train = any(ctx.needs_input_grad[:3])
        with _on(x):
            stats = torch.empty((n, groups, 2), device=x.device, dtype=torch.float64) if train else None
            if xr.numel():
                nbytes = _C.query("vspw_group_norm_fwd_workspace", n, hw, c, groups, dt)
                ws = _ws(nbytes, x.device)
                _C.call("vspw_group_norm_fwd", _p(xr), _p(y), n, hw, c, groups, dt, _p(weight), _p(bias), eps, act, p,
                        _p(rng), channelwise, _p(stats), _p(ws), nbytes, _stream())
        ctx.meta = (groups, act, p, channelwise, tuple(x.shape))
        ctx.save_for_backward(xr, weight, bias, rng, stats)
        return y.reshape(x.shape)

    @staticmethod
    def backward(ctx, g):
        xr, weight, bias, rng, stats = ctx.saved_tensors
        groups, act, p, channelwise, shape = ctx.meta
        n, c, h, w = xr.shape
        hw = h * w
        dt = _DTYPES[xr.dtype]
        need = ctx.needs_input_grad
        with _on(xr):
            gr = _aligned(_rows(g))
            dx = torch.empty_like(xr) if need[0] else None
            dw = torch.empty_like(weight) if need[1] else None
            db = torch.empty_like(bias) if need[2] else None
            if xr.numel():
                nbytes = _C.query("vspw_group_norm_bwd_workspace", n, hw, c, groups, dt)
                ws = _ws(nbytes, xr.device)
                _C.call("vspw_group_norm_bwd", _p(xr), _p(gr), _p(dx), n, hw, c, groups, dt, _p(weight), _p(bias), act, p,
                        _p(rng), channelwise, _p(stats), _p(dw), _p(db), _p(ws), nbytes, _stream())
            else:
                for t in (dw, db):
                    if t is not None:
                        t.zero_()
        return (None if dx is None else dx.reshape(shape), dw, db) + (None,) * 6


def group_norm_act(x, num_groups, weight=None, bias=None, eps=1e-5, act="none", p=0.0, rng=None, channelwise=False):
    """dropout(act(weight * (x - mean) / sqrt(var + eps) + bias)) for x [N,C,...] (float32 / bfloat16 / float16), mean and
    variance over the positions and the C / num_groups channels of a group.  act: "none", "relu", "silu" or "gelu" (erf);
    p, rng, channelwise: see dropout().  weight / bias [C] are used in float32, their gradients come back in their own type."""
    _require_float(x, "group_norm_act")
    if x.dim() < 2:
        raise RuntimeError("group_norm_act: a [N,C,...] tensor expected, got %s" % (tuple(x.shape),))
    c = x.shape[1]
    num_groups = int(num_groups)
    if num_groups <= 0 or c % num_groups or c == 0:
        raise ValueError("group_norm_act: %d channels do not divide into %d groups" % (c, num_groups))
    if act not in _ACTS:
        raise ValueError("group_norm_act: act must be one of %s, got %r" % (", ".join(_ACTS), act))
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("group_norm_act: eps must not be negative, got %r" % eps)
    p = _check_rng("group_norm_act", p, rng)
    _same_device("group_norm_act", x, weight, bias, rng)
    for t, name in ((weight, "weight"), (bias, "bias")):
        if t is not None and tuple(t.shape) != (c,):
            raise RuntimeError("group_norm_act: %s must be [%d], got %s" % (name, c, tuple(t.shape)))
    weight = None if weight is None else weight.float().contiguous()
    bias = None if bias is None else bias.float().contiguous()
    return GroupNormActFn.apply(x, weight, bias, num_groups, eps, _ACTS[act], p, rng if p > 0.0 else None,
                                1 if channelwise else 0)
