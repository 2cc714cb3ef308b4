"""Differential attention (csrc/diff_attn.hip): softmax attention as the difference of two maps, fp32 and bf16, the maps never
written.  The softmax counterpart of ops.non_local_dot for the non-local blocks."""
import ctypes
import math

import torch

from . import _C
from ._ops_norm import _DTYPES, _addr, _on_device, _raw_stream, _require_float, _same_device, _wants_grad
from ._opbase import _Timed, _ktimer, _ws

_ATTN_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


class AttnDesc(ctypes.Structure):
    """struct vspw_dattn_desc (include/vspw_hip.h)."""

    _fields_ = ([(n, ctypes.c_int) for n in ("b", "nq", "nk", "h", "hk", "d", "dtype", "lam_dtype", "frame")]
                + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_longlong) for n in ("q_sb", "q_sn", "q_sh", "q_sm", "k_sb", "k_sn", "k_sh", "k_sm",
                                                    "v_sb", "v_sn", "v_sh")])


_NEAR = 1 << 24  # strides between rows, maps and heads that the kernels address with 32 bits inside a tile (elements)


def _strides(t):
    """Element strides of all dimensions but the last, 0 where there is nothing to step over."""
    return [0 if n == 1 else s for n, s in zip(t.shape[:-1], t.stride()[:-1])]


def _strided(t, g=1):
    """(t, its strides) when the kernels can address it (dense last dimension, everything else on 16 bytes, near rows), else of
    a copy.  g: how many heads a tile of rows mixes."""
    st = _strides(t)
    ve = 16 // t.element_size()
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    for i, s in enumerate(st):
        ok = ok and s % ve == 0 and (i == 0 or (i == 2 and g == 1) or s * (g if i == 2 else 1) < _NEAR)
    if not ok:
        t = t.clone(memory_format=torch.contiguous_format)
        st = _strides(t)
    return t, st


def _desc(q, k, lam, scale, frame, qs, ks, vs):
    b, nq, h, _, d = q.shape
    return AttnDesc(b, nq, k.shape[1], h, k.shape[2], d, _ATTN_DTYPES[q.dtype], _ATTN_DTYPES[lam.dtype], frame, scale,
                    *qs, *ks, *vs)


def _flops(q, k, frame, per_pair):
    """For the launch timers: the mean of the visible keys."""
    b, nq, h, _, d = q.shape
    nk = k.shape[1]
    pairs = float(nk) * nq - (0.5 * nq * max(0, min(nq, nk) - frame) if frame else 0.0)
    return per_pair * b * h * d * pairs


def _timed(name, q, k, frame, per_pair):
    if not _ktimer["on"]:
        return _Timed(name, 0.0)
    return _Timed(name, _flops(q, k, frame, per_pair), "diff_attn b%d n%d/%d h%d d%d" % (q.shape[0], q.shape[1], k.shape[1],
                                                                                          q.shape[2], q.shape[4]))


@_on_device
def _attn_fwd(q, k, v, lam, scale, mask, frame, train):
    """(out, maps, lse, descriptor, q, k, v): the last three as the kernels read them"""
    hk = k.shape[2]
    b, nq, h, _, d = q.shape
    (q, qs), (k, ks), (v, vs) = _strided(q, h // hk), _strided(k), _strided(v)
    out = torch.empty((b, nq, h, 2 * d), device=q.device, dtype=q.dtype)
    maps = lse = None
    if not out.numel() or not k.shape[1]:
        return out.zero_(), None, None, None, q, k, v
    if train:
        maps = torch.empty((b, nq, h, 2, 2 * d), device=q.device, dtype=torch.float32)
        lse = torch.empty((2, b * hk, nq * (h // hk)), device=q.device, dtype=torch.float32)
    ds = _desc(q, k, lam, scale, frame, qs, ks, vs)
    ref = ctypes.byref(ds)
    nbytes = _C.query("vspw_diff_attn_fwd_workspace", ref)
    ws = _ws(nbytes, q.device) if nbytes else None
    with _timed("diff_attn_fwd", q, k, frame, 12.0):
        _C.call("vspw_diff_attn_fwd", ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), _addr(mask), out.data_ptr(),
                _addr(maps), _addr(lse), _addr(ws), nbytes, _raw_stream(q.device.index))
    return out, maps, lse, ds, q, k, v


@_on_device
def _attn_bwd(q, k, v, lam, mask, maps, lse, ds, go, frame, need):
    dev, dt = q.device, q.dtype
    dq = torch.empty(q.shape, device=dev, dtype=dt) if need[0] else None
    dk = dv = None
    if need[1] or need[2]:
        dk, dv = torch.empty(k.shape, device=dev, dtype=dt), torch.empty(v.shape, device=dev, dtype=dt)
    dlam = torch.empty_like(lam) if need[3] else None
    if maps is None:  # no rows or no keys
        for t in (dq, dk, dv, dlam):
            if t is not None:
                t.zero_()
        return dq, dk, dv, dlam
    go = go.contiguous()
    if go.data_ptr() % 16:
        go = go.clone()
    ref = ctypes.byref(ds)
    nbytes = _C.query("vspw_diff_attn_bwd_workspace", ref)
    ws = _ws(nbytes, dev)
    with _timed("diff_attn_bwd", q, k, frame, 28.0):
        _C.call("vspw_diff_attn_bwd", ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), _addr(mask), maps.data_ptr(),
                lse.data_ptr(), go.data_ptr(), _addr(dq), _addr(dk), _addr(dv), _addr(dlam), ws.data_ptr(), nbytes,
                _raw_stream(dev.index))
    return dq, dk, dv, dlam


class DiffAttentionFn(torch.autograd.Function):
    """Forward keeps both maps' outputs in float32 and their log-sum-exps; backward recomputes the scores."""

    @staticmethod
    def forward(ctx, q, k, v, lam, scale, mask, frame):
        out, maps, lse, ds, q, k, v = _attn_fwd(q, k, v, lam, scale, mask, frame, True)
        ctx.meta = (ds, frame)
        ctx.save_for_backward(q, k, v, lam, mask, maps, lse)
        return out

    @staticmethod
    def backward(ctx, go):
        q, k, v, lam, mask, maps, lse = ctx.saved_tensors
        ds, frame = ctx.meta
        need = ctx.needs_input_grad
        dq, dk, dv, dlam = _attn_bwd(q, k, v, lam, mask, maps, lse, ds, go, frame, need)
        return dq, dk if need[1] else None, dv if need[2] else None, dlam, None, None, None


def diff_attention_supported(d):
    """Head widths the kernels are built for (values are twice as wide)."""
    return d in (16, 32, 64)


def diff_attention(q, k, v, lam, scale=None, key_mask=None, frame=0):
    """out[b,i,h] = sum_j (softmax_j(scale q1.k1) - lam[h] softmax_j(scale q2.k2)) v_j for q [B,Nq,H,2,D], k [B,Nk,Hk,2,D],
    v [B,Nk,Hk,2D] -> [B,Nq,H,2D], float32 or bfloat16, D in {16, 32, 64}; H / Hk query heads share a key/value head.

    Any strides with a dense last dimension (slices of one projection, transposed layouts) are used as they are.
    lam [H]: float32 or the inputs' type.  scale: default 1 / sqrt(D), must be positive.  key_mask [B,Nk] bool: True where the
    key takes part; what masked positions hold (infinities, NaN) is not used.  frame > 0: positions come in frames of that
    many, and a query sees the keys of its own frame and of earlier ones, the ends of queries and keys aligned (query i stands
    at position i + Nk - Nq).  A query without keys gets zeros and zero gradients.
    """
    _require_float(q, "diff_attention", _ATTN_DTYPES)
    for t in (k, v, lam):
        _require_float(t, "diff_attention", _ATTN_DTYPES)
    _same_device("diff_attention", q, k, v, lam, key_mask)
    if q.dim() != 5 or k.dim() != 5 or v.dim() != 4 or q.shape[3] != 2 or k.shape[3] != 2:
        raise RuntimeError("diff_attention: q [B,Nq,H,2,D], k [B,Nk,Hk,2,D], v [B,Nk,Hk,2D] expected, got %s, %s, %s"
                           % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    b, nq, h, _, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    if k.shape[0] != b or k.shape[4] != d or tuple(v.shape) != (b, nk, hk, 2 * d):
        raise RuntimeError("diff_attention: q %s, k %s and v %s do not belong together"
                           % (tuple(q.shape), tuple(k.shape), tuple(v.shape)))
    if h == 0 or hk == 0 or h % hk:
        raise RuntimeError("diff_attention: %d query heads do not divide over %d key heads" % (h, hk))
    if not diff_attention_supported(d):
        raise RuntimeError("diff_attention: head width %d is not one of 16, 32, 64" % d)
    if k.dtype != q.dtype or v.dtype != q.dtype or lam.dtype not in (torch.float32, q.dtype):
        raise RuntimeError("diff_attention: q, k, v of one type and lam of that type or float32 expected, got %s, %s, %s, %s"
                           % (q.dtype, k.dtype, v.dtype, lam.dtype))
    if tuple(lam.shape) != (h,):
        raise RuntimeError("diff_attention: lam must be [%d], got %s" % (h, tuple(lam.shape)))
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not (0.0 < scale < float("inf")) or not ctypes.c_float(scale).value > 0.0:
        raise ValueError("diff_attention: scale must be positive and finite, got %r" % scale)
    frame = int(frame)
    if not 0 <= frame < 2 ** 31:
        raise ValueError("diff_attention: frame must be a number of positions, got %r" % frame)
    if key_mask is not None:
        if key_mask.dtype != torch.bool or tuple(key_mask.shape) != (b, nk):
            raise RuntimeError("diff_attention: key_mask must be bool [%d,%d], got %s %s"
                               % (b, nk, key_mask.dtype, tuple(key_mask.shape)))
        key_mask = key_mask.contiguous()
    lam = lam.contiguous()
    if _wants_grad(q, k, v, lam):
        return DiffAttentionFn.apply(q, k, v, lam, scale, key_mask, frame)
    return _attn_fwd(q, k, v, lam, scale, key_mask, frame, False)[0]


@_on_device
def _lambda_fwd(lq1, lk1, lq2, lk2, init):
    h, d = lq1.shape
    lam = torch.empty(h, device=lq1.device, dtype=torch.float32)
    _C.call("vspw_diff_lambda_fwd", lq1.data_ptr(), lk1.data_ptr(), lq2.data_ptr(), lk2.data_ptr(), init, lam.data_ptr(), h, d,
            _raw_stream(lq1.device.index))
    return lam


@_on_device
def _lambda_bwd(lq1, lk1, lq2, lk2, g):
    h, d = lq1.shape
    g = g.contiguous()
    grads = [torch.empty_like(lq1) for _ in range(4)]
    _C.call("vspw_diff_lambda_bwd", lq1.data_ptr(), lk1.data_ptr(), lq2.data_ptr(), lk2.data_ptr(), g.data_ptr(),
            *[t.data_ptr() for t in grads], h, d, _raw_stream(lq1.device.index))
    return tuple(grads)


class DiffLambdaFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lq1, lk1, lq2, lk2, init):
        ctx.save_for_backward(lq1, lk1, lq2, lk2)
        return _lambda_fwd(lq1, lk1, lq2, lk2, init)

    @staticmethod
    def backward(ctx, g):
        return _lambda_bwd(*ctx.saved_tensors, g) + (None,)


def diff_lambda(lq1, lk1, lq2, lk2, init):
    """The learned weight of the second map per head: exp(lq1.lk1) - exp(lq2.lk2) + init for float32 [H,D] vectors -> [H]."""
    ts = (lq1, lk1, lq2, lk2)
    for t in ts:
        _require_float(t, "diff_lambda", {torch.float32: _DTYPES[torch.float32]})
    _same_device("diff_lambda", *ts)
    if lq1.dim() != 2 or lq1.numel() == 0 or any(t.shape != lq1.shape for t in ts):
        raise RuntimeError("diff_lambda: four [H,D] vectors of equal shape expected, got %s" % (tuple(tuple(t.shape) for t in ts),))
    return DiffLambdaFn.apply(*[t.contiguous() for t in ts], float(init))
