"""Differential attention (csrc/diff_attn.hip): softmax attention as the difference of two maps, fp32 and bf16, the maps never
written.  The softmax counterpart of ops.non_local_dot for the non-local blocks."""
import ctypes
import functools
import math

import torch
from torch.autograd.function import once_differentiable

from . import _C
from ._ops_norm import _DTYPES, _addr, _on_device, _raw_stream, _require_float, _require_ints, _same_device, _wants_grad
from ._opbase import _Timed, _ktimer, _ws

_ATTN_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


class AttnDesc(ctypes.Structure):
    """struct vspw_dattn_desc (include/vspw_hip.h)."""

    _fields_ = ([(n, ctypes.c_int) for n in ("b", "nq", "nk", "h", "hk", "d", "dtype", "lam_dtype", "frame")]
                + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_longlong) for n in ("q_sb", "q_sn", "q_sh", "q_sm", "k_sb", "k_sn", "k_sh", "k_sm",
                                                    "v_sb", "v_sn", "v_sh")])


_NEAR = 1 << 24  # strides between rows, maps and heads that the kernels address with 32 bits inside a tile (elements)


def _strides(shape, stride, ve, g=1):
    """The strides of all dimensions but the last, 0 where there is nothing to step over, and whether the kernels can address
    them (dense last dimension, everything else on 16 bytes, near rows).  g: how many heads a tile of rows mixes."""
    st = [0 if n == 1 else s for n, s in zip(shape[:-1], stride[:-1])]
    ok = stride[-1] == 1
    for i, s in enumerate(st):
        ok = ok and s % ve == 0 and (i == 0 or (i == 2 and g == 1) or s * (g if i == 2 else 1) < _NEAR)
    return st, ok


class _Plan:
    __slots__ = ("desc", "ref", "fwd_bytes", "bwd_bytes", "q_ok", "k_ok", "v_ok", "empty", "frame", "scale")


@functools.lru_cache(maxsize=1024)
def _plan(qd, kd, vd, ld, qs, ks, vs, ls, q_stride, k_stride, v_stride, scale, frame):
    """Checks and descriptor of a call, a function of types, shapes and strides (a call for one token costs the host more than
    the GPU)."""
    if len(qs) != 5 or len(ks) != 5 or len(vs) != 4 or qs[3] != 2 or ks[3] != 2:
        raise RuntimeError("diff_attention: q [B,Nq,H,2,D], k [B,Nk,Hk,2,D], v [B,Nk,Hk,2D] expected, got %s, %s, %s"
                           % (tuple(qs), tuple(ks), tuple(vs)))
    b, nq, h, _, d = qs
    nk, hk = ks[1], ks[2]
    _require_ints("diff_attention", b, nq, nk, h)
    if ks[0] != b or ks[4] != d or tuple(vs) != (b, nk, hk, 2 * d):
        raise RuntimeError("diff_attention: q %s, k %s and v %s do not belong together" % (tuple(qs), tuple(ks), tuple(vs)))
    if h == 0 or hk == 0 or h % hk:
        raise RuntimeError("diff_attention: %d query heads do not divide over %d key heads" % (h, hk))
    if not diff_attention_supported(d):
        raise RuntimeError("diff_attention: head width %d is not one of 16, 32, 64" % d)
    if h * 2 * d >= _NEAR:
        raise RuntimeError("diff_attention: %d heads of 2 x %d columns are more than a row may hold" % (h, d))
    if kd != qd or vd != qd or ld not in (torch.float32, qd):
        raise RuntimeError("diff_attention: q, k, v of one type and lam of that type or float32 expected, got %s, %s, %s, %s"
                           % (qd, kd, vd, ld))
    if tuple(ls) != (h,):
        raise RuntimeError("diff_attention: lam must be [%d], got %s" % (h, tuple(ls)))
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    if not (0.0 < scale < float("inf")) or not ctypes.c_float(scale).value > 0.0:
        raise ValueError("diff_attention: scale must be positive and finite, got %r" % scale)
    if not 0 <= frame < 2 ** 31:
        raise ValueError("diff_attention: frame must be a number of positions, got %r" % frame)
    p = _Plan()
    ve = 8 if qd == torch.bfloat16 else 4
    qt, p.q_ok = _strides(qs, q_stride, ve, h // hk)
    kt, p.k_ok = _strides(ks, k_stride, ve)
    vt, p.v_ok = _strides(vs, v_stride, ve)
    p.empty, p.frame, p.scale = 0 in (b, nq, nk), frame, scale
    p.desc = AttnDesc(b, nq, nk, h, hk, d, _ATTN_DTYPES[qd], _ATTN_DTYPES[ld], frame, scale, *qt, *kt, *vt)
    p.ref = ctypes.byref(p.desc)
    p.fwd_bytes = 0 if p.empty else _C.query("vspw_diff_attn_fwd_workspace", p.ref)
    p.bwd_bytes = 0 if p.empty else _C.query("vspw_diff_attn_bwd_workspace", p.ref)
    return p


def _plan_of(q, k, v, lam, scale, frame):
    return _plan(q.dtype, k.dtype, v.dtype, lam.dtype, q.shape, k.shape, v.shape, lam.shape, q.stride(), k.stride(), v.stride(),
                 scale, frame)


def _flops(q, k, frame, per_pair):
    """For the launch timers: the mean of the visible keys."""
    b, nq, h, _, d = q.shape
    nk = k.shape[1]
    pairs = float(nk) * nq - (0.5 * nq * max(0, min(nq, nk) - frame) if frame else 0.0)
    return per_pair * b * h * d * pairs


def _launch(name, q, k, frame, per_pair, *args):
    if not _ktimer["on"]:
        return _C.call("vspw_" + name, *args)
    with _Timed(name, _flops(q, k, frame, per_pair), "diff_attn b%d n%d/%d h%d d%d" % (q.shape[0], q.shape[1], k.shape[1],
                                                                                      q.shape[2], q.shape[4])):
        _C.call("vspw_" + name, *args)


@_on_device
def _attn_fwd(q, k, v, lam, mask, plan, train):
    """(out, maps, lse, plan, q, k, v): the last three as the kernels read them (a copy where they cannot address a tensor)"""
    b, nq, h, _, d = q.shape
    dev = q.device
    out = torch.empty((b, nq, h, 2 * d), device=dev, dtype=q.dtype)
    maps = lse = None
    if plan.empty:
        return out.zero_(), None, None, plan, q, k, v
    qa, ka, va = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if not (plan.q_ok and plan.k_ok and plan.v_ok) or (qa | ka | va) % 16:
        q = q if plan.q_ok and qa % 16 == 0 else q.clone(memory_format=torch.contiguous_format)
        k = k if plan.k_ok and ka % 16 == 0 else k.clone(memory_format=torch.contiguous_format)
        v = v if plan.v_ok and va % 16 == 0 else v.clone(memory_format=torch.contiguous_format)
        plan = _plan_of(q, k, v, lam, plan.scale, plan.frame)
        qa, ka, va = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if train:
        maps = torch.empty((b, nq, h, 2, 2 * d), device=dev, dtype=torch.float32)
        lse = torch.empty((2, b, h, nq), device=dev, dtype=torch.float32)
    nbytes = plan.fwd_bytes
    ws = _ws(nbytes, dev) if nbytes else None
    _launch("diff_attn_fwd", q, k, plan.frame, 12.0, plan.ref, qa, ka, va, lam.data_ptr(), _addr(mask), out.data_ptr(), _addr(maps),
            _addr(lse), _addr(ws), nbytes, _raw_stream(dev.index))
    return out, maps, lse, plan, q, k, v


@_on_device
def _attn_bwd(q, k, v, lam, mask, maps, lse, plan, go, need):
    dev, dt = q.device, q.dtype
    dq = torch.empty(q.shape, device=dev, dtype=dt) if need[0] else None
    dk = dv = None
    if need[1] or need[2]:
        dk, dv = torch.empty(k.shape, device=dev, dtype=dt), torch.empty(v.shape, device=dev, dtype=dt)
    dlam = torch.empty_like(lam) if need[3] else None
    if plan.empty:
        for t in (dq, dk, dv, dlam):
            if t is not None:
                t.zero_()
        return dq, dk, dv, dlam
    go = go.contiguous()
    if go.data_ptr() % 16:
        go = go.clone()
    nbytes = plan.bwd_bytes
    ws = _ws(nbytes, dev)
    _launch("diff_attn_bwd", q, k, plan.frame, 28.0, plan.ref, q.data_ptr(), k.data_ptr(), v.data_ptr(), lam.data_ptr(), _addr(mask),
            maps.data_ptr(), lse.data_ptr(), go.data_ptr(), _addr(dq), _addr(dk), _addr(dv), _addr(dlam), ws.data_ptr(), nbytes,
            _raw_stream(dev.index))
    return dq, dk, dv, dlam


class DiffAttentionFn(torch.autograd.Function):
    """Forward keeps both maps' outputs in float32 and their log-sum-exps; backward recomputes the scores."""

    @staticmethod
    def forward(ctx, q, k, v, lam, mask, plan):
        out, maps, lse, ctx.plan, q, k, v = _attn_fwd(q, k, v, lam, mask, plan, True)
        ctx.save_for_backward(q, k, v, lam, mask, maps, lse)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        q, k, v, lam, mask, maps, lse = ctx.saved_tensors
        need = ctx.needs_input_grad
        dq, dk, dv, dlam = _attn_bwd(q, k, v, lam, mask, maps, lse, ctx.plan, go, need)
        return dq, dk if need[1] else None, dv if need[2] else None, dlam, None, None


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
    at position i + Nk - Nq); keys and values that frame hides from some queries must be finite.  A query without keys gets
    zeros and zero gradients.
    """
    for t in (q, k, v, lam):
        _require_float(t, "diff_attention", _ATTN_DTYPES)
    _same_device("diff_attention", q, k, v, lam, key_mask)
    plan = _plan_of(q, k, v, lam, None if scale is None else float(scale), int(frame))
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != k.shape[:2]:
            raise RuntimeError("diff_attention: key_mask must be bool %s, got %s %s"
                               % (list(k.shape[:2]), key_mask.dtype, tuple(key_mask.shape)))
        key_mask = key_mask.contiguous()
    lam = lam.contiguous()
    if _wants_grad(q, k, v, lam):
        return DiffAttentionFn.apply(q, k, v, lam, key_mask, plan)
    return _attn_fwd(q, k, v, lam, key_mask, plan, False)[0]


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
    @once_differentiable
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
