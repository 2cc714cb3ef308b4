"""Differential attention (csrc/diff_attn.hip): softmax attention as the difference of two maps, fp32 and bf16, the maps never
written.  The softmax counterpart of ops.non_local_dot for the non-local blocks."""
import ctypes
import math

import torch

from . import _C
from ._ops_norm import _DTYPES, _on, _require_float, _same_device
from ._opbase import _p, _stream, _Timed, _ws

_ATTN_DTYPES = {torch.float32: 0, torch.bfloat16: 1}


class AttnDesc(ctypes.Structure):
    """struct vspw_dattn_desc (include/vspw_hip.h)."""

    _fields_ = ([(n, ctypes.c_int) for n in ("b", "nq", "nk", "h", "hk", "d", "dtype", "lam_dtype", "frame")]
                + [("scale", ctypes.c_float)]
                + [(n, ctypes.c_longlong) for n in ("q_sb", "q_sn", "q_sh", "q_sm", "k_sb", "k_sn", "k_sh", "k_sm",
                                                    "v_sb", "v_sn", "v_sh")])


def _strided(t):
    """t itself when the kernels can address it (dense last dimension, everything else on 16 bytes), else a copy."""
    ve = 16 // t.element_size()
    ok = t.stride(-1) == 1 and t.data_ptr() % 16 == 0
    ok = ok and all(n == 1 or s % ve == 0 for n, s in zip(t.shape[:-1], t.stride()[:-1]))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _strides(t):
    return [0 if n == 1 else s for n, s in zip(t.shape[:-1], t.stride()[:-1])]


def _desc(q, k, v, lam, scale, frame):
    b, nq, h, _, d = q.shape
    qs, ks, vs = _strides(q), _strides(k), _strides(v)
    return AttnDesc(b, nq, k.shape[1], h, k.shape[2], d, _ATTN_DTYPES[q.dtype], _ATTN_DTYPES[lam.dtype], frame, scale,
                    *qs, *ks, *vs)


def _pairs(q, k, frame):
    nq, nk = q.shape[1], k.shape[1]
    if not frame:
        return float(nq) * nk
    return float(nk) * nq - 0.5 * nq * max(0, min(nq, nk) - frame)  # for the launch timers: the mean of the visible keys


class DiffAttentionFn(torch.autograd.Function):
    """Forward keeps both maps' outputs in float32 and their log-sum-exps; backward recomputes the scores."""

    @staticmethod
    def forward(ctx, q, k, v, lam, scale, mask, frame):
        q, k, v = _strided(q), _strided(k), _strided(v)
        b, nq, h, _, d = q.shape
        nk, hk = k.shape[1], k.shape[2]
        train = any(ctx.needs_input_grad[:4])
        out = torch.empty((b, nq, h, 2 * d), device=q.device, dtype=q.dtype)
        maps = lse = None
        if out.numel() and nk:
            with _on(q):
                if train:
                    maps = torch.empty((b, nq, h, 2, 2 * d), device=q.device, dtype=torch.float32)
                    lse = torch.empty((2, b * hk, nq * (h // hk)), device=q.device, dtype=torch.float32)
                ds = _desc(q, k, v, lam, scale, frame)
                nbytes = _C.query("vspw_diff_attn_fwd_workspace", ctypes.byref(ds))
                ws = _ws(nbytes, q.device) if nbytes else None
                with _Timed("diff_attn_fwd", 12.0 * b * h * d * _pairs(q, k, frame), "diff_attn b%d n%d/%d h%d d%d" % (b, nq, nk, h, d)):
                    _C.call("vspw_diff_attn_fwd", ctypes.byref(ds), _p(q), _p(k), _p(v), _p(lam), _p(mask), _p(out), _p(maps),
                            _p(lse), _p(ws), nbytes, _stream())
        else:
            out.zero_()
        ctx.meta = (scale, frame)
        ctx.save_for_backward(q, k, v, lam, mask, maps, lse)
        return out

    @staticmethod
    def backward(ctx, go):
        q, k, v, lam, mask, maps, lse = ctx.saved_tensors
        scale, frame = ctx.meta
        need = ctx.needs_input_grad
        b, nq, h, _, d = q.shape
        nk = k.shape[1]
        with _on(q):
            dq = torch.empty(q.shape, device=q.device, dtype=q.dtype) if need[0] else None
            dk = torch.empty(k.shape, device=q.device, dtype=q.dtype) if need[1] or need[2] else None
            dv = torch.empty(v.shape, device=q.device, dtype=q.dtype) if need[1] or need[2] else None
            dlam = torch.empty_like(lam) if need[3] else None
            if maps is None:  # no rows or no keys
                for t in (dq, dk, dv, dlam):
                    if t is not None:
                        t.zero_()
            else:
                go = _strided(go.contiguous())
                ds = _desc(q, k, v, lam, scale, frame)
                nbytes = _C.query("vspw_diff_attn_bwd_workspace", ctypes.byref(ds))
                ws = _ws(nbytes, q.device)
                with _Timed("diff_attn_bwd", 28.0 * b * h * d * _pairs(q, k, frame), "diff_attn b%d n%d/%d h%d d%d" % (b, nq, nk, h, d)):
                    _C.call("vspw_diff_attn_bwd", ctypes.byref(ds), _p(q), _p(k), _p(v), _p(lam), _p(mask), _p(maps),
                            _p(lse), _p(go), _p(dq), _p(dk), _p(dv), _p(dlam), _p(ws), nbytes, _stream())
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
    return DiffAttentionFn.apply(q, k, v, lam.contiguous(), scale, key_mask, frame)


class DiffLambdaFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, lq1, lk1, lq2, lk2, init):
        h, d = lq1.shape
        lam = torch.empty(h, device=lq1.device, dtype=torch.float32)
        with _on(lq1):
            _C.call("vspw_diff_lambda_fwd", _p(lq1), _p(lk1), _p(lq2), _p(lk2), init, _p(lam), h, d, _stream())
        ctx.save_for_backward(lq1, lk1, lq2, lk2)
        return lam

    @staticmethod
    def backward(ctx, g):
        lq1, lk1, lq2, lk2 = ctx.saved_tensors
        h, d = lq1.shape
        grads = [torch.empty_like(lq1) for _ in range(4)]
        with _on(lq1):
            _C.call("vspw_diff_lambda_bwd", _p(lq1), _p(lk1), _p(lq2), _p(lk2), _p(g.float().contiguous()),
                    *[_p(t) for t in grads], h, d, _stream())
        return tuple(grads) + (None,)


def diff_lambda(lq1, lk1, lq2, lk2, init):
    """The learned weight of the second map per head: exp(lq1.lk1) - exp(lq2.lk2) + init for float32 [H,D] vectors -> [H]."""
    ts = (lq1, lk1, lq2, lk2)
    for t in ts:
        _require_float(t, "diff_lambda", {torch.float32: _DTYPES[torch.float32]})
    _same_device("diff_lambda", *ts)
    if lq1.dim() != 2 or lq1.numel() == 0 or any(t.shape != lq1.shape for t in ts):
        raise RuntimeError("diff_lambda: four [H,D] vectors of equal shape expected, got %s" % (tuple(tuple(t.shape) for t in ts),))
    return DiffLambdaFn.apply(*[t.contiguous() for t in ts], float(init))
