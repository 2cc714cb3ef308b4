"""Differential attention against the maps written out in float64, forward and gradients.

Tolerances are computed with the reference, element by element.  u = 2^-24; a float32 sum of n terms is allowed
2 u sqrt(n) sum |terms| (independent roundings, twice their standard deviation); `hp` is half a step of bf16 for the weights
and the score gradients that the matrix unit takes in bf16 (0 for float32 inputs), `ho` half a step of the result's type:
  S   eS = 2 u sqrt(D) s |q||k|^T + 2 u |S|              P   rel = 2 max eS + 2 u sqrt(N) + 8 u (+ hp)
  out sum rel (P1 + lam P2)|v| + sum error + ho|out|      dP  2 u sqrt(W) |dO||v|^T
  D   sum |dO| (error of out and of the second output, both rounded to the type)
  dS  rel |dS| + P (dP and D errors) + hp |dS|            dq, dk, dv: those summed over |k|, |q|, |dO| + sum error + ho|.|"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def visible(b, nq, nk, frame, mask):
    vis = torch.ones(b, 1, nq, nk, dtype=torch.bool)
    if frame:
        pos = torch.arange(nq) + nk - nq
        vis &= torch.arange(nk)[None, :] < ((torch.div(pos, frame, rounding_mode="floor") + 1) * frame)[:, None]
    if mask is not None:
        vis &= mask[:, None, None, :]
    return vis


def reference(q, k, v, lam, scale, mask, frame, go):
    """{name: (value, tolerance)} for out, dq, dk, dv, dlam, from inputs of the tested type."""
    dt = q.dtype
    ho = torch.finfo(dt).eps / 2
    hp = ho if dt == torch.bfloat16 else 0.0
    b, nq, h, _, d = q.shape
    nk, hk = k.shape[1], k.shape[2]
    rep, w = h // hk, 2 * d
    if mask is not None:
        k, v = k.clone(), v.clone()
        k[~mask], v[~mask] = 0, 0
    q = q.double().permute(3, 0, 2, 1, 4)
    k = k.double().permute(3, 0, 2, 1, 4).repeat_interleave(rep, 2)
    v = v.double().permute(0, 2, 1, 3).repeat_interleave(rep, 1)
    go = go.double().permute(0, 2, 1, 3)
    lam_t = lam.double()
    lam = lam_t.view(1, h, 1, 1)
    al = lam.abs()
    vis = visible(b, nq, nk, frame, mask)
    P, rel = [], []
    for m in range(2):
        s = scale * q[m] @ k[m].transpose(-1, -2)
        es = 2 * U * math.sqrt(d) * scale * (q[m].abs() @ k[m].abs().transpose(-1, -2)) + 2 * U * s.abs()
        s = s.masked_fill(~vis, -math.inf)
        mx = s.amax(-1, keepdim=True)
        e = torch.exp(s - torch.where(mx.isinf(), torch.zeros_like(mx), mx))
        den = e.sum(-1, keepdim=True)
        P.append(torch.where(den > 0, e / den, torch.zeros_like(e)))
        rel.append(2 * es.masked_fill(~vis, 0).amax(-1, keepdim=True) + 2 * U * math.sqrt(nk) + 8 * U)
    su = 2 * U * math.sqrt(nk)
    out = (P[0] - lam * P[1]) @ v
    o2 = P[1] @ v
    t1 = (rel[0] + hp + su) * (P[0] @ v.abs())
    t2 = (rel[1] + hp + su) * (P[1] @ v.abs())
    tout = t1 + al * t2 + 4 * U * (P[0] @ v.abs() + al * o2.abs()) + ho * out.abs()
    # gradients
    dp = go @ v.transpose(-1, -2)
    edp = 2 * U * math.sqrt(w) * (go.abs() @ v.abs().transpose(-1, -2))
    ed2 = (go.abs() * (t2 + ho * o2.abs())).sum(-1, keepdim=True)
    ed1 = (go.abs() * (tout + al * (t2 + ho * o2.abs()))).sum(-1, keepdim=True)
    D = [(dp * p).sum(-1, keepdim=True) for p in P]
    ds = [P[0] * (dp - D[0]), -lam * P[1] * (dp - D[1])]
    eds = [(rel[0] + hp) * ds[0].abs() + P[0] * (edp + ed1 + 4 * U * (dp.abs() + D[0].abs())),
           (rel[1] + hp) * ds[1].abs() + al * P[1] * (edp + ed2 + 4 * U * (dp.abs() + D[1].abs()))]
    mix = P[0] - lam * P[1]
    emix = rel[0] * P[0] + rel[1] * al * P[1] + hp * mix.abs()
    sq = 2 * U * math.sqrt(nq * rep)

    def grp(t, width):  # sum over the query heads of a key head
        return t.view(b, hk, rep, nk, width).sum(2).permute(0, 2, 1, 3)

    dq = torch.stack([scale * ds[m] @ k[m] for m in range(2)])
    tq = torch.stack([scale * (eds[m] + (su + 4 * U) * ds[m].abs()) @ k[m].abs() for m in range(2)]) + ho * dq.abs()
    dk = torch.stack([grp(scale * ds[m].transpose(-1, -2) @ q[m], d) for m in range(2)], 3)
    tk = torch.stack([grp(scale * (eds[m] + (sq + 4 * U) * ds[m].abs()).transpose(-1, -2) @ q[m].abs(), d) for m in range(2)], 3)
    dv = grp(mix.transpose(-1, -2) @ go, w)
    tv = grp((emix + (sq + 4 * U) * (P[0] + al * P[1])).transpose(-1, -2) @ go.abs(), w) + ho * dv.abs()
    dl = -D[1].sum((0, 2, 3))
    tl = ed2.sum((0, 2, 3)) + 2 * U * math.sqrt(b * nq) * (go.abs() * o2.abs()).sum((0, 2, 3)) + ho * dl.abs()
    return {"out": (out.permute(0, 2, 1, 3), tout.permute(0, 2, 1, 3)), "dq": (dq.permute(1, 3, 2, 0, 4), tq.permute(1, 3, 2, 0, 4)),
            "dk": (dk, tk + ho * dk.abs()), "dv": (dv, tv), "dlam": (dl, tl)}


def check(got, ref, what):
    val, tol = ref
    got = got.detach().double().cpu()
    assert got.shape == val.shape, what
    err = (got - val).abs()
    bad = ~(err <= tol + 1e-30)
    assert not bad.any(), "%s: %d of %d off, worst error %.3e at tolerance %.3e" % (
        what, int(bad.sum()), bad.numel(), err[bad].max().item(), tol[bad][err[bad].argmax()].item())


def inputs(b, nq, nk, h, hk, d, dt, seed=0, qs=1.5):
    g = torch.Generator().manual_seed(seed + 7 * nq + nk + h + d)
    q = (torch.randn((b, nq, h, 2, d), generator=g) * qs).to(DT[dt])
    k = torch.randn((b, nk, hk, 2, d), generator=g).to(DT[dt])
    v = torch.randn((b, nk, hk, 2 * d), generator=g).to(DT[dt])
    lam = (0.2 + 0.6 * torch.rand(h, generator=g)).to(DT[dt])
    go = torch.randn((b, nq, h, 2 * d), generator=g).to(DT[dt])
    return q, k, v, lam, go


def run_case(dev, q, k, v, lam, go, mask=None, frame=0, scale=None, place=lambda t: t):
    from cvpr2021_vspw_implement_amd import ops

    sc = 1 / math.sqrt(q.shape[-1]) if scale is None else scale
    ref = reference(q, k, v, lam, sc, mask, frame, go)
    qd, kd, vd = (place(t.to(dev)).detach().requires_grad_(True) for t in (q, k, v))
    ld = lam.to(dev).requires_grad_(True)
    md = None if mask is None else mask.to(dev)
    out = ops.diff_attention(qd, kd, vd, ld, scale, md, frame)
    check(out, ref["out"], "out")
    out.backward(go.to(dev))
    for name, t in (("dq", qd), ("dk", kd), ("dv", vd), ("dlam", ld)):
        check(t.grad, ref[name], name)
        assert t.grad.dtype == t.dtype
    with torch.no_grad():
        assert torch.equal(ops.diff_attention(qd, kd, vd, ld, scale, md, frame), out)
    return out, (qd, kd, vd, ld)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", [
    (1, 1, 1, 1, 1, 16), (1, 1, 2, 1, 1, 32), (2, 3, 31, 2, 2, 32), (1, 32, 32, 1, 1, 64), (2, 33, 33, 1, 1, 16),
    (1, 65, 64, 2, 1, 32), (1, 129, 127, 2, 2, 64), (2, 300, 257, 4, 2, 16), (1, 7, 130, 8, 2, 64), (2, 200, 5, 3, 1, 32),
    (1, 1, 25200, 4, 1, 64), (1, 3, 17000, 2, 2, 16), (2, 2, 7000, 2, 1, 32),
    (1, 40, 700, 2, 2, 32), (1, 1, 1500, 4, 1, 64), (2, 1, 999, 2, 2, 16), (1, 500, 40, 4, 1, 64)])
def test_sizes_and_heads(dev, dt, case):
    run_case(dev, *inputs(*case, dt))


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("nq,nk,frame", [(1, 1, 1), (40, 40, 1), (64, 64, 16), (150, 150, 50), (30, 120, 30), (31, 100, 31),
                                         (90, 40, 10), (200, 200, 1000), (5, 300, 7), (33, 70, 2 ** 31 - 1)])
def test_frames(dev, dt, nq, nk, frame):
    run_case(dev, *inputs(2, nq, nk, 4, 2, 32, dt), frame=frame)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("nq,nk,frame,d", [(1500, 1500, 250, 64), (900, 2100, 300, 16), (2000, 700, 100, 32), (700, 1400, 1, 64),
                                           (130, 5000, 65, 32)])
def test_frames_in_parts(dev, dt, nq, nk, frame, d):
    """Long enough that tiles stream different numbers of parts, one of them or none; with keys hidden as well."""
    mask = torch.rand(1, nk, generator=torch.Generator().manual_seed(nk)) < 0.7
    run_case(dev, *inputs(1, nq, nk, 2, 1, d, dt), mask, frame=frame)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("d", [16, 32, 64])
def test_masks(dev, dt, d):
    """A batch entry without any key, one with a single key, one with alternating keys; then together with frames."""
    q, k, v, lam, go = inputs(3, 50, 90, 2, 1, d, dt)
    mask = torch.zeros(3, 90, dtype=torch.bool)
    mask[1, 77] = True
    mask[2, ::2] = True
    out, leaves = run_case(dev, q, k, v, lam, go, mask)
    assert (out[0] == 0).all() and all((t.grad[0] == 0).all() for t in leaves[:3])
    run_case(dev, q, k, v, lam, go, mask, frame=30)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_what_masked_positions_hold_is_not_used(dev, dt, junk):
    q, k, v, lam, go = inputs(2, 45, 100, 2, 2, 32, dt)
    mask = torch.rand(2, 100, generator=torch.Generator().manual_seed(1)) < 0.6
    k[~mask], v[~mask] = junk, junk
    _, leaves = run_case(dev, q, k, v, lam, go, mask)
    assert (leaves[1].grad[~mask.to(dev)] == 0).all() and (leaves[2].grad[~mask.to(dev)] == 0).all()


@pytest.mark.parametrize("dt", list(DT))
def test_layouts(dev, dt):
    q, k, v, lam, go = inputs(2, 70, 70, 2, 2, 32, dt)
    heads_first = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    maps_first = lambda t: t.movedim(3, 0).contiguous().movedim(0, 3) if t.dim() == 5 else t  # noqa: E731
    wide = lambda t: torch.cat((t, t), -1)[..., :t.shape[-1]]  # noqa: E731
    odd = lambda t: torch.cat((t.reshape(-1)[:1], t.reshape(-1)))[1:].view(t.shape)  # noqa: E731  (off 16-byte alignment)
    last = lambda t: t.transpose(-1, -2).contiguous().transpose(-1, -2)  # noqa: E731  (last dimension not dense)
    ref = None
    for place in (lambda t: t, heads_first, maps_first, wide, odd, last):
        out, leaves = run_case(dev, q, k, v, lam, go, place=place)
        got = [out] + [t.grad for t in leaves]
        if ref is not None:
            assert all(torch.equal(a, b) for a, b in zip(got, ref))
        ref = got


def test_broadcast_keys(dev):
    """Keys and values of one batch entry expanded over the batch: the gradient sums over it."""
    from cvpr2021_vspw_implement_amd import ops

    q, k, v, lam, go = (t.to(dev) for t in inputs(3, 20, 50, 2, 2, 32, "f32"))
    k1, v1 = k[:1].clone().requires_grad_(True), v[:1].clone().requires_grad_(True)
    kf, vf = k[:1].repeat(3, 1, 1, 1, 1).requires_grad_(True), v[:1].repeat(3, 1, 1, 1).requires_grad_(True)
    a = ops.diff_attention(q, k1.expand(3, -1, -1, -1, -1), v1.expand(3, -1, -1, -1), lam)
    b = ops.diff_attention(q, kf, vf, lam)
    assert torch.equal(a, b)
    a.backward(go)
    b.backward(go)
    assert torch.equal(k1.grad, kf.grad.sum(0, keepdim=True)) and torch.equal(v1.grad, vf.grad.sum(0, keepdim=True))


@pytest.mark.parametrize("dt", list(DT))
def test_growing_and_large_scores(dev, dt):
    """Scores that grow along the keys by hundreds (the running maximum moves in every tile), and all-equal ones."""
    q, k, v, lam, go = inputs(1, 40, 200, 1, 1, 32, dt)
    q = q.abs() + 0.5
    k = (k * 0.1 + torch.linspace(-4, 4, 200)[None, :, None, None, None]).to(DT[dt])
    run_case(dev, q, k, v, lam, go)
    run_case(dev, torch.zeros_like(q), k, v, lam, go)


def test_lam_float32_with_bf16(dev):
    q, k, v, lam, go = inputs(1, 40, 60, 4, 2, 32, "bf16")
    _, leaves = run_case(dev, q, k, v, lam.float(), go)
    assert leaves[3].grad.dtype == torch.float32


def test_partial_gradients_and_reproducibility(dev):
    from cvpr2021_vspw_implement_amd import ops

    q, k, v, lam, go = (t.to(dev) for t in inputs(2, 300, 400, 2, 1, 32, "bf16"))

    def grads(which):
        ts = [t.detach().requires_grad_(i in which) for i, t in enumerate((q, k, v, lam))]
        out = ops.diff_attention(*ts, frame=100)
        return dict(zip(which, torch.autograd.grad(out, [ts[i] for i in which], go)))

    full = grads((0, 1, 2, 3))
    for which in ((0,), (1,), (2,), (3,), (0, 3), (1, 2), (0, 1, 2, 3)):
        got = grads(which)
        assert all(torch.equal(got[i], full[i]) for i in which), which


def test_empty(dev):
    from cvpr2021_vspw_implement_amd import ops

    lam = torch.ones(2, device=dev, requires_grad=True)
    q = torch.randn(2, 3, 2, 2, 16, device=dev, requires_grad=True)
    k = torch.randn(2, 0, 2, 2, 16, device=dev, requires_grad=True)
    v = torch.randn(2, 0, 2, 32, device=dev, requires_grad=True)
    out = ops.diff_attention(q, k, v, lam)
    assert out.shape == (2, 3, 2, 32) and (out == 0).all()
    out.sum().backward()
    assert (q.grad == 0).all() and (lam.grad == 0).all() and k.grad.shape == k.shape
    assert ops.diff_attention(q[:, :0], q, torch.randn(2, 3, 2, 32, device=dev), lam).shape == (2, 0, 2, 32)


def test_gradient_differences(dev):
    """The gradients against central differences of the forward kernel in float32 (step 2^-7)."""
    from cvpr2021_vspw_implement_amd import ops

    ts = [t.to(dev) for t in inputs(1, 6, 9, 1, 1, 16, "f32", qs=0.7)]
    go = ts.pop()

    def f(args):
        return (ops.diff_attention(*args).double() * go).sum().item()

    leaves = [t.clone().requires_grad_(True) for t in ts]
    (ops.diff_attention(*leaves) * go).sum().backward()
    h = 2.0 ** -7
    for i, t in enumerate(ts):
        for j in range(0, t.numel(), max(1, t.numel() // 12)):
            d = torch.zeros_like(t)
            d.view(-1)[j] = h
            up, dn = list(ts), list(ts)
            up[i], dn[i] = t + d, t - d
            num = (f(up) - f(dn)) / (2 * h)
            # |f| < 100: rounding 100 * 2^-22 / h = 3e-3; truncation h^2 / 6 * third derivative (< 30) = 3e-4
            assert abs(num - leaves[i].grad.view(-1)[j].item()) < 5e-3, (i, j)


def test_captured_step(dev):
    """Forward and backward of two different sizes captured in two graphs, replayed in turn with eager work between."""
    from cvpr2021_vspw_implement_amd import ops

    def make(nq, nk):
        ts = [t.to(dev) for t in inputs(1, nq, nk, 2, 1, 32, "bf16")]
        go = ts.pop()

        def step():
            leaves = [t.detach().requires_grad_(True) for t in ts]
            out = ops.diff_attention(*leaves, frame=64)
            return (out.detach(),) + torch.autograd.grad(out, leaves, go)

        eager = [t.clone() for t in step()]
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step()
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        return g, out, eager, step

    a, b = make(200, 200), make(3, 900)
    for _ in range(3):
        for g, out, eager, step in (a, b):
            for t in out:
                t.zero_()
            g.replay()
            step()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, eager))


def test_diff_lambda(dev):
    from cvpr2021_vspw_implement_amd import ops

    g = torch.Generator().manual_seed(4)
    ts = [0.1 * torch.randn((3, 70), generator=g) for _ in range(4)]
    r = [t.double().requires_grad_(True) for t in ts]
    ref = torch.exp((r[0] * r[1]).sum(1)) - torch.exp((r[2] * r[3]).sum(1)) + 0.8
    w = torch.tensor([1.0, -2.0, 0.5])
    (ref * w).sum().backward()
    d = [t.to(dev).requires_grad_(True) for t in ts]
    lam = ops.diff_lambda(*d, 0.8)
    (lam * w.to(dev)).sum().backward()
    # values O(1): a 70-term sum, expf, two additions
    assert (lam.double().cpu() - ref).abs().max() < 32 * U
    assert all((a.grad.double().cpu() - b.grad).abs().max() < 32 * U for a, b in zip(d, r))


def test_refusals(dev):
    from cvpr2021_vspw_implement_amd import ops

    q, k, v, lam, _ = (t.to(dev) for t in inputs(1, 4, 6, 2, 1, 16, "f32"))
    bad = [
        (q[..., :8], k[..., :8], v[..., :16], lam), (q.half(), k.half(), v.half(), lam), (q, k.bfloat16(), v, lam),
        (q, k, v[..., :16], lam), (q, k[:, :5], v, lam), (q[:, :, :1], torch.cat((k, k), 2), v, lam[:1]), (q, k, v, lam[:1]),
        (q[0], k[0], v[0], lam), (q.cpu(), k, v, lam), (q, k, v, lam.bfloat16()), (q, k, v, lam.double())]
    for args in bad:
        with pytest.raises(RuntimeError):
            ops.diff_attention(*args)
    for mask in (torch.ones(1, 5, dtype=torch.bool, device=dev), torch.ones(1, 6, device=dev), torch.ones(1, 6, dtype=torch.bool)):
        with pytest.raises(RuntimeError):
            ops.diff_attention(q, k, v, lam, key_mask=mask)
    for kw in (dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=1e-60),
               dict(frame=-1), dict(frame=2 ** 31)):
        with pytest.raises(ValueError):
            ops.diff_attention(q, k, v, lam, **kw)
    with pytest.raises(RuntimeError):
        ops.diff_lambda(lam, lam, lam, lam, 0.1)


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("case", [(1, 1152, 1152, 4, 2, 16), (2, 700, 900, 2, 1, 32), (1, 600, 1300, 2, 2, 64)])
def test_waves_of_a_workgroup_wait_for_each_other(dev, dt, case):
    """Workgroups of four waves on short tiles: the values, and the same bits from every run."""
    from cvpr2021_vspw_implement_amd import ops

    q, k, v, lam, go = inputs(*case, dt)
    out, leaves = run_case(dev, q, k, v, lam, go)
    qd, kd, vd, ld = (t.detach().requires_grad_(True) for t in leaves)
    god = go.to(dev)
    for _ in range(40):
        again = ops.diff_attention(qd, kd, vd, ld)
        assert torch.equal(again, out)
        assert all(torch.equal(g, t.grad) for g, t in zip(torch.autograd.grad(again, (qd, kd, vd, ld), god), leaves))


def test_a_second_derivative_is_refused(dev):
    from cvpr2021_vspw_implement_amd import ops

    ts = [t.to(dev).requires_grad_(True) for t in inputs(1, 4, 6, 2, 1, 16, "f32")[:4]]
    out = ops.diff_attention(*ts)
    g, = torch.autograd.grad((out * out).sum(), ts[0], create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_many_layouts_of_one_shape(dev):
    """Calls whose types and shapes agree and whose strides, alignment and scale differ."""
    from cvpr2021_vspw_implement_amd import ops

    q, k, v, lam, go = (t.to(dev) for t in inputs(2, 70, 70, 4, 2, 16, "f32"))
    big = torch.zeros(q.numel() + 4, device=dev)
    odd = big[1:1 + q.numel()].view(q.shape).copy_(q)  # 4 bytes past a boundary
    turned = q.transpose(1, 2).contiguous().transpose(1, 2)
    for scale in (None, 0.5):
        a = ops.diff_attention(q, k, v, lam, scale)
        for other in (odd, turned, q.clone()):
            leaf = other.detach().requires_grad_(True)
            b = ops.diff_attention(leaf, k, v, lam, scale)
            g, = torch.autograd.grad(b, leaf, go)
            assert torch.equal(a, b) and g.shape == q.shape
    assert not torch.equal(ops.diff_attention(q, k, v, lam, 0.5), ops.diff_attention(q, k, v, lam, 0.25))


def test_queries_that_are_the_keys_and_another_stream(dev):
    """One tensor as q and k (its gradient is the sum of both), a broadcast output gradient, work on a stream of its own."""
    from cvpr2021_vspw_implement_amd import ops

    q, _, v, lam, _ = (t.to(dev) for t in inputs(2, 150, 150, 2, 2, 32, "f32"))
    a, b, c = q.clone().requires_grad_(True), q.clone().requires_grad_(True), q.clone().requires_grad_(True)
    out = ops.diff_attention(a, b, v, lam)
    out.sum().backward()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.diff_attention(c, c, v, lam)
        other.sum().backward()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(out, other) and torch.equal(c.grad, a.grad + b.grad)


def test_two_threads(dev):
    import threading

    from cvpr2021_vspw_implement_amd import ops

    cases = [[t.to(dev) for t in inputs(1, 64 + 8 * i, 96, 2, 1, 16, "f32")[:4]] for i in range(4)]
    refs = [ops.diff_attention(*c) for c in cases]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(10):
                got = [ops.diff_attention(*c) for c in cases]
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(x, y) for x, y in zip(got, refs)):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("dt", list(DT))
@pytest.mark.parametrize("nq,nk,keys", [(1, 1, None), (70, 1, None), (300, 40, [17]), (5, 9000, [4097]), (140, 9000, []), (3, 9000, [0, 8999])])
def test_a_single_key_has_no_score_gradient(dev, dt, nq, nk, keys):
    """The softmax of one key is 1 whatever the score: dq and dk are zero, not rounding; two keys are an ordinary case."""
    mask = None
    if keys is not None:
        mask = torch.zeros(2, nk, dtype=torch.bool)
        mask[:, keys] = True
    out, (q, k, v, lam) = run_case(dev, *inputs(2, nq, nk, 2, 1, 16, dt), mask)
    few = nk == 1 or (keys is not None and len(keys) < 2)
    assert bool((q.grad == 0).all()) == few and bool((k.grad == 0).all()) == few


def test_offsets_beyond_32_bits(dev):
    """A cache of 2^31 and more elements per tensor, three keys of it visible: the values and gradients of those three alone."""
    from cvpr2021_vspw_implement_amd import ops

    nk, at = (1 << 24) + 70000, [5, (1 << 24) + 3, (1 << 24) + 69999]
    q, k3, v3, lam, go = (t.to(dev) for t in inputs(1, 2, 3, 2, 1, 64, "bf16"))
    k, v = (torch.zeros((1, nk) + t.shape[2:], dtype=t.dtype, device=dev) for t in (k3, v3))
    mask = torch.zeros(1, nk, dtype=torch.bool, device=dev)
    k[:, at], v[:, at], mask[:, at] = k3, v3, True
    assert k.numel() > 2 ** 31
    got, want = [], []
    for res, kk, vv, m in ((got, k, v, mask), (want, k3, v3, None)):
        leaves = [t.detach().requires_grad_(True) for t in (q, kk, vv, lam)]
        out = ops.diff_attention(*leaves, key_mask=m)
        g = torch.autograd.grad(out, leaves, go)
        pick = (lambda t: t[:, at]) if m is not None else (lambda t: t)
        res += [out.detach(), g[0], pick(g[1]), pick(g[2]), g[3]]
        if m is not None:  # the last rows of the cache behind the last visible key, and the first
            assert not g[1][:, :5].any() and not g[2][:, at[1] + 1:at[2]].any()
        del g, leaves
    for x, y in zip(got, want):  # sums in another order, then one rounding each: neighbours in bf16
        assert (x.float() - y.float()).abs().max() <= 2.0 ** -7 * y.float().abs().max()
