"""Host side of the group norm / dropout entry points: refusals and workspace arithmetic that need no GPU."""
import ctypes

import pytest
import torch


def test_cpu_tensors_are_refused():
    from cvpr2021_vspw_implement_amd import ops

    rng = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError):
        ops.dropout(torch.ones(4), 0.5, rng)
    with pytest.raises(RuntimeError):
        ops.group_norm_act(torch.ones(1, 4, 2, 2), 2)
    with pytest.raises(RuntimeError):
        ops.rng_next(rng)


def test_c_entry_points_refuse_bad_arguments():
    """Every refusal comes before a launch; the pointers are never followed."""
    from cvpr2021_vspw_implement_amd import _C

    lib = _C.load()
    p = ctypes.c_void_p(4096)
    ok = dict(x=p, y=p, n=2, hw=9, c=8, dtype=0, p=0.5, rng=p)

    def drop(**kw):
        a = dict(ok, **kw)
        return lib.vspw_dropout(a["x"], a["y"], a["n"], a["hw"], a["c"], a["dtype"], a["p"], a["rng"], 0, None)

    for kw in (dict(x=None), dict(y=None), dict(rng=None), dict(n=0), dict(hw=0), dict(c=0), dict(dtype=3), dict(p=-0.1),
               dict(p=1.1), dict(p=float("nan")), dict(n=2 ** 40), dict(hw=2 ** 62)):
        assert drop(**kw) == -1, kw
    assert lib.vspw_rng_next(None, p, None) == -1 and lib.vspw_rng_next(p, None, None) == -1

    def norm(**kw):
        a = dict(dict(x=p, y=p, n=2, hw=9000, c=8, groups=2, dtype=0, eps=1e-5, act=0, p=0.0, rng=None, ws=p, wsb=1 << 20), **kw)
        return lib.vspw_group_norm_fwd(a["x"], a["y"], a["n"], a["hw"], a["c"], a["groups"], a["dtype"], None, None, a["eps"],
                                       a["act"], a["p"], a["rng"], 0, None, a["ws"], a["wsb"], None)

    for kw in (dict(x=None), dict(y=None), dict(n=0), dict(groups=3), dict(groups=0), dict(dtype=-1), dict(eps=-1.0),
               dict(act=4), dict(act=-1), dict(p=0.5), dict(ws=None), dict(wsb=0), dict(x=ctypes.c_void_p(4100)),
               dict(hw=2 ** 61)):
        assert norm(**kw) == -1, kw
    assert lib.vspw_group_norm_bwd(p, p, p, 2, 9, 8, 2, 0, None, None, 0, 0.0, None, 0, None, None, None, p, 1 << 20, None) == -1


@pytest.mark.parametrize("n,hw,c,groups,dt", [(1, 1, 1, 1, 0), (10, 3600, 512, 32, 0), (4, 14161, 256, 32, 1), (3, 7, 33, 11, 2)])
def test_workspaces_cover_the_partials(n, hw, c, groups, dt):
    from cvpr2021_vspw_implement_amd import _C

    fwd = _C.query("vspw_group_norm_fwd_workspace", n, hw, c, groups, dt)
    bwd = _C.query("vspw_group_norm_bwd_workspace", n, hw, c, groups, dt)
    # one workgroup per image and group needs no partial sums in the forward pass
    assert (fwd == 0) == (hw <= 7) and bwd >= n * 2 * c * 8
    assert _C.query("vspw_group_norm_fwd_workspace", n, hw, c, c + 1, dt) == 0


def test_fused_sequential_still_refuses_bare_layers():
    from cvpr2021_vspw_implement_amd import nn as vnn

    for m in (torch.nn.ReLU(), torch.nn.Dropout2d(0.1)):
        with pytest.raises(NotImplementedError):
            vnn.FusedSequential(m)(torch.ones(1, 4, 2, 2))
    with pytest.raises(NotImplementedError):
        vnn.GroupNorm(2, 4)(torch.ones(1, 4, 2, 2), "none", torch.nn.Dropout2d(0.1))


def test_dropout_layers_keep_state_dicts_and_draw_their_seed_from_torch():
    from cvpr2021_vspw_implement_amd import nn as vnn

    torch.manual_seed(3)
    a = vnn.Dropout(0.1)
    torch.manual_seed(3)
    b = vnn.Dropout2d(0.1)
    assert torch.equal(a.rng_state, b.rng_state) and not a.state_dict() and a.rng_state[1] == 0
    assert a.manual_seed(7, 2).rng_state.tolist() == [7, 2]
