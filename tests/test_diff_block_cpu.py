"""Host side of the differential non-local block: construction, parameters, optimizer groups, the config switch."""
import pytest
import torch


def test_construction_and_refusals():
    from cvpr2021_vspw_implement_amd.models.non_local import NLBlockND

    m = NLBlockND(in_channels=256, mode="differential", dimension=2)
    assert m.heads == 2 and tuple(m.lambda_q1.shape) == (2, 32) and m.norm.num_groups == 2
    assert torch.allclose(m.norm.weight, torch.full((128,), 0.2))
    keys = set(m.state_dict())
    dot = set(NLBlockND(in_channels=256, mode="dot", dimension=2).state_dict())
    assert dot < keys and keys - dot == {"lambda_q1", "lambda_k1", "lambda_q2", "lambda_k2", "norm.weight", "norm.bias"}
    for kw in (dict(heads=3), dict(heads=16), dict(frame_causal=True)):
        with pytest.raises(ValueError):
            NLBlockND(in_channels=256, mode="differential", dimension=2, **kw)
    with pytest.raises(ValueError):
        NLBlockND(in_channels=256, mode="difference")
    with pytest.raises(NotImplementedError):
        NLBlockND(in_channels=256, mode="embedded")


def test_the_dot_block_draws_the_same_initial_weights_as_before():
    """Mode 'dot' makes no further draws: the generator stands where g, W_z, theta and phi left it."""
    from cvpr2021_vspw_implement_amd import nn as vnn
    from cvpr2021_vspw_implement_amd.models.non_local import NLBlockND

    torch.manual_seed(5)
    NLBlockND(in_channels=16, mode="dot", dimension=2)
    a = torch.rand(4)
    torch.manual_seed(5)
    for cin, cout in ((16, 8), (8, 16), (16, 8), (16, 8)):
        vnn.Conv2d(cin, cout, 1)
    assert torch.equal(a, torch.rand(4))


def test_optimizer_groups_take_every_parameter():
    import cvpr2021_vspw_implement_amd.models as M
    from cvpr2021_vspw_implement_amd.train import group_weight

    dec = M.ModelBuilder.build_decoder(arch="nonlocal2d_differential", fc_dim=2048, num_class=12)
    decay, rest = (g["params"] for g in group_weight(dec))
    ids = {id(p): n for n, p in dec.named_parameters()}
    assert len(decay) + len(rest) == len(ids)
    assert all(ids[id(p)].endswith("weight") and "norm" not in ids[id(p)] for p in decay)


@pytest.mark.parametrize("arch,mode", [("ppm_deepsup", "dot"), ("nonlocal2d", "dot"), ("nonlocal2d_differential", "differential")])
def test_the_config_selects_the_block_of_the_clip_model(arch, mode):
    from cvpr2021_vspw_implement_amd import train_clip2
    from cvpr2021_vspw_implement_amd.config import cfg

    cfg = cfg.clone()
    cfg.merge_from_list(["MODEL.arch_encoder", "resnet18dilated", "MODEL.arch_decoder", arch, "MODEL.fc_dim", 512])
    args = train_clip2.build_parser().parse_args(["--method", "nonlocal3d"])
    args.num_class = 7
    module = train_clip2.build_module(cfg, args, 7, training=False)
    assert module.nonlocalblock.mode == mode
