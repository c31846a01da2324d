"""Augmentations of runs of steps [B, T, C, N]: every cloud of a run is a row with draws of its own, and tensors that hold too few rows never reach
the encoder."""
from types import SimpleNamespace

import pytest
import torch

from pointcloud_rl_amd.augmentations import ColorJitterPoints, GlobalRotScaleTrans, RandomDownSample, RandomJitterPoints
from pointcloud_rl_amd.networks.pointnet import AugmentedObs, batch_rows, checked_aug_desc

B, T, N = 3, 4, 32


def run(device="cpu", seed=0):
    g = torch.Generator().manual_seed(seed)
    return AugmentedObs(xyz=torch.randn(B, T, 3, N, generator=g).to(device), rgb=torch.randint(0, 256, (B, T, 3, N), generator=g).to(torch.uint8).to(device))


def rows_of(obs):
    out = AugmentedObs({k: v.reshape((-1,) + tuple(v.shape[2:])) for k, v in obs.items()})
    out.aug, out.repeat = obs.aug, obs.repeat
    return out


def test_draws_are_made_for_every_cloud():
    obs = run()
    assert batch_rows(obs) == batch_rows(rows_of(obs)) == B * T
    assert GlobalRotScaleTrans(main_key="xyz")(obs).aug["affine"].shape == (B * T, 3, 4)
    jitter = RandomJitterPoints(main_key="xyz")
    jitter.noise_override = [torch.zeros(B * T, 3, N)]
    assert jitter(obs).aug["jitter_noise"].shape == (B * T, 3, N)
    with pytest.raises(NotImplementedError, match="rgb"):
        RandomDownSample(main_key="xyz", req_keys=["xyz"], max_num_points=8)(obs)


@pytest.mark.parametrize("aug", [dict(affine=torch.zeros(B, 3, 4)), dict(jitter_noise=torch.zeros(B * T - 1, 3, N)),
                                 dict(affine=torch.zeros(B * T, 3, 4), row_mul=2), dict(affine=torch.zeros(B * T, 3, 4), row_add=1),
                                 dict(affine=torch.zeros(B * T, 3, 4, dtype=torch.float64)), dict(affine=torch.zeros(B * T, 4, 3).transpose(1, 2)),
                                 dict(affine=torch.zeros(B * T, 3, 4)),
                                 dict(color=dict(order=[0, 1, 2, 3], factors=[None, 0.5, None, None], mean=torch.zeros(B)))])
def test_too_few_rows_are_refused(aug):
    """(The last affine has its rows, on the wrong device.)"""
    with pytest.raises(ValueError, match="clouds"):
        checked_aug_desc(aug, SimpleNamespace(B=B * T, N=N, row_div=1))
    assert checked_aug_desc({}, SimpleNamespace(B=B * T, N=N, row_div=1)) is None


@pytest.mark.gpu
def test_an_augmented_run_is_its_clouds_augmented(cuda):
    """The recurrent backbone's features of an augmented run: the encoder's on the same rows with the same draws, to the bit."""
    from pointcloud_rl_amd import configs
    from pointcloud_rl_amd.methods import build_agent
    torch.manual_seed(0)
    cfg = configs.recurrent(configs.sac_dmc(6, 4, 4, head_hidden=64), state_dim=8)
    cfg["env_params"] = configs.env_params({"xyz": [3, N], "rgb": [3, N]}, 4)
    backbone = build_agent(cfg).to(cuda).actor.backbone
    obs = run(cuda)
    seen = []
    for make in (lambda: GlobalRotScaleTrans(main_key="xyz", translation_range=[0.1, 0.1, 0.1]), lambda: RandomJitterPoints(main_key="xyz", seed=3),
                 lambda: RandomDownSample(main_key="xyz", req_keys=["xyz", "rgb"], max_num_points=20), lambda: ColorJitterPoints(main_key="rgb", req_keys="rgb")):
        augmented = make()(obs)
        with torch.no_grad():
            got = backbone._encode(augmented, None, False)
            want = backbone.visual_nn(rows_of(augmented))
            plain = backbone._encode(obs, None, False)
        assert got.shape[:2] == (B, T) and torch.equal(got.reshape(B * T, -1), want) and not torch.equal(got, plain)
        seen.append(got)
    assert not any(torch.equal(a, b) for i, a in enumerate(seen) for b in seen[:i])
    repeated = AugmentedObs(obs)
    repeated.repeat = 2
    with pytest.raises(NotImplementedError, match="repeated"):
        backbone._encode(repeated, None, False)
