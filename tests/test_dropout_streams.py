"""Where a Dropout module's masks come from: its seed and its count of calls, through checkpoints and copies of a network."""
import pytest
import torch

from pointcloud_rl_amd import configs
from pointcloud_rl_amd.methods import build_agent
from pointcloud_rl_amd.networks import Dropout, LinearMLP

OBS = {"xyz": [3, 64], "rgb": [3, 64]}


def drops(module):
    return [m for m in module.modules() if isinstance(m, Dropout)]


def make_agent(seed, device="cpu", batch_size=6, **kw):
    torch.manual_seed(seed)
    cfg = dict(configs.sac_dmc(6, 4, batch_size, head_hidden=64), **kw)
    cfg["critic_cfg"]["nn_cfg"]["mlp_cfg"]["dropout"] = 0.1
    cfg["env_params"] = configs.env_params(OBS, 4)
    return build_agent(cfg).to(device)


def test_checkpoints_keep_the_masks_to_come(tmp_path):
    """A strict load of an agent's own checkpoint: every entry has its place, and every Dropout goes on where the saved one stood."""
    from pointcloud_rl_amd.utils.checkpoint import load_checkpoint, save_checkpoint
    agent, path = make_agent(0), str(tmp_path / "model.ckpt")
    for i, d in enumerate(drops(agent)):
        d.calls.fill_(i + 3)
    save_checkpoint(agent, path)
    other = make_agent(1)
    assert {d.seed for d in drops(agent)}.isdisjoint(d.seed for d in drops(other))
    load_checkpoint(other, path, map_location="cpu", strict=True)
    assert [(d.seed, int(d.calls)) for d in drops(other)] == [(d.seed, int(d.calls)) for d in drops(agent)]
    assert len({d.seed for d in drops(agent)}) == len(drops(agent)) == 8         # two hidden layers of two heads, and of their targets


def test_files_without_masks_leave_a_module_its_own(tmp_path):
    from pointcloud_rl_amd.utils.checkpoint import load_checkpoint, save_checkpoint
    plain, path = LinearMLP([5, 8, 3]), str(tmp_path / "plain.ckpt")
    save_checkpoint(plain, path)
    mlp = LinearMLP([5, 8, 3], dropout=0.5)
    drop = mlp.mlp.drop0
    drop.calls.fill_(4)
    before = (drop.seed, int(drop.calls))
    load_checkpoint(mlp, path, strict=True)
    mlp.load_state_dict(plain.state_dict(), strict=True)
    assert (drop.seed, int(drop.calls)) == before and torch.equal(mlp.mlp.linear0.weight, plain.mlp.linear0.weight)
    drop._load_from_state_dict({"calls": torch.tensor([9])}, "", {}, True, [], [], [])      # half of a stream is none
    assert (drop.seed, int(drop.calls)) == before


@pytest.mark.parametrize("shared", [False, True])
def test_online_and_target_networks_draw_masks_of_their_own(shared):
    """The target network is built afresh or copied from the online one: no two of their Dropouts share a seed.  The weights are copies."""
    agent = make_agent(0, shared_backbone=shared)
    online, target = agent.critic, agent.target_critic
    seeds = [d.seed for d in drops(online) + drops(target)]
    assert len(seeds) == 8 and len(set(seeds)) == 8
    for a, b in zip(online.parameters(), target.parameters()):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_a_resumed_run_draws_the_masks_it_would_have_drawn(cuda, tmp_path):
    """Three steps, a checkpoint, three more in a freshly built agent: the parameters of six steps, to the bit."""
    from pointcloud_rl_amd.synthetic import SyntheticReplay
    from pointcloud_rl_amd.utils.checkpoint import load_checkpoint, save_checkpoint
    mem = SyntheticReplay(6, 64, 4, seed=3, device=cuda)
    g = torch.Generator().manual_seed(11)
    eps = [[torch.randn(6, 4, generator=g).to(cuda) for _ in range(2)] for _ in range(6)]

    def run(agent, lo, hi):
        for u in range(lo, hi + 1):
            agent.actor.head.noise_override = list(eps[u - 1][:2 if u % 2 == 0 else 1])
            agent.update_parameters(mem, u)

    whole, first, path = make_agent(0, cuda), make_agent(0, cuda), str(tmp_path / "model.ckpt")
    run(whole, 1, 6)
    run(first, 1, 3)
    save_checkpoint(first, path)
    resumed = make_agent(123, cuda)
    load_checkpoint(resumed, path, map_location="cpu", strict=True)
    run(resumed, 4, 6)
    for (n, p), (_, q) in zip(whole.named_parameters(), resumed.named_parameters()):
        assert torch.equal(p, q), n
    assert [int(d.calls) for d in drops(whole)] == [int(d.calls) for d in drops(resumed)]
