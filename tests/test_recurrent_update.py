"""What a recurrent agent's update learns from: the histories its target is formed over, on runs of any number of episodes."""
import numpy as np
import pytest
import torch

from pointcloud_rl_amd import configs
from pointcloud_rl_amd.methods import build_agent

OBS = {"xyz": [3, 64], "rgb": [3, 64]}


def make_agent(device, batch_size=3, **kw):
    torch.manual_seed(0)
    cfg = configs.recurrent(configs.sac_dmc(6, 4, batch_size, head_hidden=64), state_dim=8, **kw)
    cfg["env_params"] = configs.env_params(OBS, 4)
    agent = build_agent(cfg).to(device)
    agent._prepare()
    return agent


def make_batch(device, lengths, H, ends=(), seed=6):
    """[B, H] runs with valid steps in front, episodes ending at (row, step); next_obs is the next step's obs inside an episode."""
    g = torch.Generator().manual_seed(seed)
    B = len(lengths)
    r = lambda *s: torch.randn(*s, generator=g).to(device)
    obs = lambda: {"xyz": r(B, H, 3, 64), "rgb": torch.randint(0, 256, (B, H, 3, 64), generator=g).to(torch.uint8).to(device)}
    valid = (torch.arange(H)[None] < torch.tensor(lengths)[:, None])[..., None].to(device)
    batch = dict(obs=obs(), next_obs=obs(), actions=r(B, H, 4).clamp(-1, 1), rewards=r(B, H, 1), dones=torch.zeros(B, H, 1, dtype=torch.bool, device=device),
                 episode_dones=torch.zeros(B, H, 1, dtype=torch.bool, device=device), is_valid=valid)
    for b, t in ends:
        batch["episode_dones"][b, t] = True
    for k, v in batch["next_obs"].items():
        for b in range(B):
            for t in range(H - 1):
                if not batch["episode_dones"][b, t]:
                    v[b, t] = batch["obs"][k][b, t + 1]
    return batch


def episodes(batch):
    """(row, first step, behind the last step, number of episodes of the row in front) of every episode of every run."""
    ends, valid = batch["episode_dones"][..., 0].cpu(), batch["is_valid"][..., 0].cpu()
    for b in range(len(ends)):
        n, lo, before = int(valid[b].sum()), 0, 0
        for t in range(n):
            if ends[b, t] or t == n - 1:
                yield b, lo, t + 1, before
                lo, before = t + 1, before + 1


@pytest.mark.parametrize("seed", range(20))
def test_every_next_observation_follows_its_episodes_first_one(seed):
    """The runs of the target, against lists put together episode by episode: what they hold, where they restart, where they end."""
    from pointcloud_rl_amd.methods.recurrent import with_target_history
    g = np.random.RandomState(seed)
    B, H = g.randint(1, 5), g.randint(1, 9)
    lengths = g.randint(0 if B > 1 else 1, H + 1, size=B)
    lengths[0] = max(1, lengths[0])
    obs, nxt = torch.arange(B * H).reshape(B, H, 1), 1000 + torch.arange(B * H).reshape(B, H, 1)
    batch = dict(obs=dict(state=obs), next_obs=dict(state=nxt), rewards=torch.zeros(B, H, 1),
                 episode_dones=torch.from_numpy(g.rand(B, H, 1) < (0.0, 0.3, 1.0)[seed % 3]),
                 is_valid=(torch.arange(H)[None] < torch.from_numpy(lengths)[:, None])[..., None])
    out = with_target_history(batch)
    runs, dones = [[] for _ in range(B)], [[] for _ in range(B)]
    for b, lo, hi, _ in episodes(batch):
        runs[b] += [int(obs[b, lo])] + nxt[b, lo:hi, 0].tolist()
        dones[b] += [False] + batch["episode_dones"][b, lo:hi, 0].tolist()
    width = out["next_obs"]["state"].shape[1]
    assert out["next_is_valid"].shape == out["next_episode_dones"].shape == (B, width, 1)
    for b in range(B):
        n = len(runs[b])
        assert out["next_is_valid"][b, :, 0].tolist() == [True] * n + [False] * (width - n)
        assert out["next_obs"]["state"][b, :n, 0].tolist() == runs[b]
        assert out["next_episode_dones"][b, :n, 0].tolist() == dones[b]
        for t in range(lengths[b]):
            assert int(out["next_obs"]["state"][b, out["next_at"][b, t, 0], 0]) == int(nxt[b, t])
    assert torch.equal(out["obs"]["state"], obs) and torch.equal(batch["next_obs"]["state"], nxt)
    whole = dict(batch)
    del whole["is_valid"]                                # every step counts
    assert bool(with_target_history(whole)["next_is_valid"].any(1).all())


# float32 networks evaluated row by row instead of in one batch, as in tests/test_recurrent_gpu.py: other orders of the sums
LOSS_TOL, GRAD_TOL = 1e-4, 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,ends", [([5, 2, 4], [(0, 2)]), ([5, 5, 5], []), ([4, 1, 5], [(0, 0), (0, 1), (2, 4), (2, 2)])])
def test_the_target_has_seen_what_the_policy_has_seen(cuda, lengths, ends):
    """The update's loss and gradient: those of the same networks over each episode on its own, the target's run beginning with the episode's
    first observation."""
    agent = make_agent(cuda)
    batch = make_batch(cuda, lengths, 5, ends)
    most = max(before + 1 for _, _, _, before in episodes(batch))
    eps = torch.randn(3, 5 + most, 4, generator=torch.Generator().manual_seed(8)).to(cuda)
    state = {k: v.clone() for k, v in agent.state_dict().items()}
    agent.actor.head.noise_override = [eps]
    loss = float(agent._step_body(batch, False, False)["critic_loss"])
    grad = agent._flat["critic"].grad.clone()
    agent.load_state_dict(state)
    agent.encoder.invalidate_packed()
    agent._flat["critic"].zero_grad()
    want = 0.0
    for b, lo, hi, before in episodes(batch):
        cut = lambda o: {k: v[b:b + 1, lo:hi] for k, v in o.items()}
        with torch.no_grad():
            history = {k: torch.cat((batch["obs"][k][b:b + 1, lo:lo + 1], v), 1) for k, v in cut(batch["next_obs"]).items()}
            agent.actor.head.noise_override = [eps[b:b + 1, lo + before:hi + before + 1]]
            a, nlp = agent.actor(history, mode="max-entropy")
            q = (agent.target_critic(history, a).min(-1, keepdim=True).values + agent._alpha_t * nlp)[:, 1:]
            y = batch["rewards"][b:b + 1, lo:hi] + agent.gamma * q
        part = (agent.critic(cut(batch["obs"]), batch["actions"][b:b + 1, lo:hi]) - y).square().sum() / sum(lengths)
        part.backward()
        want += float(part.detach())
    assert loss == pytest.approx(want, rel=LOSS_TOL)
    by_episode = agent._flat["critic"].grad
    assert float((grad - by_episode).norm() / by_episode.norm()) < GRAD_TOL


@pytest.mark.gpu
def test_the_targets_features_are_the_online_ones_of_the_next_step(cuda):
    """Inside an episode next_obs[t] is obs[t + 1]: the core's result behind it is the one that the online networks form there."""
    from pointcloud_rl_amd.methods.recurrent import with_target_history
    agent = make_agent(cuda)
    batch = make_batch(cuda, [6, 6, 3], 6, [(0, 2)])
    out = with_target_history(batch)
    value = agent.critic.values[0]

    def features(obs, dones, valid):
        value(obs, batch["actions"].new_zeros(valid.shape[:2] + (4,)), save_feature=True, episode_dones=dones, is_valid=valid)
        return value.backbone.pop_attr("saved_feature")

    with torch.no_grad():
        online = features(batch["obs"], batch["episode_dones"], batch["is_valid"])
        target = features(out["next_obs"], out["next_episode_dones"], out["next_is_valid"])
    inside = 0
    for b, lo, hi, _ in episodes(batch):
        for t in range(lo, hi - 1):
            a, c = target[b, int(out["next_at"][b, t])], online[b, t + 1]
            assert float((a - c).abs().max()) <= 2000 * 2.0 ** -24 * max(1.0, float(c.abs().max())), (b, t)      # tests/test_recurrent_gpu.py's bound
            inside += 1
    assert inside == 2 + 2 + 5 + 2


@pytest.mark.gpu
def test_padding_may_hold_anything(cuda):
    """NaN and infinities behind the valid steps, in every tensor that can hold them: the metrics and gradients of clean padding."""
    lengths, H = [5, 2, 4], 5
    g = torch.Generator().manual_seed(9)
    eps = [torch.randn(3, n, 4, generator=g).to(cuda) for n in (H + 1, H)]

    def run(fill):
        batch = make_batch(cuda, lengths, H)
        for v in (batch["obs"]["xyz"], batch["next_obs"]["xyz"], batch["actions"], batch["rewards"]):
            for b, n in enumerate(lengths):
                v[b, n:] = fill
        agent = make_agent(cuda)                         # (a step moves the temperature and the optimizers too)
        agent.actor.head.noise_override = list(eps)
        stats = agent._step_body(batch, True, False)
        return {k: float(v) for k, v in stats.items()}, agent._flat["critic"].grad.clone(), agent._flat["actor"].grad.clone()

    want = run(0.25)
    assert all(np.isfinite(v) for v in want[0].values())
    for fill in (float("nan"), float("inf")):
        stats, critic, actor = run(fill)
        assert stats == pytest.approx(want[0], rel=1e-5), fill
        for a, b in ((critic, want[1]), (actor, want[2])):
            assert float((a - b).norm() / b.norm()) < GRAD_TOL, fill


class _Flat:
    """A pre-processor that leaves a pending augmentation: every cloud's coordinates times 0."""

    def __init__(self):
        self.shapes = []

    def __call__(self, data):
        from pointcloud_rl_amd.networks.pointnet import AugmentedObs, batch_rows
        out = AugmentedObs(data["obs"])
        out.aug = dict(affine=torch.zeros(batch_rows(out), 3, 4, device=out["xyz"].device))
        self.shapes.append(tuple(out["xyz"].shape))
        return dict(data, obs=out)


@pytest.mark.gpu
def test_a_pre_processors_augmentation_reaches_the_encoder(cuda):
    """Its draws are made for the target's rows too, and what it leaves pending is applied: with every coordinate taken to 0 the update does not
    depend on the coordinates."""
    from pointcloud_rl_amd.replay import DeviceReplay

    def update(scale, flat):
        agent = make_agent(cuda)
        if flat is not None:
            from pointcloud_rl_amd.augmentations import build_data_augmentations
            agent.obs_processor = build_data_augmentations([flat])
        mem = DeviceReplay(64, device=cuda, sampling_cfg=dict(type="TStepTransition", horizon=4, seed=5))
        g = np.random.RandomState(5)
        obs = lambda: {"xyz": (scale * g.randn(20, 3, 64)).astype(np.float32), "rgb": g.randint(0, 256, (20, 3, 64)).astype(np.uint8)}
        mem.push_batch(dict(obs=obs(), next_obs=obs(), actions=g.uniform(-1, 1, (20, 4)).astype(np.float32), rewards=g.randn(20, 1).astype(np.float32),
                            dones=np.zeros((20, 1), bool), episode_dones=np.zeros((20, 1), bool)))
        noise = torch.Generator().manual_seed(9)
        agent.actor.head.noise_override = [torch.randn(3, 5, 4, generator=noise).to(cuda)]
        return agent.update_parameters(mem, 1)["sac/critic_loss"]

    flat = _Flat()
    assert update(1.0, flat) == update(2.0, flat)
    assert update(1.0, None) != update(2.0, None)
    assert flat.shapes == [(3, 4, 3, 64), (3, 5, 3, 64)] * 2


def test_observations_are_augmented_behind_the_history():
    from pointcloud_rl_amd.methods.recurrent import with_target_history
    from pointcloud_rl_amd.networks.pointnet import AugmentedObs
    batch = make_batch("cpu", [3, 2], 3)
    batch["next_obs"] = AugmentedObs(batch["next_obs"])
    with_target_history(batch)                           # nothing pending
    batch["next_obs"].aug = dict(affine=torch.zeros(6, 3, 4))
    with pytest.raises(ValueError, match="augmented"):
        with_target_history(batch)


def test_single_transitions_have_no_run():
    from pointcloud_rl_amd.methods.recurrent import with_target_history
    with pytest.raises(ValueError, match="TStepTransition"):
        with_target_history(dict(rewards=torch.zeros(4, 1), episode_dones=torch.zeros(4, 1)))
