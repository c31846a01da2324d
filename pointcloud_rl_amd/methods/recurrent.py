"""SAC update on runs of consecutive transitions ([B, H, ...] batches of a T-step replay) for an agent with a recurrent core.

The loss of sac.py:125-195 with the mean over the valid steps of every run (`is_valid`; the padding of short episodes takes no part), networks
evaluated over whole runs from a zero state, the state restarted behind `episode_dones`.  Eager: autograd through the sequence operators."""
import torch


def _kwargs(batch, prefix=""):
    return dict(episode_dones=batch[prefix + "episode_dones"], is_valid=batch.get(prefix + "is_valid"))


def _check_runs(batch):
    if batch["rewards"].ndim != 3:
        raise ValueError(f"a recurrent agent is updated on [B, H, ...] batches (DeviceReplay with sampling_cfg=dict(type='TStepTransition', "
                         f"horizon=...)); rewards are {tuple(batch['rewards'].shape)}")


def _blank(batch, padding):
    """The batch with 0 in every floating-point tensor where padding [B, H] says so."""
    def blank(v):
        if isinstance(v, dict):
            return {k: blank(x) for k, x in v.items()}
        if not torch.is_tensor(v) or not v.is_floating_point() or v.shape[:2] != padding.shape:
            return v
        return v.masked_fill(padding.reshape(padding.shape + (1,) * (v.ndim - 2)), 0.0)
    return {k: blank(v) for k, v in batch.items()}


def with_target_history(batch):
    """The batch with `next_obs` as the runs that the target's networks have to see.

    What stands behind step t has the history obs[s], next_obs[s], ..., next_obs[t], with s the first step of t's episode in the run: the states
    that the online networks reach one step later, and the policy when it acts.  Over next_obs alone the first observation of every episode
    would be missing.  So each episode's first observation is put in front of its next ones: next_obs becomes [B, H + E, ...] (E: the most
    episodes of a run), with next_episode_dones and next_is_valid to go with it, and next_at [B, H] says where next_obs[t] has gone."""
    _check_runs(batch)
    if any(getattr(batch[k], "aug", None) or getattr(batch[k], "repeat", 1) not in (None, 1) for k in ("obs", "next_obs")):
        raise ValueError("observations are augmented behind with_target_history: its rows are not the ones that the draws were made for")
    B, H = batch["rewards"].shape[:2]
    ended = batch["episode_dones"].reshape(B, H).bool()
    valid = torch.ones_like(ended) if batch.get("is_valid") is None else batch["is_valid"].reshape(B, H).bool()
    starts = valid.clone()
    starts[:, 1:] &= ended[:, :-1]
    begun = starts.cumsum(1)                                   # episodes of the run up to and including step t's
    episodes, whole = torch.stack((begun[:, -1].max(), valid.all().to(begun.dtype))).tolist()
    if not whole:
        batch = _blank(batch, ~valid)
    width, steps = H + episodes, torch.arange(H, device=ended.device).expand(B, H)
    at = steps + begun
    if episodes == 1:
        pick = lambda first, rest: torch.cat((first[:, :1], rest), dim=1)
    else:
        # row numbers of (obs, next_obs) side by side; what is no start goes to a last place that is cut off
        source = steps.new_zeros(B, width + 1).scatter_(1, at, H + steps).scatter_(1, torch.where(starts, at - 1, width), steps)[:, :width]
        rows = torch.arange(B, device=ended.device)[:, None]
        pick = lambda first, rest: torch.cat((first, rest), dim=1)[rows, source]
    length = valid.sum(1, keepdim=True) + begun[:, -1:]
    return dict(batch, next_obs={k: pick(batch["obs"][k], v) for k, v in batch["next_obs"].items()}, next_at=at[..., None],
                next_episode_dones=torch.zeros(B, width, dtype=torch.bool, device=ended.device).scatter_(1, at, ended & valid)[..., None],
                next_is_valid=(torch.arange(width, device=ended.device) < length)[..., None])


def _mean(x, weight):
    """Mean of x [B, H, 1] over the valid steps."""
    return (x * weight).sum() / weight.sum()


def _q_values(agent, critic, obs, actions, kw, feature=None):
    """Q of every head [B, H, heads].  A shared backbone (encoder and recurrent core) is evaluated once, not once per head."""
    if not agent._dedup:
        return critic(obs, actions, **kw)
    qs = []
    for value in critic.values:
        qs.append(value(obs, actions, save_feature=feature is None, **(dict(feature=feature) if feature is not None else {}), **kw))
        if feature is None:
            feature = value.backbone.pop_attr("saved_feature")
    return torch.cat(qs, dim=-1)


def recurrent_step(agent, batch, do_actor, polyak):
    """One critic (and actor, temperature) step; returns the metrics of SAC._step_body.  A batch without `next_at` (with_target_history) has
    its target formed over next_obs as it stands."""
    _check_runs(batch)
    kw, rewards = _kwargs(batch), batch["rewards"]
    at = batch.get("next_at")
    next_kw = kw if at is None else _kwargs(batch, "next_")
    weight = torch.ones_like(rewards) if kw["is_valid"] is None else kw["is_valid"].to(rewards.dtype)
    stats = {}
    with torch.no_grad():
        next_actions, neg_logp = agent.actor(batch["next_obs"], mode="max-entropy", save_feature=agent._dedup, **next_kw)
        q_next = _q_values(agent, agent.target_critic, batch["next_obs"], next_actions, next_kw, agent.actor.backbone.pop_attr("saved_feature"))
        min_q = q_next.min(dim=-1, keepdim=True).values + agent._alpha_t * neg_logp
        min_q = min_q if at is None else min_q.gather(1, at)
        r = rewards * agent.reward_scale
        y = r + agent.gamma * min_q if agent.ignore_dones else r + (1 - batch["dones"].float()) * agent.gamma * min_q
    fb = agent._flat["critic"]
    q = _q_values(agent, agent.critic, batch["obs"], batch["actions"], kw)
    critic_loss = _mean((q - y).square().sum(-1, keepdim=True), weight)
    fb.zero_grad()
    critic_loss.backward()
    grad_norm = agent._optim_step("critic", agent._allreduce(fb.grad), polyak=polyak)
    with torch.no_grad():
        stats["critic_loss"] = critic_loss.detach()
        stats["max_critic_abs_err"] = ((q - y).abs() * weight).max()
        stats["q"] = _mean(q.min(dim=-1, keepdim=True).values, weight)
        stats["q_target"] = _mean(y, weight)
        stats["critic_grad"] = grad_norm
    if do_actor:
        _actor_step(agent, batch["obs"], kw, weight, stats)
    return stats


def _actor_step(agent, obs, kw, weight, stats):
    fb = agent._flat["actor"]
    pi, neg_logp = agent.actor(obs, mode="max-entropy", save_feature=agent.shared_backbone, detach_visual=agent.detach_actor_feature, **kw)[:2]
    feature = agent.actor.backbone.pop_attr("saved_feature")
    entropy = _mean(neg_logp, weight)
    # only d(q)/d(pi) is needed from the Q heads; with a shared backbone they start from the actor's own feature
    params = [p for p in agent.critic.parameters() if p.requires_grad]
    for p in params:
        p.requires_grad_(False)
    try:
        q_pi = _q_values(agent, agent.critic, obs, pi, kw, feature.detach() if feature is not None and agent._dedup else None)
    finally:
        for p in params:
            p.requires_grad_(True)
    actor_loss = -(_mean(q_pi.min(dim=-1, keepdim=True).values, weight) + agent._alpha_t * entropy)
    fb.zero_grad()
    actor_loss.backward()
    stats["actor_grad"] = agent._optim_step("actor", agent._allreduce(fb.grad))
    stats["actor_loss"], stats["entropy"] = actor_loss.detach(), entropy.detach()
    if agent.automatic_alpha_tuning:
        alpha_loss = agent.log_alpha.exp() * (entropy - agent.target_entropy).detach()
        agent._flat["alpha"].zero_grad()
        alpha_loss.backward()
        agent._optim_step("alpha", agent._allreduce(agent._flat["alpha"].grad) if agent.sync_alpha else 1.0)
        agent._alpha_t.copy_(agent.log_alpha.detach().exp())
        stats["alpha_loss"] = alpha_loss.detach().reshape(())
    else:
        stats["alpha_loss"] = torch.zeros((), device=agent.device)
    stats["new_alpha"] = agent._alpha_t.reshape(()).clone()
