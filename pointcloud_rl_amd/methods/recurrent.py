"""SAC update on runs of consecutive transitions ([B, H, ...] batches of a T-step replay) for an agent with a recurrent core.

The loss of sac.py:125-195 with the mean over the valid steps of every run (`is_valid`; the padding of short episodes takes no part), networks
evaluated over whole runs from a zero state, the state restarted behind `episode_dones`.  Eager: autograd through the sequence operators."""
import torch


def _kwargs(batch):
    return dict(episode_dones=batch["episode_dones"], is_valid=batch.get("is_valid"))


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
    """One critic (and actor, temperature) step; returns the metrics of SAC._step_body."""
    kw = _kwargs(batch)
    rewards = batch["rewards"]
    if rewards.ndim != 3:
        raise ValueError(f"a recurrent agent is updated on [B, H, ...] batches (DeviceReplay with sampling_cfg=dict(type='TStepTransition', "
                         f"horizon=...)); rewards are {tuple(rewards.shape)}")
    weight = torch.ones_like(rewards) if kw["is_valid"] is None else kw["is_valid"].to(rewards.dtype)
    stats = {}
    with torch.no_grad():
        next_actions, neg_logp = agent.actor(batch["next_obs"], mode="max-entropy", save_feature=agent._dedup, **kw)
        q_next = _q_values(agent, agent.target_critic, batch["next_obs"], next_actions, kw, agent.actor.backbone.pop_attr("saved_feature"))
        min_q = q_next.min(dim=-1, keepdim=True).values + agent._alpha_t * neg_logp
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
