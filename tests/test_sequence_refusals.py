"""Calls that the sequence operators and the modules made of them cannot answer: refused, not answered wrongly."""
import pytest
import torch


def _zeros(*s):
    return torch.zeros(*s)


CALLS = {
    "short_conv": dict(x=_zeros(1, 2, 8), weight=_zeros(8, 4), bias=_zeros(8), state=_zeros(1, 3, 8)),
    "short_conv_step": dict(x=_zeros(1, 8), state=_zeros(1, 3, 8), weight=_zeros(8, 4), bias=_zeros(8)),
    "ssm_scan": dict(u=_zeros(1, 2, 8), dt=_zeros(1, 2, 8), A=_zeros(8, 4), B=_zeros(1, 2, 4), C=_zeros(1, 2, 4), D=_zeros(8), z=_zeros(1, 2, 8),
                     dt_bias=_zeros(8), state=_zeros(1, 8, 4)),
    "ssm_step": dict(u=_zeros(1, 8), dt=_zeros(1, 8), A=_zeros(8, 4), B=_zeros(1, 4), C=_zeros(1, 4), state=_zeros(1, 8, 4), D=_zeros(8), z=_zeros(1, 8),
                     dt_bias=_zeros(8)),
    "dropout": dict(x=_zeros(4), residual=_zeros(4), p=0.5, seed=1),
}


@pytest.mark.parametrize("name,arg", [(n, a) for n, kw in CALLS.items() for a, v in kw.items() if torch.is_tensor(v)])
def test_forward_mode_derivatives_are_refused(name, arg):
    """A dual tensor in any place: the result would have no tangent.  (Without one the call gets as far as wanting a GPU.)"""
    import torch.autograd.forward_ad as fwd
    from pointcloud_rl_amd import sequence
    kw = CALLS[name]
    with pytest.raises(RuntimeError, match="no CPU path"):
        getattr(sequence, name)(**kw)
    with fwd.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            getattr(sequence, name)(**dict(kw, **{arg: fwd.make_dual(kw[arg], torch.ones_like(kw[arg]))}))
        with pytest.raises(RuntimeError, match="no CPU path"):
            getattr(sequence, name)(**kw)


def _checkpointed(x, module, reentrant):
    from torch.utils.checkpoint import checkpoint
    checkpoint(module, x, use_reentrant=reentrant).sum().backward()


@pytest.mark.parametrize("reentrant", [False, True])
def test_dropout_is_not_evaluated_again_in_a_backward_pass(monkeypatch, reentrant):
    """Activation checkpointing would multiply the gradient with another mask than the forward's.  (The kernel is replaced: what is tested is
    which calls reach it.)"""
    from pointcloud_rl_amd.networks import Dropout, ssm
    offsets = []
    monkeypatch.setattr(ssm.sequence, "dropout", lambda x, p, seed, offset, residual=None: offsets.append(int(offset)) or x * x)
    drop, x = Dropout(0.5), torch.ones(4, requires_grad=True)
    with pytest.raises(RuntimeError, match="activation checkpointing"):
        _checkpointed(x, drop, reentrant)
    assert offsets == [1] and int(drop.calls) == 1
    _checkpointed(x, drop.eval(), reentrant)             # nothing is drawn: fine
    drop.train()(x).sum().backward()                     # an ordinary pass goes on
    assert offsets == [1, 2]


@pytest.mark.gpu
@pytest.mark.parametrize("reentrant", [False, True])
def test_dropout_under_activation_checkpointing(cuda, reentrant):
    """The module refuses; the operator with an offset that the caller holds draws the forward's mask again."""
    from pointcloud_rl_amd import sequence
    from pointcloud_rl_amd.networks import Dropout
    x = torch.randn(64, 33, device=cuda, requires_grad=True)
    with pytest.raises(RuntimeError, match="activation checkpointing"):
        _checkpointed(x, Dropout(0.5).to(cuda), reentrant)
    x.grad = None
    _checkpointed(x, lambda t: sequence.dropout(t, 0.5, 7, 3), reentrant)
    want, = torch.autograd.grad(sequence.dropout(x, 0.5, 7, 3).sum(), x)
    assert torch.equal(x.grad, want)


def test_a_recurrent_critic_without_a_recurrent_actor_is_refused():
    """Such an agent counted as not recurrent: its step took the critic's core for absent."""
    import copy
    from pointcloud_rl_amd import configs
    from pointcloud_rl_amd.methods import build_agent
    cfg = configs.recurrent(configs.sac_dmc(6, 4, 6, head_hidden=64), state_dim=8)
    cfg["env_params"] = configs.env_params({"xyz": [3, 64], "rgb": [3, 64]}, 4)
    assert build_agent(copy.deepcopy(cfg)).is_recurrent
    cfg["critic_cfg"]["nn_cfg"]["rnn_cfg"] = cfg["actor_cfg"]["nn_cfg"].pop("rnn_cfg")
    with pytest.raises(ValueError, match="rnn_cfg"):
        build_agent(cfg)


def test_states_that_overlap_are_refused_at_the_c_entry_points():
    """A last state in the memory of the incoming one: chunks of the scan and runs of the convolution would read what others have written.  Nothing
    is dereferenced: the calls that are not refused here fail on a later check (no scratch, a null output)."""
    import ctypes
    from pointcloud_rl_amd import _lib
    from test_sequence_gpu import ConvDesc, SsmDesc
    lib = _lib.lib()
    at = lambda v: ctypes.c_void_p(v)
    y, none, base = at(1 << 40), ctypes.c_size_t(0), 1 << 20

    def scan(last, T=64):
        d = SsmDesc(B=2, T=T, D=8, N=4, G=1, u=4096, dt=4096, Bm=4096, Cm=4096, A=4096, state=base)
        return lib.pcrl_ssm_scan_fwd(ctypes.byref(d), y, at(last), None, None, none, None)

    size = 4 * 2 * 8 * 4
    for last in (base, base + 4, base - 4, base + size - 4, base - size + 4):
        assert scan(last) == -1 and b"overlaps" in lib.pcrl_last_error(), last
    for last in (base + size, base - size):
        assert scan(last) == -2 and b"workspace" in lib.pcrl_last_error(), last      # 64 steps of one block: chunks, which need scratch
    for T, last in ((2, base), (2, base + 4), (1, base + 4), (1, base - 2 * 3 * 8 * 4 + 4)):
        d = ConvDesc(B=2, T=T, D=8, W=4, x=4096, weight=4096, state=base)
        assert lib.pcrl_short_conv_fwd(ctypes.byref(d), y, at(last), None) == -1 and b"overlaps" in lib.pcrl_last_error(), (T, last)
    for out in (base + 4, base - size + 4):
        d = SsmDesc(B=2, T=1, D=8, N=4, G=1, u=4096, dt=4096, Bm=4096, Cm=4096, A=4096, state=base)
        assert lib.pcrl_ssm_step(ctypes.byref(d), y, at(out), None) == -1 and b"overlaps" in lib.pcrl_last_error(), out
