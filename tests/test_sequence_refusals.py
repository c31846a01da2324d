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
