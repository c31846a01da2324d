"""Sequence operators on libpcrl_hip.so: what a recurrent core is made of, and dropout.

    short_conv / short_conv_step    causal convolution over time, one short filter per channel, optional SiLU
    ssm_scan / ssm_step             selective state space scan, gated
    dropout                         counter-based, the mask is never stored

The whole-sequence forms are differentiable in every floating-point input (the incoming state and the outgoing one included); the step forms
are for acting.  Activations are float32, bfloat16 or float16, [B, T, D] with adjacent channels and any strides for batch and time (other layouts
are copied); parameters, the scan's state and every sum are float32.  Everything runs on the current stream of the tensors' device, allocates
from torch's caching allocator and reads nothing on the host, so calls can be captured in a hipGraph.  There is no CPU path.
Arguments that do not fit raise ValueError, a failing launch RuntimeError; the gradients are not differentiable again, and a dual tensor
(forward-mode derivatives) raises NotImplementedError.

starts [B, T] (bool): step t is the first of a new sequence -- what came before, the incoming state included, does not reach it.
lengths [B] (integers): row b has lengths[b] steps; outputs and gradients behind them are 0, inputs behind them are not looked at, and the
last state is the one after step lengths[b] - 1.
"""
import torch

from . import hip
from ._lib import sequence_ext

_ext = None


def _call(name, *args):
    global _ext
    if _ext is None:
        _ext = sequence_ext()
    if hip.TIMER is None:
        return getattr(_ext, name)(*args)
    with hip._span(name):
        return getattr(_ext, name)(*args)


def short_conv(x, weight, bias=None, state=None, starts=None, lengths=None, activation="silu"):
    """y[b, t, d] = act(bias[d] + sum_k weight[d, k] x[b, t - (W - 1) + k, d]) with W = 1 ... 4 taps; act is SiLU or nothing.

    x [B, T, D]; weight [D, W], bias [D] float32; state [B, W - 1, D] of x's type: the inputs in front of this call, oldest first (default:
    zeros); starts, lengths: see the module.  Returns (y [B, T, D], last_state [B, W - 1, D]); differentiable in x, weight, bias and state."""
    return _call("short_conv", x, weight, bias, state, starts, lengths, activation)


def short_conv_step(x, state, weight, bias=None, starts=None, activation="silu", state_out=None):
    """One step of `short_conv`: x [B, D], state [B, W - 1, D] -> y [B, D].  The state is updated in place, or written to `state_out` (which must
    not overlap it); starts [B]: rows whose sequence begins here.  Not differentiable."""
    return _call("short_conv_step", x, state, weight, bias, starts, activation, state_out)


def ssm_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, starts=None, lengths=None):
    """Selective state space scan over a sequence, for every channel d and its states n:

        s_t = softplus(dt_t + dt_bias)  (softplus=False: dt_t + dt_bias)
        h_t[n] = exp(s_t A[d, n]) h_{t-1}[n] + s_t B_t[n] u_t,     y_t = (sum_n C_t[n] h_t[n] + D u_t) * silu(z_t)

    u, dt, z [B, T, D]; B, C [B, T, N] or [B, T, G, N] (G groups share the channels in order, evenly); A [D, N] with 1 to 32 states, D [D],
    dt_bias [D], state [B, D, N] (default: zeros) float32; starts, lengths: see the module.  Returns (y [B, T, D], last_state [B, D, N]);
    differentiable in all of them.  A call that will be differentiated keeps the state in front of every 16th step (N / 4 bytes an element)."""
    return _call("ssm_scan", u, dt, A, B, C, D, z, dt_bias, bool(softplus), state, starts, lengths)


def ssm_step(u, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus=True, starts=None, state_out=None):
    """One step of `ssm_scan`: u, dt, z [B, D], B, C [B, N] or [B, G, N], state [B, D, N] float32 -> y [B, D].  The state is updated in place, or
    written to `state_out` (which must not overlap it); starts [B]: rows whose sequence begins here.  Not differentiable."""
    return _call("ssm_step", u, dt, A, B, C, state, D, z, dt_bias, bool(softplus), starts, state_out)


def dropout(x, p, seed, offset=0, residual=None):
    """x with each element dropped (set to 0, whatever it holds) with probability p and the kept ones scaled by 1 / (1 - p), plus `residual`.

    p is taken in steps of 2^-16 (round(65536 p) / 65536, for the scale too).  Which elements go is a function of (seed, offset, position in x)
    alone: Philox4x32-10 keyed by `seed`, one 16-bit draw per element, so the backward draws the same mask again and nothing is stored.  offset:
    an integer, or a device int64 tensor of one element that is read when the kernel runs (a captured graph draws a new mask on every replay when
    the tensor is advanced in between); it must keep its value until the backward has run."""
    at = offset if torch.is_tensor(offset) else None
    return _call("dropout", x, p, int(seed) & 0xFFFFFFFFFFFFFFFF, 0 if at is not None else int(offset) & 0xFFFFFFFFFFFFFFFF, at, residual)
