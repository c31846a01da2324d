"""SelectiveSSM: the recurrent core (`rnn_cfg`) of a Visuomotor, and Dropout, both on the sequence operators (sequence.py).

The reference carries the plumbing of a recurrent backbone (pyrl/networks/backbones/visuomotor.py:95-125: rnn_states, episode_dones, is_valid,
rnn_mode) and ships no module for it; parameter names here are this package's own."""
import math

import torch
import torch.nn as nn
import torch.nn.functional as F

from .. import sequence
from ..utils.torch_utils import ExtendedModule
from .builder import NETWORK


class Dropout(ExtendedModule):
    """Counter-based dropout (sequence.dropout) with an optional residual, active in training mode.

    The seed is drawn from torch's generator when the module is made; the count of calls is the generator's offset and lives in device memory,
    advanced by the call itself, so a captured step draws a new mask on every replay.  Neither is part of the state_dict; checkpoints
    (utils/checkpoint.py) keep both, so a resumed run draws the masks that the run would have drawn.

    A call inside a backward pass -- activation checkpointing, which evaluates a module a second time there -- is refused: it would draw the next
    mask, not the one of the forward pass.  There, call sequence.dropout with an offset of your own."""

    def __init__(self, p):
        super().__init__()
        if not 0.0 <= float(p) < 1.0:
            raise ValueError(f"dropout probability {p}: 0 <= p < 1")
        self.p = float(p)
        self.reseed()
        self.register_buffer("calls", torch.zeros(1, dtype=torch.int64), persistent=False)

    def reseed(self):
        """Masks independent of every other module's from here on: a copied module otherwise draws its original's."""
        self.seed = int(torch.randint(0, 2 ** 62, (1,)).item())

    def forward(self, x, residual=None):
        if not self.training or self.p == 0.0:
            return x if residual is None else x + residual
        if torch._C._current_graph_task_id() != -1:
            raise RuntimeError("Dropout is evaluated again inside a backward pass (activation checkpointing): its mask would not be the forward's; "
                               "checkpoint a part without it, or call sequence.dropout with an offset of your own")
        self.calls.add_(1)
        if residual is None or residual.dtype == x.dtype:
            return sequence.dropout(x, self.p, self.seed, self.calls.clone(), residual=residual)
        return residual + sequence.dropout(x, self.p, self.seed, self.calls.clone())         # the wider type, as without dropout

    def checkpoint_state(self):
        """What a checkpoint keeps beside the state_dict's entries."""
        return dict(seed=torch.tensor([self.seed]), calls=self.calls.detach())

    def _load_from_state_dict(self, state_dict, prefix, *args):
        seed, calls = state_dict.pop(prefix + "seed", None), state_dict.pop(prefix + "calls", None)
        if seed is not None and calls is not None:              # (a file without them leaves the module its own masks)
            self.seed = int(seed)
            with torch.no_grad():
                self.calls.copy_(calls)
        super()._load_from_state_dict(state_dict, prefix, *args)

    def extra_repr(self):
        return f"p={self.p}"


@NETWORK.register_module()
class SelectiveSSM(ExtendedModule):
    """x + dropout(out(core(norm(x)))), core = gated selective scan behind a short causal convolution.

        [v, z] = in(norm(x));  v = silu(conv(v));  [dt, B, C] = proj(v);  y = scan(v, dt_proj(dt), A, B, C, D, z)

    feat_dim: width of x and of the result; expand: inner width / feat_dim; state_dim: states per inner channel (1 to 32); conv_width: taps (2 to 4);
    dt_rank: width of the step size's bottleneck ("auto": feat_dim / 16); groups: channel groups with a B and C of their own.

    forward(x, states, starts, lengths) -> (y, states).  x [B, T, feat_dim]: a run of steps, differentiable in x and in the states it starts from;
    x [B, feat_dim]: one step (acting), without gradients and without dropout.  states: dict(conv [B, conv_width - 1, inner], ssm [B, inner,
    state_dim]) or None (zeros); the returned ones follow the last step.  starts [B, T] / [B]: steps that begin a new episode; lengths [B].

    The operators run in the type of the projections (float32, or 16 bits under autocast or with 16-bit weights: so does the convolution's state),
    with their parameters and the scan's state in float32."""

    def __init__(self, feat_dim, expand=2, state_dim=16, conv_width=4, dt_rank="auto", groups=1, dropout=0.0, dt_range=(1e-3, 1e-1), **kwargs):
        super().__init__()
        self.feat_dim, self.inner, self.state_dim, self.groups = int(feat_dim), int(round(feat_dim * expand)), int(state_dim), int(groups)
        if not 1 <= self.state_dim <= 32 or not 2 <= conv_width <= 4 or self.inner % self.groups:
            raise ValueError(f"state_dim {state_dim} (1 to 32), conv_width {conv_width} (2 to 4), {self.inner} channels in {groups} groups")
        self.dt_rank = max(1, math.ceil(feat_dim / 16)) if dt_rank == "auto" else int(dt_rank)
        self.is_recurrent = True
        self.norm = nn.LayerNorm(self.feat_dim)
        self.in_proj = nn.Linear(self.feat_dim, 2 * self.inner, bias=False)
        bound = 1.0 / math.sqrt(conv_width)
        self.conv_weight = nn.Parameter(torch.empty(self.inner, conv_width).uniform_(-bound, bound))
        self.conv_bias = nn.Parameter(torch.zeros(self.inner))
        self.x_proj = nn.Linear(self.inner, self.dt_rank + 2 * self.groups * self.state_dim, bias=False)
        self.dt_proj = nn.Linear(self.dt_rank, self.inner)          # its bias is added inside the scan (dt_bias)
        step = torch.exp(torch.rand(self.inner) * math.log(dt_range[1] / dt_range[0]) + math.log(dt_range[0]))
        with torch.no_grad():
            self.dt_proj.bias.copy_(step + torch.log(-torch.expm1(-step)))           # softplus(bias) = step
        self.A_log = nn.Parameter(torch.log(torch.arange(1, self.state_dim + 1, dtype=torch.float32)).repeat(self.inner, 1))
        self.D = nn.Parameter(torch.ones(self.inner))
        self.out_proj = nn.Linear(self.inner, self.feat_dim, bias=False)
        self.dropout = Dropout(dropout) if dropout else None

    def init_states(self, batch_size, device=None, dtype=torch.float32):
        device = self.D.device if device is None else device
        return dict(conv=torch.zeros(batch_size, self.conv_weight.shape[1] - 1, self.inner, dtype=dtype, device=device),
                    ssm=torch.zeros(batch_size, self.inner, self.state_dim, dtype=torch.float32, device=device))

    def _scan_inputs(self, v):
        """dt before its bias, B, C of the convolved inputs v [..., inner]."""
        dt, B, C = self.x_proj(v).split([self.dt_rank, self.groups * self.state_dim, self.groups * self.state_dim], dim=-1)
        shape = v.shape[:-1] + (self.groups, self.state_dim)
        return F.linear(dt, self.dt_proj.weight), B.reshape(shape), C.reshape(shape)

    def _scan_parameters(self):
        return dict(A=-torch.exp(self.A_log.float()), D=self.D.float(), dt_bias=self.dt_proj.bias.float())

    def forward(self, x, states=None, starts=None, lengths=None):
        if x.ndim == 2:
            return self.step(x, states, starts)
        v, z = self.in_proj(self.norm(x)).chunk(2, dim=-1)
        conv, ssm = (None, None) if states is None else (states["conv"].to(v.dtype), states["ssm"])
        v, conv = sequence.short_conv(v, self.conv_weight.float(), self.conv_bias.float(), state=conv, starts=starts, lengths=lengths)
        dt, B, C = self._scan_inputs(v)
        y, ssm = sequence.ssm_scan(v, dt, B=B, C=C, z=z, state=ssm, starts=starts, lengths=lengths, **self._scan_parameters())
        y = self.out_proj(y)
        return (x + y if self.dropout is None else self.dropout(y, residual=x)), dict(conv=conv, ssm=ssm)

    @torch.no_grad()
    def step(self, x, states=None, starts=None):
        """One step for a batch of environments: x [B, feat_dim], starts [B] -> (y, new states); the given states are left as they are."""
        v, z = self.in_proj(self.norm(x)).chunk(2, dim=-1)
        states = self.init_states(x.shape[0], x.device, v.dtype) if states is None else dict(states, conv=states["conv"].to(v.dtype))
        conv, ssm = torch.empty_like(states["conv"]), torch.empty_like(states["ssm"])
        v = sequence.short_conv_step(v, states["conv"], self.conv_weight.float(), self.conv_bias.float(), starts=starts, state_out=conv)
        dt, B, C = self._scan_inputs(v)
        y = sequence.ssm_step(v, dt, B=B, C=C, state=states["ssm"], z=z, starts=starts, state_out=ssm, **self._scan_parameters())
        return x + self.out_proj(y), dict(conv=conv, ssm=ssm)
