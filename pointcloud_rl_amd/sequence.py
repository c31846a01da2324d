"""Sequence operators on libpcrl_hip.so: what a recurrent core is made of, and dropout.

    short_conv / short_conv_step    causal convolution over time, one short filter per channel, optional SiLU
    ssm_scan / ssm_step             selective state space scan, gated
    dropout                         counter-based, the mask is never stored

The whole-sequence forms are differentiable in every floating-point input (the incoming state and the outgoing one included); the step forms
are for acting.  Activations are float32, bfloat16 or float16, [B, T, D] with adjacent channels and any strides for batch and time (other layouts
are copied); parameters, the scan's state and every sum are float32.  Everything runs on the current stream of the tensors' device, allocates
from torch's caching allocator and reads nothing on the host, so calls can be captured in a hipGraph.  There is no CPU path.

starts [B, T] (bool): step t is the first of a new sequence -- what came before, the incoming state included, does not reach it.
lengths [B] (integers): row b has lengths[b] steps; outputs and gradients behind them are 0, inputs behind them are not looked at, and the
last state is the one after step lengths[b] - 1.
"""
import ctypes
from ctypes import byref

import torch

from . import _lib, hip
from ._lib import ConvDesc, SsmDesc, SsmGrads, check, lib

_DTYPES = {torch.float32: _lib.DT_F32, torch.bfloat16: _lib.DT_BF16, torch.float16: _lib.DT_F16}
_getDevice, _getStream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream
_empty_like = torch.empty_like


def _on_gpu(t):
    if not t.is_cuda:
        raise RuntimeError(f"the sequence operators run on the MI355X (got a tensor on {t.device}); there is no CPU path")


def _launch(name, device, fn, *args):
    """fn(*args, stream) on `device` (an index) and torch's current stream there."""
    if hip.TIMER is None and device == _getDevice():
        check(fn(*args, _getStream(device)))
    else:
        with torch.cuda.device(device), hip._span(name):
            check(fn(*args, _getStream(device)))


def _at(t):
    return t.data_ptr() if t is not None else None


def _activation(name, t, shape, like):
    """t checked against a shape and against the type and device of `like`; its channels made adjacent."""
    if t.shape != shape:
        raise ValueError(f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, the sequence is {like.dtype} on {like.device}")
    return t if t.stride(-1) == 1 else t.contiguous()


def _parameter(name, t, shape, like):
    if t.shape != shape:
        raise ValueError(f"{name} is {tuple(t.shape)}, expected {tuple(shape)}")
    if t.dtype != torch.float32 or t.device != like.device:
        raise ValueError(f"{name} is {t.dtype} on {t.device}, expected float32 on {like.device}")
    return t if t.is_contiguous() else t.contiguous()


def _sequence_dtype(t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"activations are float32, bfloat16 or float16, not {t.dtype}")
    return code


def _marks(starts, lengths, rows, like):
    """starts as contiguous bytes, lengths as int32, on the device of the sequence."""
    if starts is not None:
        if starts.shape != rows or starts.dtype not in (torch.bool, torch.uint8) or starts.device != like.device:
            raise ValueError(f"starts is {starts.dtype} {tuple(starts.shape)} on {starts.device}, expected bool {tuple(rows)} on {like.device}")
        if not starts.is_contiguous():
            starts = starts.contiguous()
    if lengths is not None:
        if lengths.shape != rows[:1] or lengths.dtype not in (torch.int32, torch.int64) or lengths.device != like.device:
            raise ValueError(f"lengths is {lengths.dtype} {tuple(lengths.shape)} on {lengths.device}, expected int32 {tuple(rows[:1])} on {like.device}")
        if lengths.dtype != torch.int32 or not lengths.is_contiguous():
            lengths = lengths.to(torch.int32).contiguous()
    return starts, lengths


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ---- short causal convolution ----------------------------------------------------------------------------------------------------------------
def _conv_desc(x, weight, bias, state, starts, lengths, silu, T):
    step = x.dim() == 2
    return ConvDesc(x.shape[0], T, x.shape[-1], weight.shape[1], _DTYPES[x.dtype], silu, x.data_ptr(), x.stride(0), 0 if step else x.stride(1),
                    weight.data_ptr(), _at(bias), _at(state), _at(starts), T, _at(lengths))


def _conv_checked(x, weight, bias, state, starts, lengths, activation, dims):
    if x.dim() != dims:
        raise ValueError(f"x is {tuple(x.shape)}, expected {'[B, D]' if dims == 2 else '[B, T, D]'}")
    _sequence_dtype(x)
    if activation not in (None, "silu"):
        raise ValueError(f"activation {activation!r}: None or 'silu'")
    D = x.shape[-1]
    if weight.dim() != 2 or not 1 <= weight.shape[1] <= 4:
        raise ValueError(f"weight is {tuple(weight.shape)}, expected [{D}, W] with 1 to 4 taps")
    x = x if x.stride(-1) == 1 else x.contiguous()
    weight = _parameter("weight", weight, (D, weight.shape[1]), x)
    bias = _parameter("bias", bias, (D,), x) if bias is not None else None
    if state is not None:
        state = _activation("state", state, (x.shape[0], weight.shape[1] - 1, D), x)
        if dims == 3 and not state.is_contiguous():
            state = state.contiguous()
    starts, lengths = _marks(starts, lengths, x.shape[:-1], x)
    return x, weight, bias, state, starts, lengths, int(activation == "silu")


def _conv_forward(x, weight, bias, state, starts, lengths, silu):
    B, T, D = x.shape
    y = torch.empty((B, T, D), dtype=x.dtype, device=x.device)
    last = torch.empty((B, weight.shape[1] - 1, D), dtype=x.dtype, device=x.device)
    if y.numel():
        desc = _conv_desc(x, weight, bias, state, starts, lengths, silu, T)
        _launch("short_conv_fwd", x.device.index, lib().pcrl_short_conv_fwd, byref(desc), y.data_ptr(), last.data_ptr())
    elif state is not None:
        last.copy_(state)
    else:
        last.zero_()
    return y, last


class _ShortConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, starts, lengths, silu):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, weight, bias, state, starts, lengths)
        ctx.silu = silu
        return _conv_forward(x, weight, bias, state, starts, lengths, silu)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        if dy is None and dlast is None:
            return (None,) * 7
        x, weight, bias, state, starts, lengths = ctx.saved_tensors
        B, T, D = x.shape
        dx = torch.empty((B, T, D), dtype=x.dtype, device=x.device)
        dweight = _empty_like(weight)
        dbias = _empty_like(bias) if bias is not None else None
        dstate = _empty_like(state) if state is not None else None
        if dy is None:
            dy = torch.zeros(D, dtype=x.dtype, device=x.device).expand(B, T, D)
        elif dy.stride(2) != 1:
            dy = dy.contiguous()
        if dlast is not None and not dlast.is_contiguous():
            dlast = dlast.contiguous()
        if x.numel():
            desc, need, fn = _conv_desc(x, weight, bias, state, starts, lengths, ctx.silu, T), ctypes.c_size_t(), lib()
            check(fn.pcrl_short_conv_bwd_workspace_bytes(byref(desc), byref(need)))
            work = torch.empty(need.value, dtype=torch.uint8, device=x.device)
            _launch("short_conv_bwd", x.device.index, fn.pcrl_short_conv_bwd, byref(desc), dy.data_ptr(), dy.stride(0), dy.stride(1), _at(dlast),
                    dx.data_ptr(), dweight.data_ptr(), _at(dbias), _at(dstate), work.data_ptr(), need.value)
        else:                                                   # no step: the state passes through
            dweight.zero_()
            if dbias is not None:
                dbias.zero_()
            if dstate is not None:
                dstate.copy_(dlast) if dlast is not None else dstate.zero_()
        return dx, dweight, dbias, dstate, None, None, None


def short_conv(x, weight, bias=None, state=None, starts=None, lengths=None, activation="silu"):
    """y[b, t, d] = act(bias[d] + sum_k weight[d, k] x[b, t - (W - 1) + k, d]) with W = 1 ... 4 taps; act is SiLU or nothing.

    x [B, T, D]; weight [D, W], bias [D] float32; state [B, W - 1, D] of x's type: the inputs in front of this call, oldest first (default:
    zeros); starts, lengths: see the module.  Returns (y [B, T, D], last_state [B, W - 1, D]); differentiable in x, weight, bias and state."""
    args = _conv_checked(x, weight, bias, state, starts, lengths, activation, 3)
    _on_gpu(x)
    if _wants_grad(*args[:4]):
        return _ShortConv.apply(*args)
    return _conv_forward(*args)


@torch.no_grad()
def short_conv_step(x, state, weight, bias=None, starts=None, activation="silu", state_out=None):
    """One step of `short_conv`: x [B, D], state [B, W - 1, D] -> y [B, D].  The state is updated in place, or written to `state_out` (which must
    not overlap it); starts [B]: rows whose sequence begins here.  Not differentiable."""
    x, weight, bias, state, starts, _, silu = _conv_checked(x, weight, bias, state, starts, None, activation, 2)
    out = _state_out(state, state_out)
    _on_gpu(x)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if y.numel():
        desc = _conv_desc(x, weight, bias, state, starts, None, silu, 1)
        _launch("short_conv_step", x.device.index, lib().pcrl_short_conv_fwd, byref(desc), y.data_ptr(), out.data_ptr())
    return y


def _state_out(state, out):
    """Where a step leaves the new state: `state` itself, or a tensor that does not overlap it."""
    if state is None:
        raise ValueError("a step needs a state")
    if not state.is_contiguous():
        raise ValueError("the state of a step must be contiguous (it is updated in place)")
    if out is None:
        return state
    if out.shape != state.shape or out.dtype != state.dtype or out.device != state.device or not out.is_contiguous():
        raise ValueError(f"state_out is {out.dtype} {tuple(out.shape)} on {out.device}, expected a contiguous twin of the state")
    size = state.numel() * state.element_size()
    if out.data_ptr() != state.data_ptr() and abs(out.data_ptr() - state.data_ptr()) < size:
        raise ValueError("state_out overlaps the state")
    return out


# ---- selective state space scan -------------------------------------------------------------------------------------------------------------
def _ssm_checked(u, dt, A, B, C, D, z, dt_bias, state, starts, lengths, dims):
    if u.dim() != dims:
        raise ValueError(f"u is {tuple(u.shape)}, expected {'[B, D]' if dims == 2 else '[B, T, D]'}")
    _sequence_dtype(u)
    u = u if u.stride(-1) == 1 else u.contiguous()
    rows, width = u.shape[:-1], u.shape[-1]
    dt = _activation("dt", dt, u.shape, u)
    z = _activation("z", z, u.shape, u) if z is not None else None
    if A.dim() != 2 or not 1 <= A.shape[1] <= 32:
        raise ValueError(f"A is {tuple(A.shape)}, expected [{width}, N] with 1 to 32 states")
    N = A.shape[1]
    A = _parameter("A", A, (width, N), u)
    D = _parameter("D", D, (width,), u) if D is not None else None
    dt_bias = _parameter("dt_bias", dt_bias, (width,), u) if dt_bias is not None else None
    if state is not None:
        state = _parameter("state", state, (u.shape[0], width, N), u) if dims == 3 else state
    G = B.shape[-2] if B.dim() == dims + 1 else 1
    if B.dim() == dims:
        B = B.unsqueeze(-2)
    if C.dim() == dims:
        C = C.unsqueeze(-2)
    if G < 1 or width % G:
        raise ValueError(f"{width} channels are not shared evenly by {G} groups")
    B, C = _activation("B", B, rows + (G, N), u), _activation("C", C, rows + (G, N), u)
    starts, lengths = _marks(starts, lengths, rows, u)
    return u, dt, A, B, C, D, z, dt_bias, state, starts, lengths


def _ssm_desc(u, dt, A, B, C, D, z, dt_bias, state, starts, lengths, softplus):
    step = u.dim() == 2
    if step:
        T, su, sd, sz, sb, sc = 1, u.stride(), dt.stride(), z.stride() if z is not None else (0,), B.stride(), C.stride()
        su, sd, sz, sb, sc = (su[0], 0), (sd[0], 0), (sz[0], 0), (sb[0], 0, sb[1]), (sc[0], 0, sc[1])
    else:
        T, su, sd, sz, sb, sc = u.shape[1], u.stride(), dt.stride(), z.stride() if z is not None else (0, 0), B.stride(), C.stride()
    return SsmDesc(u.shape[0], T, u.shape[-1], A.shape[1], B.shape[-2], _DTYPES[u.dtype], softplus, 0, u.data_ptr(), dt.data_ptr(), _at(z),
                   su[0], su[1], sd[0], sd[1], sz[0], sz[1], B.data_ptr(), C.data_ptr(), sb[0], sb[1], sb[2], sc[0], sc[1], sc[2],
                   A.data_ptr(), _at(D), _at(dt_bias), _at(state), _at(starts), T, _at(lengths))


def _ssm_forward(args, softplus, keep):
    """(y, last state, what a backward needs: the kept states and the size of its workspace)"""
    u, A, state = args[0], args[2], args[8]
    B, T, D = u.shape
    y = torch.empty((B, T, D), dtype=u.dtype, device=u.device)
    last = torch.empty((B, D, A.shape[1]), dtype=torch.float32, device=u.device)
    if not y.numel():
        last.copy_(state) if state is not None else last.zero_()
        return y, last, None, 0
    desc, need, kept, bwd, fn = _ssm_desc(*args, softplus), ctypes.c_size_t(), ctypes.c_size_t(), ctypes.c_size_t(), lib()
    check(fn.pcrl_ssm_scan_bytes(byref(desc), byref(need), byref(kept), byref(bwd)))
    work = torch.empty(need.value, dtype=torch.uint8, device=u.device) if need.value else None
    saved = torch.empty(kept.value // 4, dtype=torch.float32, device=u.device) if keep else None
    _launch("ssm_scan_fwd", u.device.index, fn.pcrl_ssm_scan_fwd, byref(desc), y.data_ptr(), last.data_ptr(), _at(saved), _at(work), need.value)
    return y, last, saved, bwd.value


class _SsmScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, softplus, *args):
        ctx.set_materialize_grads(False)
        ctx.softplus = softplus
        y, last, saved, ctx.work_bytes = _ssm_forward(args, softplus, True)
        ctx.save_for_backward(*args, saved)
        return y, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dlast):
        if dy is None and dlast is None:
            return (None,) * 12
        *args, saved = ctx.saved_tensors
        u, dt, A, B, C, D, z, dt_bias, state = args[:9]
        shape, dev = u.shape, u.device
        dense = u.is_contiguous()
        full = (lambda t: _empty_like(t)) if dense and dt.is_contiguous() and (z is None or z.is_contiguous()) else \
            (lambda t: torch.empty(shape, dtype=u.dtype, device=dev))
        du, ddt, dz = full(u), full(dt), full(z) if z is not None else None
        dB, dC = torch.empty(B.shape, dtype=u.dtype, device=dev), torch.empty(C.shape, dtype=u.dtype, device=dev)
        dA, dD, dbias, dstate = _empty_like(A), *((_empty_like(t) if t is not None else None) for t in (D, dt_bias, state))
        if dy is None:
            dy = torch.zeros(shape[2], dtype=u.dtype, device=dev).expand(shape)
        elif dy.stride(2) != 1 or dy.stride(1) < 0:
            dy = dy.contiguous()
        if dlast is not None and not dlast.is_contiguous():
            dlast = dlast.contiguous()
        if u.numel():
            grads = SsmGrads(du.data_ptr(), ddt.data_ptr(), _at(dz), dB.data_ptr(), dC.data_ptr(), dA.data_ptr(), _at(dD), _at(dbias), _at(dstate))
            work = torch.empty(ctx.work_bytes, dtype=torch.uint8, device=dev)
            _launch("ssm_scan_bwd", dev.index, lib().pcrl_ssm_scan_bwd, byref(_ssm_desc(*args, ctx.softplus)), saved.data_ptr(), dy.data_ptr(),
                    dy.stride(0), dy.stride(1), _at(dlast), byref(grads), work.data_ptr(), ctx.work_bytes)
        else:                                                   # no step: the state passes through
            for t in (du, ddt, dA, dB, dC, dD, dz, dbias):
                if t is not None:
                    t.zero_()
            if dstate is not None:
                dstate.copy_(dlast) if dlast is not None else dstate.zero_()
        return None, du, ddt, dA, dB, dC, dD, dz, dbias, dstate, None, None


def ssm_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, starts=None, lengths=None):
    """Selective state space scan over a sequence, for every channel d and its states n:

        s_t = softplus(dt_t + dt_bias)  (softplus=False: dt_t + dt_bias)
        h_t[n] = exp(s_t A[d, n]) h_{t-1}[n] + s_t B_t[n] u_t,     y_t = (sum_n C_t[n] h_t[n] + D u_t) * silu(z_t)

    u, dt, z [B, T, D]; B, C [B, T, N] or [B, T, G, N] (G groups share the channels in order, evenly); A [D, N] with 1 to 32 states, D [D],
    dt_bias [D], state [B, D, N] (default: zeros) float32; starts, lengths: see the module.  Returns (y [B, T, D], last_state [B, D, N]);
    differentiable in all of them.  A call that will be differentiated keeps the state in front of every 16th step (N / 4 bytes an element)."""
    args = _ssm_checked(u, dt, A, B, C, D, z, dt_bias, state, starts, lengths, 3)
    _on_gpu(u)
    if _wants_grad(*args[:9]):
        return _SsmScan.apply(int(bool(softplus)), *args)
    return _ssm_forward(args, int(bool(softplus)), False)[:2]


@torch.no_grad()
def ssm_step(u, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus=True, starts=None, state_out=None):
    """One step of `ssm_scan`: u, dt, z [B, D], B, C [B, N] or [B, G, N], state [B, D, N] float32 -> y [B, D].  The state is updated in place, or
    written to `state_out` (which must not overlap it); starts [B]: rows whose sequence begins here.  Not differentiable."""
    args = _ssm_checked(u, dt, A, B, C, D, z, dt_bias, state, starts, None, 2)
    u, A = args[0], args[2]
    out = _state_out(state, state_out)
    if state.shape != (u.shape[0], u.shape[1], A.shape[1]) or state.dtype != torch.float32 or state.device != u.device:
        raise ValueError(f"state is {state.dtype} {tuple(state.shape)} on {state.device}, expected float32 {(u.shape[0], u.shape[1], A.shape[1])} on {u.device}")
    _on_gpu(u)
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    if y.numel():
        _launch("ssm_step", u.device.index, lib().pcrl_ssm_step, byref(_ssm_desc(*args, int(bool(softplus)))), y.data_ptr(), out.data_ptr())
    return y


# ---- dropout ----------------------------------------------------------------------------------------------------------------------------------
def _rows(t):
    """t as rows x columns with adjacent columns: (tensor that owns the memory, rows, cols, row stride)."""
    if t.is_contiguous():
        return t, 1, t.numel(), t.numel()
    if t.stride(-1) == 1:
        try:
            flat = t.view(-1, t.shape[-1])
            return flat, flat.shape[0], flat.shape[1], flat.stride(0)
        except RuntimeError:
            pass
    t = t.contiguous()
    return t, 1, t.numel(), t.numel()


def _dropout(x, residual, threshold, seed, offset):
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if not out.numel():
        return out
    x, rows, cols, ld = _rows(x)
    res_ld = 0
    if residual is not None:
        residual, r_rows, r_cols, res_ld = _rows(residual)
        if r_cols != cols:                      # one is dense and the other is not: walk both by the shorter rows
            cols = min(cols, r_cols)
            rows = out.numel() // cols
            ld = cols if x.is_contiguous() else ld
            res_ld = cols if residual.is_contiguous() else res_ld
    at = offset if torch.is_tensor(offset) else None
    _launch("dropout", out.device.index, lib().pcrl_dropout, x.data_ptr(), ld, _at(residual), res_ld, out.data_ptr(), rows, cols, _DTYPES[out.dtype],
            threshold, seed, 0 if at is not None else offset, _at(at))
    return out


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, threshold, seed, offset):
        ctx.threshold, ctx.seed = threshold, seed
        ctx.offset = None if torch.is_tensor(offset) else offset
        ctx.save_for_backward(*([offset] if ctx.offset is None else []))
        return _dropout(x, residual, threshold, seed, offset)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        offset = ctx.saved_tensors[0] if ctx.offset is None else ctx.offset
        dx = _dropout(dy, None, ctx.threshold, ctx.seed, offset) if ctx.needs_input_grad[0] else None
        return dx, dy if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p, seed, offset=0, residual=None):
    """x with each element dropped (set to 0, whatever it holds) with probability p and the kept ones scaled by 1 / (1 - p), plus `residual`.

    p is taken in steps of 2^-16 (round(65536 p) / 65536, for the scale too).  Which elements go is a function of (seed, offset, position in x)
    alone: Philox4x32-10 keyed by `seed`, one 16-bit draw per element, so the backward draws the same mask again and nothing is stored.  offset:
    an integer, or a device int64 tensor of one element that is read when the kernel runs (a captured graph draws a new mask on every replay when
    the tensor is advanced in between); it must keep its value until the backward has run."""
    _sequence_dtype(x)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability {p}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual is {residual.dtype} {tuple(residual.shape)} on {residual.device}, x is {x.dtype} {tuple(x.shape)} on {x.device}")
    if torch.is_tensor(offset) and (offset.dtype != torch.int64 or offset.numel() != 1 or offset.device != x.device):
        raise ValueError("offset: an integer, or an int64 tensor of one element on the device of x")
    _on_gpu(x)
    threshold, seed = int(round(65536.0 * p)), int(seed) & 0xFFFFFFFFFFFFFFFF
    offset = offset if torch.is_tensor(offset) else int(offset) & 0xFFFFFFFFFFFFFFFF
    if _wants_grad(x, residual):
        return _Dropout.apply(x, residual, threshold, seed, offset)
    return _dropout(x, residual, threshold, seed, offset)
