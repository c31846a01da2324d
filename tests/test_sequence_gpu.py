"""Sequence operators (pointcloud_rl_amd/sequence.py) against their 64-bit definitions (oracle/sequence_ref.py).

Tolerances.  An output of type t is rounded once: eps(t) / 2 of its value.  In front of that stand float32 roundings of the terms it is summed from:
k 2^-24 of the sum of their magnitudes (the oracle's magnitude=True), with k the longest chain of roundings a term goes through --
  scan: at most 4 roundings a step of the recurrence (the decay's exponential 2, its product and the sum), once forward and once backward;
  N states, 64 for the gates' elementary functions (softplus, sigmoid, silu and their slopes: below 10 each); the argument of a decay carries
  its own 4 relative roundings, 4 X with X the summed argument -- no more than 40 of it, beyond which e^-X is below every other term's rounding;
  the sums over channels (dB, dC) and over batch and steps (parameters) add one rounding per term.
  conv: W + 1 terms, 16 for silu and its slope, and the same sums over batch and steps.
float16 also stops at its smallest subnormal: 2^-25 absolute."""
import ctypes

import pytest
import torch

from oracle import sequence_ref as ref

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
U = 2.0 ** -24


def close(name, got, want, mag, k):
    """got within the bound above of want."""
    got = got.detach().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    half = torch.finfo(got.dtype).eps / 2 if got.dtype != F32 else 0.0
    tol = half * want.abs() + k * U * mag * (1 + half) + (2.0 ** -25 if got.dtype == F16 else 1e-37)
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / tol.clamp(min=1e-300)).nan_to_num(1e9).max()):.3g} times the bound"


# ctypes mirrors of the sequence descriptors of include/pcrl.h, for calls of the C entry points themselves
class ConvDesc(ctypes.Structure):
    _fields_ = [("B", ctypes.c_int32), ("T", ctypes.c_int32), ("D", ctypes.c_int32), ("W", ctypes.c_int32), ("dtype", ctypes.c_int32),
                ("silu", ctypes.c_int32), ("x", ctypes.c_void_p), ("x_sb", ctypes.c_int64), ("x_st", ctypes.c_int64), ("weight", ctypes.c_void_p),
                ("bias", ctypes.c_void_p), ("state", ctypes.c_void_p), ("starts", ctypes.c_void_p), ("starts_sb", ctypes.c_int64),
                ("lengths", ctypes.c_void_p)]


class SsmDesc(ctypes.Structure):
    _fields_ = [("B", ctypes.c_int32), ("T", ctypes.c_int32), ("D", ctypes.c_int32), ("N", ctypes.c_int32), ("G", ctypes.c_int32),
                ("dtype", ctypes.c_int32), ("softplus", ctypes.c_int32), ("_pad", ctypes.c_int32),
                ("u", ctypes.c_void_p), ("dt", ctypes.c_void_p), ("z", ctypes.c_void_p),
                ("u_sb", ctypes.c_int64), ("u_st", ctypes.c_int64), ("dt_sb", ctypes.c_int64), ("dt_st", ctypes.c_int64),
                ("z_sb", ctypes.c_int64), ("z_st", ctypes.c_int64), ("Bm", ctypes.c_void_p), ("Cm", ctypes.c_void_p),
                ("b_sb", ctypes.c_int64), ("b_st", ctypes.c_int64), ("b_sg", ctypes.c_int64),
                ("c_sb", ctypes.c_int64), ("c_st", ctypes.c_int64), ("c_sg", ctypes.c_int64),
                ("A", ctypes.c_void_p), ("D_skip", ctypes.c_void_p), ("dt_bias", ctypes.c_void_p), ("state", ctypes.c_void_p),
                ("starts", ctypes.c_void_p), ("starts_sb", ctypes.c_int64), ("lengths", ctypes.c_void_p)]


class SsmGrads(ctypes.Structure):
    _fields_ = [(k, ctypes.c_void_p) for k in ("du", "ddt", "dz", "dB", "dC", "dA", "dD", "ddt_bias", "dstate")]


# ---- scan ------------------------------------------------------------------------------------------------------------------------------------
def scan_inputs(dev, dtype, Bt, T, Dm, N, G=1, z=True, skip=True, bias=True, state=True, starts=0.0, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    kw = dict(u=r(Bt, T, Dm).to(dtype), dt=(0.5 * r(Bt, T, Dm)).to(dtype), A=-torch.arange(1, N + 1).float() * (0.5 + torch.rand(Dm, N, generator=g)),
              B=r(Bt, T, G, N).to(dtype), C=r(Bt, T, G, N).to(dtype), D=r(Dm) if skip else None, z=r(Bt, T, Dm).to(dtype) if z else None,
              dt_bias=r(Dm) * 0.5 - 2.0 if bias else None, state=r(Bt, Dm, N) if state else None)
    if starts:
        kw["starts"] = torch.rand(Bt, T, generator=g) < starts
    if lengths is not None:
        kw["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    on = {k: v.to(dev) if v is not None else None for k, v in kw.items()}
    return kw, on, r(Bt, T, Dm).to(dtype), r(Bt, Dm, N)


def scan_k(kw, softplus):
    raw = kw["dt"].double() + (kw["dt_bias"].double() if kw["dt_bias"] is not None else 0.0)
    step = torch.nn.functional.softplus(raw) if softplus else raw
    X = float(torch.einsum("btd,dn->bdn", step.abs(), kw["A"].double().abs()).max())
    return 4 * kw["u"].shape[1] + kw["A"].shape[1] + 64 + 4 * min(X, 40.0)


LEAVES = ("u", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")
GRAD = dict(u="du", dt="ddt", A="dA", B="dB", C="dC", D="dD", z="dz", dt_bias="ddt_bias", state="dstate")


def check_scan(dev, kw, on, dy, dlast, softplus=True, backward=True):
    from pointcloud_rl_amd import sequence
    want = ref.scan(**kw, softplus=softplus, dy=dy if backward else None, dlast=dlast)
    mag = ref.scan(**kw, softplus=softplus, dy=dy if backward else None, dlast=dlast, magnitude=True)
    k = scan_k(kw, softplus)
    plain = sequence.ssm_scan(**on, softplus=softplus)
    close("y", plain[0], want["y"], mag["y"], k)
    close("last", plain[1], want["last"], mag["last"], k)
    if not backward:
        return
    on = {n: v.clone().requires_grad_() if n in LEAVES and v is not None else v for n, v in on.items()}
    y, last = sequence.ssm_scan(**on, softplus=softplus)
    assert torch.equal(y, plain[0]) and torch.equal(last, plain[1])          # keeping states for the backward changes no bit
    names = [n for n in LEAVES if on[n] is not None]
    grads = torch.autograd.grad((y, last), [on[n] for n in names], (dy.to(dev), dlast.to(dev)))
    Bt, T, Dm = kw["u"].shape
    for n, got in zip(names, grads):
        more = Dm if n in ("B", "C") else Bt * T if n in ("A", "D", "dt_bias") else 0
        close(GRAD[n], got, want[GRAD[n]], mag[GRAD[n]], 2 * k + more)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Bt,T,Dm,N,G", [(1, 1, 1, 1, 1), (2, 16, 64, 16, 1), (3, 17, 65, 11, 1), (2, 33, 130, 4, 2), (1, 70, 96, 32, 3), (2, 15, 20, 17, 1),
                                         (130, 3, 64, 16, 1), (260, 2, 40, 16, 1)])
def test_scan_forward_and_gradients(cuda, dtype, Bt, T, Dm, N, G):
    kw, on, dy, dlast = scan_inputs(cuda, dtype, Bt, T, Dm, N, G, seed=T)
    check_scan(cuda, kw, on, dy, dlast)


@pytest.mark.gpu
@pytest.mark.parametrize("opts", [dict(z=False), dict(skip=False), dict(bias=False), dict(state=False), dict(z=False, skip=False, bias=False, state=False)])
def test_scan_without_its_optional_inputs(cuda, opts):
    kw, on, dy, dlast = scan_inputs(cuda, F32, 2, 37, 70, 16, **opts)
    check_scan(cuda, kw, on, dy, dlast)


@pytest.mark.gpu
def test_scan_without_softplus(cuda):
    kw, on, dy, dlast = scan_inputs(cuda, F32, 2, 20, 33, 8, bias=False)
    kw["dt"] = kw["dt"].abs() * 0.1
    on["dt"] = kw["dt"].to(cuda)
    check_scan(cuda, kw, on, dy, dlast, softplus=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("starts,lengths", [(0.2, None), (1.0, None), (0.0, [40, 0, 1, 17]), (0.15, [33, 40, 16, 0])])
def test_scan_starts_and_lengths(cuda, dtype, starts, lengths):
    kw, on, dy, dlast = scan_inputs(cuda, dtype, 4, 40, 72, 16, starts=starts, lengths=lengths)
    check_scan(cuda, kw, on, dy, dlast)


@pytest.mark.gpu
@pytest.mark.parametrize("Bt,T,Dm,N,starts,lengths", [(1, 1500, 64, 16, 0.0, None), (2, 1100, 40, 5, 0.002, [1100, 517])])
def test_scan_long_sequences_are_cut_and_joined(cuda, Bt, T, Dm, N, starts, lengths):
    """Few channels, many steps: the sequence is walked in chunks that start from the combined summaries of the ones in front of them."""
    kw, on, dy, dlast = scan_inputs(cuda, F32, Bt, T, Dm, N, starts=starts, lengths=lengths)
    check_scan(cuda, kw, on, dy, dlast)


@pytest.mark.gpu
def test_scan_reads_strided_inputs(cuda):
    """u and z as halves of one projection, dt, B and C as slices of another, a transposed (channel-strided) u, an expanded B: the same bits as
    the contiguous call; gradients of an expanded input add up."""
    from pointcloud_rl_amd import sequence
    Bt, T, Dm, N = 3, 21, 40, 8
    g = torch.Generator().manual_seed(3)
    xz = torch.randn(Bt, T, 2 * Dm + 1, generator=g).to(cuda)
    rest = torch.randn(Bt, T, Dm + 2 * N + 3, generator=g).to(cuda)
    A = -torch.rand(Dm, N, generator=g).to(cuda) - 0.1
    u, z, dt = xz[..., 1:Dm + 1], xz[..., Dm + 1:], rest[..., :Dm]
    B, C = rest[..., Dm:Dm + N], rest[..., Dm + N:Dm + 2 * N]
    dense = [t.contiguous() for t in (u, dt, A, B, C)]
    want = sequence.ssm_scan(*dense, z=z.contiguous())
    got = sequence.ssm_scan(u, dt, A, B, C, z=z)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    ut = u.transpose(1, 2).contiguous().transpose(1, 2)
    assert ut.stride(-1) != 1
    got = sequence.ssm_scan(ut, dt, A, B, C, z=z)
    assert torch.equal(got[0], want[0])
    one = B[:1, :1].clone().requires_grad_()
    full = one.detach().expand(Bt, T, N).clone().requires_grad_()
    for b in (one.expand(Bt, T, N), full):
        y, _ = sequence.ssm_scan(u, dt, A, b, C, z=z)
        y.square().sum().backward()
    assert torch.allclose(one.grad, full.grad.sum((0, 1), keepdim=True), rtol=1e-4, atol=1e-5 * float(full.grad.abs().sum()))


@pytest.mark.gpu
def test_scan_masked_places_may_hold_anything(cuda):
    """NaN and infinities behind the length and in what a start cuts off reach nothing; grads there are exactly 0."""
    from pointcloud_rl_amd import sequence
    kw, on, dy, dlast = scan_inputs(cuda, F32, 2, 24, 33, 8, lengths=[24, 10])
    starts = torch.zeros(2, 24, dtype=torch.bool)
    starts[:, 5] = True
    kw["starts"], on["starts"] = starts, starts.to(cuda)
    want = sequence.ssm_scan(**on)
    dirty = {n: (v.clone() if v is not None else None) for n, v in on.items()}
    for n in ("u", "dt", "B", "C", "z"):
        dirty[n][1, 10:] = float("nan")
    dirty["state"][0, 3] = float("inf")
    dirty["u"][0, 2, 4] = float("nan")
    leaves = {n: dirty[n].requires_grad_() for n in LEAVES}
    y, last = sequence.ssm_scan(**dict(dirty, **leaves))
    assert torch.equal(y[:, 5:].cpu(), want[0][:, 5:].cpu()) and torch.equal(last, want[1])
    gy = dy.to(cuda).clone()
    gy[:, :5] = 0.0
    gy[1, 10:] = float("nan")
    du, dz = torch.autograd.grad((y, last), [leaves["u"], leaves["z"]], (gy, dlast.to(cuda)))
    assert torch.isfinite(du[:, 5:]).all() and (du[1, 10:] == 0).all() and (dz[1, 10:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("Bt,Dm,N,G,starts", [(1, 1, 1, 1, False), (5, 70, 16, 1, True), (3, 66, 11, 2, True), (2, 40, 32, 1, False), (9, 24, 6, 1, True)])
def test_step_equals_the_scan_and_the_definition(cuda, dtype, Bt, Dm, N, G, starts):
    """Steps one after the other, in place and to another tensor, against the 64-bit scan of the whole run."""
    from pointcloud_rl_amd import sequence
    T = 5
    kw, on, _, _ = scan_inputs(cuda, dtype, Bt, T, Dm, N, G, starts=0.3 if starts else 0.0)
    want, mag = ref.scan(**kw), ref.scan(**kw, magnitude=True)
    k = scan_k(kw, True)
    state, ys = on["state"].clone(), []
    for t in range(T):
        st = on["starts"][:, t] if starts else None
        args = (on["u"][:, t], on["dt"][:, t], on["A"], on["B"][:, t], on["C"][:, t])
        kept = state.clone()
        other = torch.full_like(state, float("nan"))
        y2 = sequence.ssm_step(*args, state, D=on["D"], z=on["z"][:, t], dt_bias=on["dt_bias"], starts=st, state_out=other)
        assert torch.equal(state, kept)
        y = sequence.ssm_step(*args, state, D=on["D"], z=on["z"][:, t], dt_bias=on["dt_bias"], starts=st)
        assert torch.equal(y, y2) and torch.equal(state, other)
        ys.append(y)
    close("y", torch.stack(ys, 1), want["y"], mag["y"], k)
    close("state", state, want["last"], mag["last"], k)


# ---- convolution -----------------------------------------------------------------------------------------------------------------------------
def conv_inputs(dev, dtype, B, T, D, W, bias=True, state=True, starts=0.0, lengths=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    kw = dict(x=r(B, T, D).to(dtype), weight=r(D, W), bias=r(D) if bias else None, state=r(B, W - 1, D).to(dtype) if state else None)
    if starts:
        kw["starts"] = torch.rand(B, T, generator=g) < starts
    if lengths is not None:
        kw["lengths"] = torch.tensor(lengths, dtype=torch.int32)
    on = {k: v.to(dev) if v is not None else None for k, v in kw.items()}
    return kw, on, r(B, T, D).to(dtype), r(B, W - 1, D).to(dtype)


def check_conv(dev, kw, on, dy, dlast, silu=True):
    from pointcloud_rl_amd import sequence
    want = ref.conv(**kw, silu=silu, dy=dy, dlast=dlast)
    mag = ref.conv(**kw, silu=silu, dy=dy, dlast=dlast, magnitude=True)
    W, (B, T, _) = kw["weight"].shape[1], kw["x"].shape
    act = "silu" if silu else None
    plain = sequence.short_conv(**on, activation=act)
    close("y", plain[0], want["y"], mag["y"], W + 1 + 16)
    assert torch.equal(plain[1].cpu().double(), want["last"])
    on = {n: v.clone().requires_grad_() if n in ("x", "weight", "bias", "state") and v is not None else v for n, v in on.items()}
    y, last = sequence.short_conv(**on, activation=act)
    names = [n for n in ("x", "weight", "bias", "state") if on[n] is not None]
    if W == 1 and "state" in names:
        names.remove("state")
    grads = torch.autograd.grad((y, last), [on[n] for n in names], (dy.to(dev), dlast.to(dev)))
    for n, got in zip(names, grads):
        close("d" + n, got, want["d" + n], mag["d" + n], 2 * W + 32 + (B * T if n in ("weight", "bias") else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,T,D,W", [(1, 1, 1, 4), (2, 2, 8, 4), (3, 17, 65, 3), (2, 33, 130, 2), (4, 70, 64, 4), (2, 9, 16, 1), (70, 5, 24, 4)])
def test_conv_forward_and_gradients(cuda, dtype, B, T, D, W):
    kw, on, dy, dlast = conv_inputs(cuda, dtype, B, T, D, W, seed=T)
    check_conv(cuda, kw, on, dy, dlast)


@pytest.mark.gpu
@pytest.mark.parametrize("opts,silu", [(dict(bias=False), True), (dict(state=False), False), (dict(bias=False, state=False), True), (dict(), False)])
def test_conv_without_its_optional_parts(cuda, opts, silu):
    kw, on, dy, dlast = conv_inputs(cuda, F32, 2, 19, 36, 4, **opts)
    check_conv(cuda, kw, on, dy, dlast, silu)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("starts,lengths", [(0.2, None), (1.0, None), (0.0, [40, 0, 1, 2, 17, 8]), (0.2, [39, 3, 16, 0, 32, 33])])
def test_conv_starts_and_lengths(cuda, dtype, starts, lengths):
    kw, on, dy, dlast = conv_inputs(cuda, dtype, 6, 40, 20, 4, starts=starts, lengths=lengths)
    check_conv(cuda, kw, on, dy, dlast)


@pytest.mark.gpu
def test_conv_reads_strided_inputs_and_masked_places_may_hold_anything(cuda):
    from pointcloud_rl_amd import sequence
    kw, on, dy, dlast = conv_inputs(cuda, F32, 2, 24, 32, 4, lengths=[24, 10])
    want = sequence.short_conv(**on)
    wide = torch.randn(2, 24, 67, device=cuda)
    wide[..., 3:35] = on["x"]
    got = sequence.short_conv(**dict(on, x=wide[..., 3:35]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    dirty = on["x"].clone()
    dirty[1, 10:] = float("nan")
    dirty.requires_grad_()
    got = sequence.short_conv(**dict(on, x=dirty))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    gy = dy.to(cuda).clone()
    gy[1, 10:] = float("inf")
    dx, = torch.autograd.grad(got, dirty, (gy, dlast.to(cuda)))
    assert torch.isfinite(dx).all() and (dx[1, 10:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,D,W,starts", [(1, 1, 4, False), (5, 70, 4, True), (3, 64, 2, True), (2, 9, 3, False)])
def test_conv_steps_equal_the_sequence(cuda, dtype, B, D, W, starts):
    """Steps one after the other, in place and to another tensor: the same bits as the sequence form."""
    from pointcloud_rl_amd import sequence
    T = 6
    kw, on, _, _ = conv_inputs(cuda, dtype, B, T, D, W, starts=0.4 if starts else 0.0)
    y, last = sequence.short_conv(**on)
    state = on["state"].clone()
    for t in range(T):
        st = on["starts"][:, t] if starts else None
        other, kept = torch.empty_like(state), state.clone()
        y2 = sequence.short_conv_step(on["x"][:, t], state, on["weight"], on["bias"], starts=st, state_out=other)
        assert torch.equal(state, kept)
        yt = sequence.short_conv_step(on["x"][:, t], state, on["weight"], on["bias"], starts=st)
        assert torch.equal(yt, y2) and torch.equal(state, other) and torch.equal(yt, y[:, t]), t
    assert torch.equal(state, last)


# ---- dropout -----------------------------------------------------------------------------------------------------------------------------------
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", [(1,), (7,), (3, 5, 11), (64, 1024), (1000, 33)])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_dropout_values_and_gradient(cuda, dtype, shape, p):
    from pointcloud_rl_amd import sequence
    g = torch.Generator().manual_seed(1)
    x, res, dy = (torch.randn(*shape, generator=g).to(dtype) for _ in range(3))
    threshold, seed, offset = round(p * 65536), 0x123456789ABCDEF, (1 << 40) + 5
    keep = ref.dropout_keep(x.numel(), threshold, seed, offset).reshape(shape)
    scale = 0.0 if threshold == 65536 else 65536.0 / (65536 - threshold)
    xd, rd = x.to(cuda).requires_grad_(), res.to(cuda).requires_grad_()
    y = sequence.dropout(xd, p, seed, offset, residual=rd)
    want = torch.where(keep, x.double() * scale, 0.0)
    close("y", y, want + res.double(), want.abs() * 2 + (want + res.double()).abs(), 1)       # scale, product (2), sum (1)
    dx, dr = torch.autograd.grad(y, (xd, rd), dy.to(cuda))
    assert torch.equal(dr.cpu(), dy)
    want = torch.where(keep, dy.double() * scale, 0.0)
    close("dx", dx, want, want.abs(), 2)
    assert torch.equal(dx.cpu() == 0, (~keep) | (dy * scale == 0) | (dx.cpu() == 0))
    assert (dx.cpu()[~keep] == 0).all()


@pytest.mark.gpu
def test_dropout_layouts_offsets_and_bad_values(cuda):
    from pointcloud_rl_amd import sequence
    wide = torch.randn(6, 5, 50, device=cuda)
    x = wide[..., 4:37]
    want = sequence.dropout(x.contiguous(), 0.3, 9, 4)
    assert torch.equal(sequence.dropout(x, 0.3, 9, 4), want)                                          # row stride
    assert torch.equal(sequence.dropout(x.transpose(0, 1), 0.3, 9, 4), sequence.dropout(x.transpose(0, 1).contiguous(), 0.3, 9, 4))
    assert torch.equal(sequence.dropout(x, 0.3, 9, 4, residual=x.contiguous()), sequence.dropout(x.contiguous(), 0.3, 9, 4, residual=x))
    flat = torch.randn(1001, device=cuda)
    assert torch.equal(sequence.dropout(flat[1:], 0.3, 9, 4), sequence.dropout(flat[1:].clone(), 0.3, 9, 4))     # unaligned
    at = torch.tensor([4], device=cuda)
    assert torch.equal(sequence.dropout(x, 0.3, 9, at), want) and not torch.equal(sequence.dropout(x, 0.3, 9, 5), want)
    bad = torch.full((4096,), float("nan"), device=cuda)
    out = sequence.dropout(bad, 0.5, 1, 0)
    keep = ref.dropout_keep(4096, 32768, 1, 0).to(cuda)
    assert (out[~keep] == 0).all() and out[keep].isnan().all()
    assert (sequence.dropout(bad, 1.0, 1, 0) == 0).all()
    # an offset that is advanced between forward and backward is an error, not another mask
    xg = flat.clone().requires_grad_()
    y = sequence.dropout(xg, 0.5, 1, at)
    at += 1
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()


# ---- what holds for all of them ------------------------------------------------------------------------------------------------------------------
def _train_pass(sequence, conv, scan, offset):
    x = conv["x"]
    y, _ = sequence.short_conv(x, conv["weight"], conv["bias"], starts=scan["starts"])
    y, last = sequence.ssm_scan(y, scan["dt"], scan["A"], scan["B"], scan["C"], D=scan["D"], z=scan["z"], dt_bias=scan["dt_bias"], starts=scan["starts"])
    y = sequence.dropout(y, 0.1, 77, offset, residual=x)
    leaves = [x, conv["weight"], scan["dt"], scan["A"], scan["B"], scan["C"], scan["z"]]
    return (y.detach(), last.detach()) + torch.autograd.grad((y, last), leaves, (2 * y.detach(), torch.ones_like(last)))      # of sum y^2 + sum last


def _train_inputs(dev, dtype=F32, Bt=4, T=50, Dm=48):
    _, conv, _, _ = conv_inputs(dev, dtype, Bt, T, Dm, 4)
    _, scan, _, _ = scan_inputs(dev, dtype, Bt, T, Dm, 16, starts=0.05)
    for d, names in ((conv, ("x", "weight")), (scan, ("dt", "A", "B", "C", "z"))):
        for n in names:
            d[n].requires_grad_()
    return conv, scan


@pytest.mark.gpu
def test_convolution_scan_and_dropout_in_a_row(cuda):
    """The three as a recurrent core runs them, forward and backward, against the chained 64-bit definitions."""
    from pointcloud_rl_amd import sequence
    conv, scan = _train_inputs(cuda)
    got = _train_pass(sequence, conv, scan, 3)
    x = conv["x"].detach().double().cpu()
    c = ref.conv(x, conv["weight"], conv["bias"], starts=scan["starts"])
    args = dict(dt=scan["dt"], A=scan["A"], B=scan["B"], C=scan["C"], D=scan["D"], z=scan["z"], dt_bias=scan["dt_bias"], starts=scan["starts"])
    s = ref.scan(u=c["y"], **args)
    keep = ref.dropout_keep(x.numel(), 6554, 77, 3).reshape(x.shape)
    scale = 65536.0 / (65536 - 6554)
    y = torch.where(keep, s["y"] * scale, 0.0) + x
    dy = 2 * y
    back = ref.scan(u=c["y"], **args, dy=torch.where(keep, dy * scale, 0.0), dlast=torch.ones_like(s["last"]))
    cb = ref.conv(x, conv["weight"], conv["bias"], starts=scan["starts"], dy=back["du"])
    want = (y, s["last"], dy + cb["dx"], cb["dweight"], back["ddt"], back["dA"], back["dB"], back["dC"], back["dz"])
    for i, (a, b) in enumerate(zip(got, want)):
        # three operators' bounds on top of each other; relative to the largest value, whose chains are the longest
        assert float((a.detach().cpu().double() - b).abs().max()) <= 3 * 1000 * U * max(1.0, float(b.abs().max())), i


@pytest.mark.gpu
def test_the_same_call_gives_the_same_bits(cuda):
    from pointcloud_rl_amd import sequence
    conv, scan = _train_inputs(cuda, BF16, 3, 130, 100)
    a, b = _train_pass(sequence, conv, scan, 1), _train_pass(sequence, conv, scan, 1)
    for i, (u, v) in enumerate(zip(a, b)):
        assert torch.equal(u, v), i


@pytest.mark.gpu
def test_captured_and_replayed(cuda):
    """Forward and backward in one hipGraph, replayed several times with eager work in between; the offset on the device moves the mask."""
    from pointcloud_rl_amd import sequence
    conv, scan = _train_inputs(cuda)
    offset = torch.zeros(1, dtype=torch.int64, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _train_pass(sequence, conv, scan, offset)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _train_pass(sequence, conv, scan, offset)
    for k in range(4):
        offset.fill_(k)
        with torch.no_grad():
            conv["x"].add_(0.01)
        want = _train_pass(sequence, conv, scan, k)
        torch.cuda.synchronize()
        graph.replay()
        for i, (u, v) in enumerate(zip(out, want)):
            assert torch.equal(u, v), (k, i)


@pytest.mark.gpu
def test_two_streams_at_once(cuda):
    """Two passes on two streams share nothing: each allocates its own scratch."""
    from pointcloud_rl_amd import sequence
    sets = [_train_inputs(cuda, F32, 2, 200, 64), _train_inputs(cuda, BF16, 3, 150, 100)]
    want = [_train_pass(sequence, *s, 5) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(3):
        got = []
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(_train_pass(sequence, *s, 5))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(u, v) for u, v in zip(a, b))


@pytest.mark.gpu
def test_nothing_to_do(cuda):
    """No steps, no rows: the state passes through, gradients are zeros."""
    from pointcloud_rl_amd import sequence
    for Bt, T in ((2, 0), (0, 3)):
        _, on, dy, dlast = scan_inputs(cuda, F32, Bt, T, 8, 4)
        leaves = {n: on[n].requires_grad_() for n in LEAVES}
        y, last = sequence.ssm_scan(**leaves)
        assert y.shape == (Bt, T, 8) and torch.equal(last, on["state"])
        grads = torch.autograd.grad((y, last), list(leaves.values()), (dy.to(cuda), dlast.to(cuda)))
        for n, gr in zip(leaves, grads):
            assert torch.equal(gr, dlast.to(cuda)) if n == "state" else (gr == 0).all()
        _, on, dy, dlast = conv_inputs(cuda, F32, Bt, T, 8, 4)
        leaves = {n: on[n].requires_grad_() for n in ("x", "weight", "bias", "state")}
        y, last = sequence.short_conv(**leaves)
        assert y.shape == (Bt, T, 8) and torch.equal(last, on["state"])
        grads = torch.autograd.grad((y, last), list(leaves.values()), (dy.to(cuda), dlast.to(cuda)))
        assert torch.equal(grads[3], dlast.to(cuda)) and all((gr == 0).all() for gr in grads[:3])
    assert sequence.dropout(torch.zeros(0, 4, device=cuda), 0.5, 1).shape == (0, 4)
    y = sequence.ssm_step(*(torch.zeros(0, n, device=cuda) for n in (8, 8)), torch.zeros(8, 4, device=cuda), torch.zeros(0, 4, device=cuda),
                          torch.zeros(0, 4, device=cuda), torch.zeros(0, 8, 4, device=cuda))
    assert y.shape == (0, 8)


@pytest.mark.gpu
def test_one_output_alone_is_differentiated(cuda):
    """Only y, or only the last state, takes part in the loss."""
    from pointcloud_rl_amd import sequence
    kw, on, dy, dlast = scan_inputs(cuda, F32, 2, 20, 36, 8)
    on = {n: v.requires_grad_() if n in LEAVES and v is not None else v for n, v in on.items()}
    names = list(LEAVES)
    for which, (gy, gl) in enumerate(((dy, torch.zeros_like(dlast)), (torch.zeros_like(dy), dlast))):
        both = torch.autograd.grad(sequence.ssm_scan(**on), [on[n] for n in names], (gy.to(cuda), gl.to(cuda)))
        out = sequence.ssm_scan(**on)[which]
        alone = torch.autograd.grad(out, [on[n] for n in names], (gy, gl)[which].to(cuda))
        for n, a, b in zip(names, alone, both):
            assert torch.equal(a, b), (which, n)


# ---- refusals (no GPU needed) ---------------------------------------------------------------------------------------------------------------------
def _cpu(*s, dtype=F32):
    return torch.zeros(*s, dtype=dtype)


def test_cpu_tensors_are_refused():
    from pointcloud_rl_amd import sequence
    with pytest.raises(RuntimeError, match="no CPU path"):
        sequence.short_conv(_cpu(1, 2, 8), _cpu(8, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        sequence.ssm_scan(_cpu(1, 2, 8), _cpu(1, 2, 8), _cpu(8, 4), _cpu(1, 2, 4), _cpu(1, 2, 4))
    with pytest.raises(RuntimeError, match="no CPU path"):
        sequence.dropout(_cpu(4), 0.5, 1)
    with pytest.raises(RuntimeError, match="no CPU path"):
        sequence.ssm_step(_cpu(1, 8), _cpu(1, 8), _cpu(8, 4), _cpu(1, 4), _cpu(1, 4), _cpu(1, 8, 4))


def test_arguments_that_do_not_fit_are_refused():
    from pointcloud_rl_amd import sequence
    x, w = _cpu(2, 3, 8), _cpu(8, 4)
    for kw in (dict(x=_cpu(3, 8)), dict(weight=_cpu(8, 5)), dict(weight=_cpu(7, 4)), dict(weight=_cpu(8, 4, dtype=BF16)), dict(bias=_cpu(4)),
               dict(state=_cpu(2, 4, 8)), dict(state=_cpu(2, 3, 8, dtype=BF16)), dict(starts=_cpu(2, 3)), dict(starts=_cpu(2, dtype=torch.bool)),
               dict(lengths=_cpu(2)), dict(lengths=_cpu(3, dtype=torch.int32)), dict(activation="relu"), dict(x=_cpu(2, 3, 8, dtype=torch.float64))):
        with pytest.raises(ValueError):
            sequence.short_conv(**dict(dict(x=x, weight=w), **kw))
    ok = dict(u=x, dt=x, A=_cpu(8, 4), B=_cpu(2, 3, 4), C=_cpu(2, 3, 4))
    for kw in (dict(u=_cpu(2, 8)), dict(dt=_cpu(2, 3, 7)), dict(dt=x.to(BF16)), dict(A=_cpu(8, 33), B=_cpu(2, 3, 33), C=_cpu(2, 3, 33)), dict(A=_cpu(7, 4)),
               dict(A=_cpu(8, 0), B=_cpu(2, 3, 0), C=_cpu(2, 3, 0)), dict(B=_cpu(2, 3, 5)), dict(B=_cpu(2, 3, 3, 4), C=_cpu(2, 3, 3, 4)), dict(C=_cpu(2, 3, 2, 4)),
               dict(z=_cpu(2, 3, 4)), dict(D=_cpu(4)), dict(dt_bias=_cpu(8, dtype=F16)), dict(state=_cpu(2, 4, 8)), dict(state=_cpu(2, 8, 4, dtype=BF16)),
               dict(starts=_cpu(2, 4, dtype=torch.bool)), dict(lengths=_cpu(2, dtype=F32))):
        with pytest.raises(ValueError):
            sequence.ssm_scan(**dict(ok, **kw))
    step = dict(u=_cpu(2, 8), dt=_cpu(2, 8), A=_cpu(8, 4), B=_cpu(2, 4), C=_cpu(2, 4), state=_cpu(2, 8, 4))
    whole = _cpu(4, 8, 4)
    for kw in (dict(u=x), dict(state=None), dict(state=_cpu(2, 4, 8).transpose(1, 2)), dict(state=_cpu(2, 8, 4, dtype=BF16)), dict(state_out=_cpu(2, 8, 5)),
               dict(state=whole[:2], state_out=whole[1:3]), dict(starts=_cpu(2, 1, dtype=torch.bool))):
        with pytest.raises(ValueError):
            sequence.ssm_step(**dict(step, **kw))
    for kw in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(residual=_cpu(3)), dict(residual=_cpu(4, dtype=BF16)), dict(offset=_cpu(1)),
               dict(x=_cpu(4, dtype=torch.int32))):
        with pytest.raises(ValueError):
            sequence.dropout(**dict(dict(x=_cpu(4), p=0.5, seed=1), **kw))


def test_the_c_entry_points_refuse_bad_descriptors():
    from pointcloud_rl_amd import _lib
    lib = _lib.lib()
    one = ctypes.c_void_p(4096)                       # never dereferenced: every call below is refused before a launch
    n = ctypes.c_size_t()

    def ssm(**kw):
        d = SsmDesc(B=1, T=2, D=8, N=4, G=1, u=4096, dt=4096, Bm=4096, Cm=4096, A=4096)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    def conv(**kw):
        d = ConvDesc(B=1, T=2, D=8, W=4, x=4096, weight=4096)
        for k, v in kw.items():
            setattr(d, k, v)
        return ctypes.byref(d)

    for kw in (dict(B=0), dict(T=-1), dict(D=0), dict(N=0), dict(N=33), dict(G=3), dict(dtype=1), dict(u=None), dict(A=None)):
        assert lib.pcrl_ssm_scan_fwd(ssm(**kw), one, None, None, None, ctypes.c_size_t(0), None) == -1, kw
        assert lib.pcrl_ssm_scan_bytes(ssm(**kw), ctypes.byref(n), None, None) == -1
    assert lib.pcrl_ssm_scan_fwd(None, one, None, None, None, ctypes.c_size_t(0), None) == -1
    assert lib.pcrl_ssm_scan_fwd(ssm(), None, None, None, None, ctypes.c_size_t(0), None) == -1
    assert lib.pcrl_ssm_scan_bwd(ssm(), one, one, ctypes.c_int64(16), ctypes.c_int64(8), None, None, one, ctypes.c_size_t(1 << 30), None) == -1
    grads = SsmGrads(*[4096] * 9)
    assert lib.pcrl_ssm_scan_bwd(ssm(), one, one, ctypes.c_int64(16), ctypes.c_int64(8), None, ctypes.byref(grads), one, ctypes.c_size_t(16), None) == -2
    assert b"workspace" in lib.pcrl_last_error()
    assert lib.pcrl_ssm_step(ssm(), one, one, None) == -1 and lib.pcrl_ssm_step(ssm(T=1), one, one, None) == -1        # T = 2; no state
    for kw in (dict(B=0), dict(W=5), dict(W=0), dict(dtype=2), dict(x=None), dict(weight=None)):
        assert lib.pcrl_short_conv_fwd(conv(**kw), one, None, None) == -1, kw
    assert lib.pcrl_short_conv_fwd(conv(state=4096), one, one, None) == -1 and b"in place" in lib.pcrl_last_error()
    assert lib.pcrl_short_conv_bwd(conv(), one, ctypes.c_int64(16), ctypes.c_int64(8), None, one, one, None, None, one, ctypes.c_size_t(8), None) == -2
    drop = lambda x, rows, cols, dtype, thr: lib.pcrl_dropout(x, ctypes.c_int64(cols), None, ctypes.c_int64(0), one, ctypes.c_int64(rows), ctypes.c_int64(cols), dtype,
                                                             thr, ctypes.c_uint64(0), ctypes.c_uint64(0), None, None)
    for args in ((None, 1, 4, 0, 1), (one, 0, 4, 0, 1), (one, 1, 0, 0, 1), (one, 1, 4, 1, 1), (one, 1, 4, 0, -1), (one, 1, 4, 0, 65537), (one, 1 << 30, 1 << 30, 0, 1)):
        assert drop(*args) == -1, args


@pytest.mark.gpu
def test_a_zero_state_stays_zero_where_the_decays_overflow(cuda):
    """Growing states (A > 0), chunks whose product of decays is beyond float32: what is zero in front of such a chunk is zero behind it, both ways."""
    kw, on, dy, dlast = scan_inputs(cuda, F32, 1, 1500, 64, 16, z=False, skip=False, bias=False, state=False)
    kw["A"] = torch.full_like(kw["A"], 8.0)                    # e^8 a step, e^128 over a tile of 16
    kw["dt"] = torch.ones_like(kw["dt"])
    kw["u"][:, :-3] = 0.0
    dy[:, 2:] = 0.0
    on.update((n, kw[n].to(cuda)) for n in ("A", "dt", "u"))
    check_scan(cuda, kw, on, dy, torch.zeros_like(dlast), softplus=False)


@pytest.mark.gpu
def test_lengths_of_64_bits(cuda):
    from pointcloud_rl_amd import sequence
    kw, on, _, _ = scan_inputs(cuda, F32, 3, 20, 24, 8)
    wide = torch.tensor([2 ** 40 + 3, -2 ** 40, 7], device=cuda)
    narrow = torch.tensor([20, 0, 7], dtype=torch.int32, device=cuda)
    for a, b in zip(sequence.ssm_scan(**on, lengths=wide), sequence.ssm_scan(**on, lengths=narrow)):
        assert torch.equal(a, b)
    w = torch.randn(24, 4, device=cuda)
    for a, b in zip(sequence.short_conv(on["u"], w, lengths=wide), sequence.short_conv(on["u"], w, lengths=narrow)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_steps_far_apart_in_memory(cuda):
    """A step stride beyond what the scan's offsets reach: the input is copied."""
    from pointcloud_rl_amd import sequence
    base = torch.zeros((1 << 26) + 64, dtype=BF16, device=cuda)
    kw, on, _, _ = scan_inputs(cuda, BF16, 1, 2, 16, 4)
    far = base.as_strided((1, 2, 16), (1 << 27, 1 << 26, 1))
    far.copy_(on["u"])
    want = sequence.ssm_scan(**on)
    for a, b in zip(sequence.ssm_scan(**dict(on, u=far)), want):
        assert torch.equal(a, b)
    w = torch.randn(16, 4, device=cuda)
    for a, b in zip(sequence.short_conv(far, w), sequence.short_conv(on["u"], w)):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_second_derivatives_are_refused(cuda):
    from pointcloud_rl_amd import sequence
    kw, on, _, _ = scan_inputs(cuda, F32, 1, 5, 8, 4)
    u = on["u"].requires_grad_()
    for y in (sequence.ssm_scan(**on)[0], sequence.short_conv(u, torch.randn(8, 4, device=cuda))[0], sequence.dropout(u, 0.5, 3)):
        with pytest.raises(RuntimeError, match="differentiable once"):
            torch.autograd.grad(y.sum(), u, create_graph=True)


@pytest.mark.gpu
def test_a_state_updated_in_place_does_not_pass_for_the_saved_one(cuda):
    from pointcloud_rl_amd import sequence
    kw, on, _, _ = scan_inputs(cuda, F32, 2, 5, 8, 4)
    y, _ = sequence.ssm_scan(**dict(on, u=on["u"].requires_grad_()))
    step = {n: on[n][:, 0] if n in ("u", "dt", "B", "C", "z") else on[n] for n in on}
    sequence.ssm_step(**step)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    conv = torch.zeros(2, 3, 8, device=cuda)
    w = torch.randn(8, 4, device=cuda, requires_grad=True)
    y, _ = sequence.short_conv(on["u"].detach(), w, state=conv)
    sequence.short_conv_step(on["u"][:, 0].detach(), conv, w)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


@pytest.mark.gpu
def test_steps_in_inference_mode(cuda):
    from pointcloud_rl_amd import sequence
    x, w = torch.randn(2, 8, device=cuda), torch.randn(8, 4, device=cuda)
    outer = torch.zeros(2, 3, 8, device=cuda)
    want = sequence.short_conv_step(x, outer.clone(), w)
    with torch.inference_mode():
        inner = torch.zeros(2, 3, 8, device=cuda)
        assert torch.equal(sequence.short_conv_step(x, inner, w), want) and torch.equal(sequence.short_conv_step(x, outer, w), want)
        assert torch.equal(inner, outer)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 7, 4099])
def test_dropout_in_place_through_the_c_entry_point(cuda, n):
    from pointcloud_rl_amd import _lib, sequence
    x, r = torch.randn(n, device=cuda), torch.randn(n, device=cuda)
    want = sequence.dropout(x, 0.25, 11, offset=5, residual=r)
    at = lambda t: ctypes.c_void_p(t.data_ptr())
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    ld, one, seed, offset = ctypes.c_int64(n), ctypes.c_int64(1), ctypes.c_uint64(11), ctypes.c_uint64(5)
    for out in (x.clone(), r.clone()):
        a, b = (out, r) if torch.equal(out, x) else (x, out)
        assert _lib.lib().pcrl_dropout(at(a), ld, at(b), ld, at(out), one, ld, 0, 1 << 14, seed, offset, None, stream) == 0
        assert torch.equal(out, want)


def test_sizes_beyond_the_kernels_indexes_are_refused():
    from pointcloud_rl_amd import _lib
    lib = _lib.lib()
    one, n = ctypes.c_void_p(4096), ctypes.c_size_t()      # never dereferenced
    for kw in (dict(T=0x7FFFFFF0), dict(B=(1 << 30) + 1), dict(D=1 << 26), dict(u_st=1 << 26), dict(dt_st=-1), dict(c_st=1 << 26)):
        d = SsmDesc(**dict(dict(B=1, T=2, D=8, N=4, G=1, u=4096, dt=4096, Bm=4096, Cm=4096, A=4096), **kw))
        assert lib.pcrl_ssm_scan_fwd(ctypes.byref(d), one, None, None, None, ctypes.c_size_t(0), None) == -1, kw
        assert lib.pcrl_ssm_scan_bytes(ctypes.byref(d), ctypes.byref(n), None, None) == -1, kw
    for kw in (dict(T=0x7FFFFFF0), dict(D=1 << 26), dict(B=1 << 24, T=1 << 12, D=64)):
        d = ConvDesc(**dict(dict(B=1, T=2, D=8, W=4, x=4096, weight=4096), **kw))
        assert lib.pcrl_short_conv_fwd(ctypes.byref(d), one, None, None) == -1, kw
    big = ctypes.c_int64(1 << 36)
    assert lib.pcrl_dropout(one, big, None, big, one, ctypes.c_int64(1), big, 0, 1, ctypes.c_uint64(0), ctypes.c_uint64(0), None, None) == -1


def test_struct_layouts_match_the_header(tmp_path):
    """sizeof / offsetof of the sequence descriptors as gcc lays them out == the ctypes mirror."""
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pairs = [("pcrl_conv_desc", ConvDesc), ("pcrl_ssm_desc", SsmDesc), ("pcrl_ssm_grads", SsmGrads)]
    lines = []
    for cname, cls in pairs:
        lines.append(f'printf("{cname} %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname}.{f} %zu\\n", offsetof({cname}, {f}));' for f, _ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "pcrl.h"\nint main(void) {\n' + "\n".join(lines) + "\nreturn 0; }\n")
    subprocess.run(["gcc", "-I", os.path.join(root, "include"), str(src), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for cname, cls in pairs:
        assert int(got[cname]) == ctypes.sizeof(cls)
        for f, _ in cls._fields_:
            assert int(got[f"{cname}.{f}"]) == getattr(cls, f).offset, f"{cname}.{f}"
