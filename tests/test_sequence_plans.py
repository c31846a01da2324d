"""The sequence operators at sizes whose launches loop: several tiles per workgroup, several rows per workgroup, several runs per walker, chunks of
several tiles -- each case with a look at the plan, so that it stays where it is meant to be.

A large batch is R different rows over and over (row b is row b % R), so that the 64-bit definition is evaluated on R rows: their outputs repeat,
and the gradients of the parameters are B / R times theirs.  R never divides the step by which a workgroup goes from row to row: the rows it
walks are different ones.  Tolerances: test_sequence_gpu.py's."""
import ctypes

import pytest
import torch

from oracle import sequence_ref as ref
from test_sequence_gpu import BF16, F16, F32, GRAD, LEAVES, ConvDesc, SsmDesc, close, conv_inputs, scan_inputs, scan_k


def cdiv(a, b):
    return -(-a // b)


def cus():
    return torch.cuda.get_device_properties(0).multi_processor_count if torch.cuda.is_available() else 256


def scan_plan(B, T, D, N, G=1):
    """(forward chunks, tiles of one; backward chunks, tiles of one; rows apart that share a workgroup of the backward), checked against the sizes of
    the scratch that the library asks for."""
    ntile, nblk, n = cdiv(T, 16), cdiv(D // G, 64), cus()
    blocks, out = B * G * nblk, []
    for per_cu in (4, 2):
        chunks = 1 if 2 * blocks >= 3 * n else min(cdiv(per_cu * n, blocks), ntile)
        tiles = cdiv(ntile, chunks)
        out += [cdiv(ntile, tiles), tiles]
    step = B if out[2] > 1 else max(1, min(B, 4 * n // (G * nblk)))
    from pointcloud_rl_amd import _lib
    sizes = [ctypes.c_size_t() for _ in range(3)]
    d = SsmDesc(B=B, T=T, D=D, N=N, G=G, u=4096, dt=4096, Bm=4096, Cm=4096, A=4096)          # (nothing is dereferenced)
    assert _lib.lib().pcrl_ssm_scan_bytes(ctypes.byref(d), *(ctypes.byref(s) for s in sizes)) == 0
    up = lambda v, to: cdiv(v, to) * to
    state, parts = N * D, step * out[2]
    sums = 0 if out[2] == 1 else B * out[2] * state
    assert sizes[0].value == (0 if out[0] == 1 else 8 * up(B * out[0] * state, 4)) and sizes[1].value == 4 * B * ntile * state
    assert sizes[2].value == 4 * sum(up(v, 64) for v in [G * nblk * B * T * N] * 2 + [parts * state, parts * D, parts * D, sums, sums])
    return tuple(out) + (step,)


def conv_plan(B, T, D, W):
    """(steps of a run, runs of a row, parts) of the backward, parts checked against the scratch that the library asks for."""
    cols, run = cdiv(D, 256), 32
    while run > 8 and cols * B * cdiv(T, run) < 8 * cus():
        run //= 2
    nrun = cdiv(T, run)
    parts = max(1, min(cdiv(B * nrun, 4), 4 * cus() // cols))
    from pointcloud_rl_amd import _lib
    size = ctypes.c_size_t()
    assert _lib.lib().pcrl_short_conv_bwd_workspace_bytes(ctypes.byref(ConvDesc(B=B, T=T, D=D, W=W, x=4096, weight=4096)), ctypes.byref(size)) == 0
    assert size.value == 4 * parts * (W + 1) * D
    return run, nrun, parts


def step_rows(D, N):
    """(rows that a workgroup of ssm_step holds at once, rows in flight over the launch)"""
    width = D * (1 if N <= 4 else 2 if N <= 8 else 4 if N <= 16 else 8)
    rows = max(1, 256 // width)
    return rows, cdiv(8 * cus(), 1 if rows > 1 else cdiv(width, 256)) * rows


# B, R, T, D, N, G; tiles of a chunk > 1 forward, backward; rows share a workgroup; chunks are joined
SCANS = [
    (400, 20, 40, 16, 16, 1, dict(one=True, tiles=3)),
    (400, 20, 40, 16, 20, 1, dict(one=True, tiles=3)),
    (400, 20, 37, 24, 32, 2, dict(one=True, tiles=3)),
    (400, 20, 35, 16, 7, 1, dict(one=True, tiles=3)),
    (400, 20, 35, 130, 16, 1, dict(one=True, tiles=3, rows=True)),
    (1100, 22, 20, 16, 16, 1, dict(one=True, tiles=2, rows=True)),
    (1100, 22, 18, 10, 24, 1, dict(one=True, tiles=2, rows=True)),
    (64, 4, 700, 64, 16, 1, dict(one=False, tiles=3)),
    (64, 4, 330, 20, 32, 1, dict(one=False, tiles=2)),
]
# B, R, T, D, W; run, lines > walkers
CONVS = [
    (2100, 21, 70, 8, 4, 32, True),
    (4200, 21, 9, 10, 4, 32, True),
    (2100, 21, 66, 12, 2, 32, True),
    (700, 20, 40, 8, 3, 16, False),
    (700, 20, 40, 300, 4, 32, False),
]
STEPS = [(1100, 22, 512, 16), (5000, 25, 24, 16), (70000, 28, 8, 4), (2500, 25, 300, 11)]      # B, R, D, N


def test_the_cases_are_where_they_are_meant_to_be():
    for B, R, T, D, N, G, want in SCANS:
        fwd, fwd_tiles, bwd, bwd_tiles, step = scan_plan(B, T, D, N, G)
        assert (fwd == 1) == (bwd == 1) == want["one"] and min(fwd_tiles, bwd_tiles) >= want["tiles"], (B, T, D)
        assert (step < B) == want.get("rows", False) and B % R == 0 and (step == B or step % R), (B, T, D)
    for B, R, T, D, W, run, more in CONVS:
        got, nrun, parts = conv_plan(B, T, D, W)
        assert got == run and (B * nrun > 4 * parts) == more and B % R == 0, (B, T, D)
        assert not more or (4 * parts) % (R * nrun)
    for B, R, D, N in STEPS:
        rows, flight = step_rows(D, N)
        assert B > flight and B % R == 0 and flight % R, (B, D, N)


def repeat(kw, on, rows, B, dev):
    """The device tensors of B rows from those of R (the ones with a batch axis)."""
    return {n: v.repeat(B // len(v), *(1,) * (v.dim() - 1)) if n in rows and v is not None else v for n, v in on.items()}


SCAN_ROWS = ("u", "dt", "B", "C", "z", "state", "starts", "lengths")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("case", range(len(SCANS)))
def test_scan_loops(cuda, case, masks, dtype):
    from pointcloud_rl_amd import sequence
    B, R, T, D, N, G, _ = SCANS[case]
    lengths = [(T * (i + 1)) // (R - 2) if i < R - 2 else (0, 1)[i - R + 2] for i in range(R)] if masks else None
    kw, on, dy, dlast = scan_inputs(cuda, dtype, R, T, D, N, G, starts=0.1 if masks else 0.0, lengths=lengths, seed=case)
    want, mag = (ref.scan(**kw, dy=dy, dlast=dlast, magnitude=m) for m in (False, True))
    k, m = scan_k(kw, True), B // R
    many = repeat(kw, on, SCAN_ROWS, B, cuda)
    plain = sequence.ssm_scan(**many)
    many = {n: v.requires_grad_() if n in LEAVES else v for n, v in many.items()}
    y, last = sequence.ssm_scan(**many)
    assert torch.equal(y, plain[0]) and torch.equal(last, plain[1])
    grads = torch.autograd.grad((y, last), [many[n] for n in LEAVES], (dy.to(cuda).repeat(m, 1, 1), dlast.to(cuda).repeat(m, 1, 1)))
    got = dict(zip((GRAD[n] for n in LEAVES), grads), y=y, last=last)
    for name, value in got.items():
        if name in ("dA", "dD", "ddt_bias"):
            close(name, value, want[name] * m, mag[name] * m, 2 * k + B * T)
            continue
        value = value.detach().reshape((m, R) + value.shape[1:])
        assert torch.equal(value, value[:1].expand_as(value)), name           # the same row, the same bits, wherever it stands
        close(name, value[0], want[name], mag[name], k if name in ("y", "last") else 2 * k + (D if name in ("dB", "dC") else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("masks", [False, True])
@pytest.mark.parametrize("case", range(len(CONVS)))
def test_conv_loops(cuda, case, masks, dtype):
    from pointcloud_rl_amd import sequence
    B, R, T, D, W, _, _ = CONVS[case]
    lengths = [(T * (i + 1)) // (R - 3) if i < R - 3 else (0, 1, 2)[i - R + 3] for i in range(R)] if masks else None
    kw, on, dy, dlast = conv_inputs(cuda, dtype, R, T, D, W, starts=0.1 if masks else 0.0, lengths=lengths, seed=case)
    want, mag = (ref.conv(**kw, dy=dy, dlast=dlast, magnitude=m) for m in (False, True))
    m = B // R
    many = repeat(kw, on, ("x", "state", "starts", "lengths"), B, cuda)
    leaves = ("x", "weight", "bias", "state")
    many = {n: v.requires_grad_() if n in leaves else v for n, v in many.items()}
    y, last = sequence.short_conv(**many)
    grads = torch.autograd.grad((y, last), [many[n] for n in leaves], (dy.to(cuda).repeat(m, 1, 1), dlast.to(cuda).repeat(m, 1, 1)))
    got = dict(zip(("d" + n for n in leaves), grads), y=y)
    assert torch.equal(last.detach().cpu().double(), want["last"].repeat(m, 1, 1))
    for name, value in got.items():
        if name in ("dweight", "dbias"):
            close(name, value, want[name] * m, mag[name] * m, 2 * W + 32 + B * T)
            continue
        value = value.detach().reshape((m, R) + value.shape[1:])
        assert torch.equal(value, value[:1].expand_as(value)), name
        close(name, value[0], want[name], mag[name], W + 17 if name == "y" else 2 * W + 32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,R,D,N", STEPS)
def test_step_loops(cuda, dtype, B, R, D, N):
    """More rows than the launch has in flight: in place and to another tensor, with fresh rows among them."""
    from pointcloud_rl_amd import sequence
    T, m = 2, B // R
    kw, on, _, _ = scan_inputs(cuda, dtype, R, T, D, N, starts=0.3)
    want, mag = ref.scan(**kw), ref.scan(**kw, magnitude=True)
    k = scan_k(kw, True)
    many = repeat(kw, on, SCAN_ROWS, B, cuda)
    state, ys = many["state"].clone(), []
    for t in range(T):
        args = [many[n][:, t] for n in ("u", "dt")] + [many["A"]] + [many[n][:, t] for n in ("B", "C")]
        rest = dict(D=many["D"], z=many["z"][:, t], dt_bias=many["dt_bias"], starts=many["starts"][:, t])
        kept, other = state.clone(), torch.full_like(state, float("nan"))
        y2 = sequence.ssm_step(*args, state, state_out=other, **rest)
        assert torch.equal(state, kept)
        ys.append(sequence.ssm_step(*args, state, **rest))
        assert torch.equal(ys[-1], y2) and torch.equal(state, other)
    for name, value in (("y", torch.stack(ys, 1)), ("last", state)):
        value = value.reshape((m, R) + value.shape[1:])
        assert torch.equal(value, value[:1].expand_as(value)), name
        close(name, value[0], want[name], mag[name], k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("B,T,D,N,rank", [(3, 40, 40, 16, 13), (2, 37, 72, 8, 5), (400, 20, 16, 16, 13), (2, 20, 24, 32, 3)])
def test_the_layout_of_the_recurrent_core(cuda, dtype, B, T, D, N, rank):
    """z the second half of one projection, B and C slices of another that start at an odd element: forward, gradients and steps against the
    definition (the slices' accesses are not whole vectors)."""
    from pointcloud_rl_amd import sequence
    R = min(B, 20)
    kw, on, dy, dlast = scan_inputs(cuda, dtype, R, T, D, N, seed=B)
    want, mag = (ref.scan(**kw, dy=dy, dlast=dlast, magnitude=v) for v in (False, True))
    k, m = scan_k(kw, True), B // R
    many = repeat(kw, on, SCAN_ROWS, B, cuda)
    both = torch.cat((torch.zeros_like(many["z"]), many["z"]), -1).requires_grad_()
    proj = torch.cat((many["u"].new_zeros(B, T, rank), many["B"][:, :, 0], many["C"][:, :, 0]), -1).requires_grad_()
    leaves = {n: many[n].requires_grad_() for n in LEAVES if n not in ("B", "C", "z")}
    seen = dict(leaves, z=both.chunk(2, -1)[1], **dict(zip("BC", proj.split([rank, N, N], -1)[1:])))
    assert seen["B"].data_ptr() % (4 * proj.element_size()) and not seen["z"].is_contiguous()
    y, last = sequence.ssm_scan(**seen)
    grads = dict(zip(list(leaves) + ["z", "p"], torch.autograd.grad((y, last), list(leaves.values()) + [both, proj],
                                                                  (dy.to(cuda).repeat(m, 1, 1), dlast.to(cuda).repeat(m, 1, 1)))))
    grads["z"], p = grads["z"][..., D:], grads.pop("p")
    grads["B"], grads["C"] = (v.reshape(B, T, 1, N) for v in p.split([rank, N, N], -1)[1:])
    got = dict({GRAD[n]: v for n, v in grads.items()}, y=y, last=last)
    for name, value in got.items():
        if name in ("dA", "dD", "ddt_bias"):
            close(name, value, want[name] * m, mag[name] * m, 2 * k + B * T)
        else:
            close(name, value.detach()[:R], want[name], mag[name], k if name in ("y", "last") else 2 * k + (D if name in ("dB", "dC") else 0))
    state = many["state"].detach().clone()
    rest = dict(D=many["D"], dt_bias=many["dt_bias"])
    ys = [sequence.ssm_step(many["u"][:, t], many["dt"][:, t], many["A"], seen["B"][:, t], seen["C"][:, t], state, z=seen["z"][:, t], **rest) for t in range(T)]
    close("steps", torch.stack(ys, 1)[:R], want["y"], mag["y"], k)
    close("state", state[:R], want["last"], mag["last"], k)
