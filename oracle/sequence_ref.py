"""Sequence operators in 64 bits, step by step from the definitions (test infrastructure only).

`magnitude=True` evaluates the same expressions with every term replaced by its absolute value: the sum of the magnitudes that were added up to
form each output, which is what a rounding error bound is relative to."""
import numpy as np
import torch


def _silu(z):
    s = torch.sigmoid(z)
    return z * s, s + z * s * (1 - s)


def _rows(lengths, starts, B, T):
    n = [T] * B if lengths is None else [max(0, min(T, int(v))) for v in lengths]
    return n, torch.zeros(B, T, dtype=torch.bool) if starts is None else starts.bool().cpu()


def conv(x, weight, bias=None, state=None, starts=None, lengths=None, silu=True, dy=None, dlast=None, magnitude=False):
    """dict(y, last[, dx, dweight, dbias, dstate]) of x [B, T, D], weight [D, W]; gradients of sum(y dy) + sum(last dlast)."""
    m = torch.abs if magnitude else (lambda t: t)
    d = lambda t: None if t is None else t.detach().double().cpu()
    x, weight, bias, state, dy, dlast = (d(t) for t in (x, weight, bias, state, dy, dlast))
    B, T, D = x.shape
    W = weight.shape[1]
    length, starts = _rows(lengths, starts, B, T)
    out = dict(y=torch.zeros(B, T, D, dtype=torch.float64), last=torch.zeros(B, W - 1, D, dtype=torch.float64))
    if dy is not None:
        out.update(dx=torch.zeros_like(x), dweight=torch.zeros_like(weight), dbias=torch.zeros(D, dtype=torch.float64),
                   dstate=torch.zeros(B, W - 1, D, dtype=torch.float64))
    for b in range(B):
        # window: (where its gradient goes, index, value) of the last W - 1 inputs; None where nothing stands
        window = [("dstate", j, state[b, j]) if state is not None else None for j in range(W - 1)]
        for t in range(length[b]):
            if starts[b, t]:
                window = [None] * (W - 1)
            taps = window + [("dx", t, x[b, t])]
            pre = torch.zeros(D, dtype=torch.float64) if bias is None else bias.clone()
            for k, tap in enumerate(taps):
                if tap is not None:
                    pre = pre + weight[:, k] * tap[2]
            mag = torch.zeros(D, dtype=torch.float64) if bias is None else bias.abs()
            for k, tap in enumerate(taps):
                if tap is not None:
                    mag = mag + (weight[:, k] * tap[2]).abs()
            val, slope = _silu(pre) if silu else (pre, torch.ones_like(pre))
            # a silu passes an error of its argument on with a slope of at most 1.1
            out["y"][b, t] = mag * 1.1 + val.abs() if magnitude else val
            if dy is not None:
                dpre = dy[b, t] * slope
                if magnitude:                                # the slope's own error: silu'' <= 0.5 times the argument's
                    dpre = dy[b, t].abs() * (slope.abs() + (0.5 * mag if silu else 0.0))
                for k, tap in enumerate(taps):
                    if tap is not None:
                        out[tap[0]][b, tap[1]] += m(weight[:, k]) * dpre
                        out["dweight"][:, k] += dpre * m(tap[2])
                out["dbias"] += dpre
            window = taps[1:]
        for j, tap in enumerate(window):
            if tap is not None:
                out["last"][b, j] = m(tap[2])
                if dlast is not None:
                    out[tap[0]][b, tap[1]] += m(dlast[b, j])
    return out


def scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, starts=None, lengths=None, dy=None, dlast=None, magnitude=False):
    """dict(y, last[, du, ddt, dA, dB, dC, dD, dz, ddt_bias, dstate]) of u [Bt, T, Dm], B, C [Bt, T, G, N]; gradients of sum(y dy) + sum(last dlast)."""
    m = torch.abs if magnitude else (lambda t: t)
    d = lambda t: None if t is None else t.detach().double().cpu()
    u, dt, A, B, C, D, z, dt_bias, state, dy, dlast = (d(t) for t in (u, dt, A, B, C, D, z, dt_bias, state, dy, dlast))
    Bt, T, Dm = u.shape
    G, N = B.shape[2], B.shape[3]
    length, starts = _rows(lengths, starts, Bt, T)
    raw = dt if dt_bias is None else dt + dt_bias
    step = torch.nn.functional.softplus(raw, threshold=1e9) if softplus else raw
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    zeros = lambda *s: torch.zeros(*s, dtype=torch.float64)
    out = dict(y=zeros(Bt, T, Dm), last=zeros(Bt, Dm, N))
    if dy is not None:
        out.update(du=zeros(Bt, T, Dm), ddt=zeros(Bt, T, Dm), dA=zeros(Dm, N), dB=zeros(Bt, T, G, N), dC=zeros(Bt, T, G, N), dD=zeros(Dm),
                   dz=zeros(Bt, T, Dm), ddt_bias=zeros(Dm), dstate=zeros(Bt, Dm, N))
    spread = lambda v: v[:, None].expand(G, Dm // G, N).reshape(Dm, N)          # [G, N] -> [Dm, N]
    gather = lambda v: v.reshape(G, Dm // G, N).sum(1)
    skip = zeros(Dm) if D is None else m(D)
    for b in range(Bt):
        h = zeros(Dm, N) if state is None else m(state[b])
        hist = []
        for t in range(length[b]):
            s = m(step[b, t])[:, None]
            a = torch.exp(step[b, t][:, None] * A)
            if starts[b, t]:
                a = torch.zeros_like(a)
                h = torch.zeros_like(h)
            before = h
            h = a * h + s * m(spread(B[b, t])) * m(u[b, t])[:, None]
            total = (m(spread(C[b, t])) * h).sum(1) + skip * m(u[b, t])
            gate, dgate = _silu(z[b, t]) if z is not None else (torch.ones(Dm, dtype=torch.float64), None)
            if magnitude and z is not None:                 # silu and its slope carry rounding errors of their arguments' size
                gate, dgate = gate.abs(), dgate.abs() + 0.5 * z[b, t].abs() + 0.5
            out["y"][b, t] = total * gate
            hist.append((a, before, h, total, gate, dgate))
        out["last"][b] = h
        if dy is None:
            continue
        carry = zeros(Dm, N) if dlast is None else m(dlast[b])
        for t in reversed(range(length[b])):
            a, before, h, total, gate, dgate = hist[t]
            s, ut, gy = m(step[b, t]), m(u[b, t]), m(dy[b, t])
            ds = gy * gate
            g = m(spread(C[b, t])) * ds[:, None] + carry
            carry = a * g
            gb = (g * m(spread(B[b, t]))).sum(1)
            w = carry * before
            out["du"][b, t] = s * gb + skip * ds
            # magnitude: the slope of softplus and the step are functions of raw, each good to a few roundings
            dstep = ut * gb + (w * m(A)).sum(1)
            out["ddt"][b, t] = dstep * slope[b, t]
            out["dA"] += w * s[:, None]
            out["dB"][b, t] = gather(g * (s * ut)[:, None])
            out["dC"][b, t] = gather(h * ds[:, None])
            out["dD"] += ds * ut
            if z is not None:
                out["dz"][b, t] = gy * total * dgate
        out["dstate"][b] = carry
    if dy is not None:
        out["ddt_bias"] = out["ddt"].sum((0, 1))
    return out


def dropout_keep(n, threshold, seed, offset):
    """bool [n]: which elements of a tensor stay (Philox4x32-10 on Python-checked 64-bit integers)."""
    i = np.arange((n + 7) // 8, dtype=np.uint64)
    low, word = np.uint64(0xFFFFFFFF), np.uint64(32)
    offset, seed = int(offset) & (2 ** 64 - 1), int(seed) & (2 ** 64 - 1)
    c = [i & low, i >> word, np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> word) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> word) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    halves = np.stack([np.stack([v & np.uint64(0xFFFF), v >> np.uint64(16)], 1) for v in c], 1).reshape(-1)[:n]
    return torch.from_numpy(halves >= np.uint64(threshold))
