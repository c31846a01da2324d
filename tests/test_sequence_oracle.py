"""The 64-bit definitions the sequence operators are tested against (oracle/sequence_ref.py): their gradient formulas equal central differences of
their own forward, and the generator equals the framework's C++ Philox restated in plain integers."""
import pytest
import torch

from oracle import sequence_ref as ref


def _inputs(seed, Bt, T, Dm, N, G, with_z, with_state, starts, lengths):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    kw = dict(u=r(Bt, T, Dm), dt=r(Bt, T, Dm), A=-torch.rand(Dm, N, generator=g, dtype=torch.float64) - 0.2, B=r(Bt, T, G, N), C=r(Bt, T, G, N), D=r(Dm),
              z=r(Bt, T, Dm) if with_z else None, dt_bias=r(Dm), state=r(Bt, Dm, N) if with_state else None)
    if starts:
        kw["starts"] = torch.rand(Bt, T, generator=g) < 0.3
    if lengths:
        kw["lengths"] = torch.tensor([T, T // 2, 0][:Bt])
    return kw, r(Bt, T, Dm), r(Bt, Dm, N)


def _difference(f, x, i, eps=1e-6):
    hi, lo = x.clone(), x.clone()
    hi.view(-1)[i] += eps
    lo.view(-1)[i] -= eps
    return (f(hi) - f(lo)) / (2 * eps)


# central differences of a function with third derivatives of order 1 at eps = 1e-6: 1e-12 of truncation, 1e-16 / 1e-6 = 1e-10 of rounding per
# unit of the loss (of order 10 here)
DIFF = 1e-8


@pytest.mark.parametrize("softplus,with_z,with_state,starts,lengths,G", [(True, True, True, True, True, 2), (False, False, False, False, False, 1),
                                                                        (True, False, True, True, False, 1), (True, True, False, False, True, 1)])
def test_scan_gradients_equal_differences(softplus, with_z, with_state, starts, lengths, G):
    Bt, T, Dm, N = 3, 6, 4, 3
    kw, dy, dlast = _inputs(1, Bt, T, Dm, N, G, with_z, with_state, starts, lengths)
    if not softplus:
        kw["dt"], kw["dt_bias"] = kw["dt"].abs() * 0.1, None
    out = ref.scan(**kw, softplus=softplus, dy=dy, dlast=dlast)

    def loss(name):
        def f(v):
            o = ref.scan(**dict(kw, **{name: v}), softplus=softplus)
            return float((o["y"] * dy).sum() + (o["last"] * dlast).sum())
        return f

    names = dict(u="du", dt="ddt", A="dA", B="dB", C="dC", D="dD", z="dz", dt_bias="ddt_bias", state="dstate")
    g = torch.Generator().manual_seed(5)
    for name, grad in names.items():
        if kw.get(name) is None:
            continue
        for i in torch.randperm(kw[name].numel(), generator=g)[:12].tolist():
            want = _difference(loss(name), kw[name], i)
            assert abs(float(out[grad].reshape(-1)[i]) - want) <= DIFF * max(1.0, abs(want)) * 10, (name, i)


@pytest.mark.parametrize("silu,with_state,starts,lengths,W", [(True, True, True, True, 4), (False, False, False, False, 2), (True, True, False, True, 3),
                                                              (True, True, True, False, 1)])
def test_conv_gradients_equal_differences(silu, with_state, starts, lengths, W):
    B, T, D = 3, 7, 3
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    kw = dict(x=r(B, T, D), weight=r(D, W), bias=r(D), state=r(B, W - 1, D) if with_state else None)
    if starts:
        kw["starts"] = torch.rand(B, T, generator=g) < 0.3
    if lengths:
        kw["lengths"] = torch.tensor([T, 2, 0])
    dy, dlast = r(B, T, D), r(B, W - 1, D)
    out = ref.conv(**kw, silu=silu, dy=dy, dlast=dlast)

    def loss(name):
        def f(v):
            o = ref.conv(**dict(kw, **{name: v}), silu=silu)
            return float((o["y"] * dy).sum() + (o["last"] * dlast).sum())
        return f

    for name, grad in dict(x="dx", weight="dweight", bias="dbias", state="dstate").items():
        if kw.get(name) is None or not kw[name].numel():
            continue
        for i in torch.randperm(kw[name].numel(), generator=g)[:12].tolist():
            want = _difference(loss(name), kw[name], i)
            assert abs(float(out[grad].reshape(-1)[i]) - want) <= DIFF * max(1.0, abs(want)) * 10, (name, i)


def test_a_sequence_cut_in_two_equals_the_whole():
    """The state carried from one call to the next, in 64 bits: both operators."""
    kw, _, _ = _inputs(3, 2, 9, 4, 3, 1, True, True, True, False)
    whole = ref.scan(**kw)
    part = lambda a, b, state: ref.scan(**{k: (v[:, a:b] if k in ("u", "dt", "z", "B", "C", "starts") else v) for k, v in dict(kw, state=state).items()})
    first = part(0, 4, kw["state"])
    second = part(4, 9, first["last"])
    assert torch.allclose(torch.cat([first["y"], second["y"]], 1), whole["y"], atol=1e-13) and torch.allclose(second["last"], whole["last"], atol=1e-13)
    g = torch.Generator().manual_seed(4)
    x, w, st = torch.randn(2, 9, 3, generator=g), torch.randn(3, 4, generator=g), torch.randn(2, 3, 3, generator=g)
    whole = ref.conv(x, w, state=st, starts=kw["starts"])
    first = ref.conv(x[:, :2], w, state=st, starts=kw["starts"][:, :2])
    second = ref.conv(x[:, 2:], w, state=first["last"], starts=kw["starts"][:, 2:])
    assert torch.allclose(torch.cat([first["y"], second["y"]], 1), whole["y"], atol=1e-13) and torch.allclose(second["last"], whole["last"], atol=1e-13)


def test_generator_known_answers():
    """Philox4x32-10 known answers of Salmon et al. (counter and key all zero, all ones): the half-words the mask is made of."""
    zero = [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    for t in (1, 0x2000, 0x8000, 0xF000, 0xFFFF):
        halves = [h for w in zero for h in (w & 0xFFFF, w >> 16)]
        assert ref.dropout_keep(8, t, 0, 0).tolist() == [h >= t for h in halves]
