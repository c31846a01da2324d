"""Dropout on views: the layouts that its row walk (csrc/torch_binding.cpp: rows_of) sees, on the CPU, and the kernel's results on the GPU."""
import random

import pytest
import torch


def views():
    """(name, view) of tensors whose elements are all different: what slices, transposes, expansions and windows leave behind."""
    base = lambda *s: torch.arange(float(torch.Size(s).numel())).reshape(s)
    yield "steps of [B, 1, T, D]", base(3, 1, 6, 8)[:, :, :4]
    yield "channels of [B, 1, T, D]", base(3, 1, 6, 8)[..., :5]
    yield "steps and channels of [B, 1, T, D]", base(2, 1, 5, 16)[..., :4, :8]
    yield "one step of [B, 1, T, D]", base(4, 1, 2, 8)[:, :, :1]
    yield "two unit axes", base(4, 2, 1, 1, 8)[:, :1, :, :, 2:7]
    yield "a unit axis in front", base(1, 5, 9, 8)[:, :, 3:7, 1:]
    yield "rows of a matrix", base(7, 12)[:, 4:9]
    yield "a column", base(7, 12)[:, 4:5]
    yield "every other row", base(8, 12)[::2]
    yield "transposed", base(4, 6, 8).transpose(0, 1)
    yield "transposed, the inner axes sliced", base(4, 6, 8).transpose(0, 1)[..., :3]
    yield "an expanded row", base(8).expand(5, 8)
    yield "an expanded row on two axes", base(8).expand(3, 4, 8)
    yield "an expanded matrix", base(4, 8).expand(3, 4, 8)
    yield "an expanded unit axis", base(4, 1, 8).expand(4, 3, 8)[..., :5]
    yield "overlapping windows", base(40).unfold(0, 8, 2)
    yield "overlapping windows behind a unit axis", base(3, 40).unfold(1, 8, 2)[:, :, None, :5]
    yield "a unit axis with a stride of its own", base(200).as_strided((4, 1, 3, 8), (48, 999, 16, 1), 3)
    yield "two unit axes with strides of their own", base(80).as_strided((4, 1, 1, 8), (16, 16, 999, 1))


def _cut(g):
    """A random view of a random tensor of two to four axes, unit axes among them."""
    shape = [g.choice((1, 1, 2, 3, 5)) for _ in range(g.randint(1, 3))] + [g.choice((1, 4, 8))]
    t = torch.arange(float(torch.Size(shape).numel())).reshape(shape)
    for axis in range(t.dim()):
        n = t.size(axis)
        lo = g.randrange(n)
        t = t.narrow(axis, lo, g.randint(1, n - lo))
    if g.random() < 0.3:
        a, b = g.randrange(t.dim()), g.randrange(t.dim())
        t = t.transpose(a, b)
    if g.random() < 0.3:
        t = t.unsqueeze(g.randrange(t.dim()))
    if g.random() < 0.3:
        t = t.expand([g.choice((2, 3)) if n == 1 and g.random() < 0.5 else n for n in t.shape])
    return t


def test_the_rows_of_a_view_are_the_view():
    """Rows, columns and stride of every layout: inside the tensor's memory, and the tensor's own elements in order."""
    from pointcloud_rl_amd import _lib
    ext = _lib.sequence_ext()
    g = random.Random(7)
    seen = list(views()) + [(f"random {i}", _cut(g)) for i in range(2000)]
    walked = 0
    for name, t in seen:
        rows, cols, ld, copied = ext.dropout_rows(t)
        assert rows * cols == t.numel(), (name, t.shape, t.stride())
        if copied:
            assert not t.is_contiguous()
            continue
        walked += not t.is_contiguous()
        last = t.storage_offset() + (rows - 1) * ld + cols - 1
        assert ld >= 0 and last < t.untyped_storage().nbytes() // 4, (name, t.shape, t.stride(), (rows, cols, ld))
        assert torch.equal(t.as_strided((rows, cols), (ld, 1)).reshape(-1), t.reshape(-1)), (name, t.shape, t.stride(), (rows, cols, ld))
    assert walked > 200                                  # views are walked where they stand, not copied


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_dropout_of_views_equals_dropout_of_their_copies(cuda, dtype):
    """x, the residual and the incoming gradient as views: the bits of the contiguous call."""
    from pointcloud_rl_amd import sequence
    for name, v in views():
        # the same view of random values of the type
        values = torch.randn(v.untyped_storage().nbytes() // 4, generator=torch.Generator().manual_seed(1)).to(dtype).to(cuda)
        v = values.as_strided(v.shape, v.stride(), v.storage_offset())
        dense = v.contiguous()
        want = sequence.dropout(dense, 0.3, 9, 4, residual=dense)
        for x, r in ((v, dense), (dense, v), (v, v)):
            assert torch.equal(sequence.dropout(x, 0.3, 9, 4, residual=r), want), name
        x = dense.clone().requires_grad_()
        y = sequence.dropout(x, 0.3, 9, 4)
        by_view, = torch.autograd.grad(y, x, v, retain_graph=True)
        by_copy, = torch.autograd.grad(y, x, dense)
        assert torch.equal(by_view, by_copy), name


@pytest.mark.gpu
def test_the_stride_of_a_single_step_may_be_anything(cuda):
    """[B, 1, D] views whose step axis has a stride beyond the scan's 32-bit offsets, which nothing steps over: the contiguous call's bits."""
    from pointcloud_rl_amd import sequence
    B, D, N = 2, 16, 4
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).to(cuda)
    dense = dict(u=r(B, 1, D), dt=r(B, 1, D), z=r(B, 1, D), B=r(B, 1, 1, N), C=r(B, 1, 1, N))
    rest = dict(A=-r(D, N).abs(), D=r(D), dt_bias=r(D), state=r(B, D, N))
    far = lambda t: t.as_strided(t.shape, (t.stride(0), 1 << 27) + t.stride()[2:])
    dy, w = r(B, 1, D), r(D, 4)

    def passes(view):
        leaves = {k: v.clone().requires_grad_() for k, v in dense.items()}
        seen = {k: view(v) for k, v in leaves.items()}
        y, last = sequence.ssm_scan(**seen, **rest)
        x = dense["u"].clone().requires_grad_()
        c, clast = sequence.short_conv(view(x), w)
        return [y, last, c, clast] + list(torch.autograd.grad(y, list(leaves.values()), view(dy))) + list(torch.autograd.grad(c, x, view(dy)))

    for i, (a, b) in enumerate(zip(passes(far), passes(lambda t: t))):
        assert torch.equal(a, b), i
