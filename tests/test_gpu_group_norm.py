"""Group norm with an activation over channels-last features against 64 bits."""

import pytest
import torch

import trnfft_b200 as trnfft
from tests.layer_refs import UNIT, norm_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = [None, "relu", "silu", "gelu"]

SHAPES = [  # shape, groups
    ((1, 1), 1),
    ((1, 8), 2),
    ((3, 1, 24), 3),
    ((2, 5, 7), 7),          # one channel a group
    ((2, 33, 6), 2),
    ((70, 96), 4),
    ((1000, 64), 4),
    ((513, 2048), 16),
    ((3, 4096), 1),
    ((2, 7, 9, 40), 5),
    ((2, 1000, 33), 3),
    ((1, 5000, 64), 8),
    ((4, 257, 31, 48), 6),
    ((2, 64, 64, 320), 32),
    ((2, 20000, 20), 1),
    ((1, 200001, 8), 8),
    ((5, 3, 8192), 2),
    ((2, 12, 1001), 77),
    ((2, 3, 9001), 1),       # more channels than a block's shared memory holds
    ((3, 20000), 5),
    ((2, 300, 8192), 8192),
    ((300, 30, 40), 4),      # samples of a few KB
    ((700, 9, 6), 1),
]


def data(shape, dtype, seed=0, shift=0.7):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(shape, device="cuda", generator=g) * 1.5 + shift).to(dtype)
    c = shape[-1]
    w = torch.randn(c, device="cuda", generator=g) * 0.2 + 1
    b = torch.randn(c, device="cuda", generator=g) * 0.2
    return x, w, b, torch.randn(shape, device="cuda", generator=g).to(dtype)


def near(got, want, dtype, what, size=None):
    """Statistics in 32 bits over up to 2^18 values, each block's sums of at most 2^9 terms in sequence, give
    mean and rstd to 2^-24 * 2^10 at worst and a value a few roundings more: 1e-4 of the value and of the
    normalised scale bounds them all (the activations' slopes are below 1.13); then half a step of the type."""
    off = (got.double() - want).abs()
    lim = 1e-4 * (1 + want.abs()) * (1 if size is None else size) + UNIT[dtype] * want.abs() + (2.0 ** -24 if dtype == torch.float16 else 0)
    assert got.shape == want.shape and got.dtype == dtype, what
    assert bool((off <= lim).all()), f"{what}: {float((off / lim).max()):.3g} times the bound"
    if want.numel() > 1 and float(want.norm()):
        rel = {torch.float32: 2e-6, torch.bfloat16: 3e-3, torch.float16: 4e-4}[dtype]
        assert float(off.norm() / want.norm()) < rel, (what, float(off.norm() / want.norm()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", SHAPES)
@pytest.mark.parametrize("act", ACTS)
def test_forward_and_gradients(shape, groups, dtype, act):
    x, w, b, dy = data(shape, dtype)
    # a single value in a group is its own mean: nothing but rounding is left of it
    lonely = x[0].numel() // groups == 1
    leaves = [p.requires_grad_() for p in (x, w, b)]
    y = trnfft.group_norm(x, groups, w, b, activation=act)
    with torch.no_grad():
        assert torch.equal(y, trnfft.group_norm(x, groups, w, b, activation=act))
    xs = [p.detach().double().requires_grad_() for p in leaves]
    want = norm_ref(xs[0], groups, xs[1], xs[2], 1e-5, act)
    near(y, want, dtype, "y")
    if act == "relu":  # its slope jumps at 0: compare where 32 bits cannot be on the other side
        z = norm_ref(xs[0], groups, xs[1], xs[2], 1e-5, None).detach()
        dy = torch.where(z.abs() < 1e-3, 0, dy).to(dtype)
    got = torch.autograd.grad(y, leaves, dy)
    ref = torch.autograd.grad(want, xs, dy.double())
    rows = x.numel() // shape[-1]
    if lonely:
        assert float(got[0].abs().max()) < 1e-3
    else:
        var = xs[0].detach().reshape(shape[0], -1, groups, shape[-1] // groups).var((1, 3), unbiased=False)
        near(got[0], ref[0], dtype, "dx", size=float((var + 1e-5).rsqrt().max().clamp_min(1)) * 4)
    for name, g, r in (("dw", got[1], ref[1]), ("db", got[2], ref[2])):
        # a sum of `rows` terms of size about 1, in blocks
        off = (g.double() - r).abs().max()
        assert g.dtype == torch.float32 and float(off) <= 2e-6 * rows ** 0.5 * 40 + 1e-4, (name, float(off))
        if rows > 1 and not lonely:
            assert float((g.double() - r).norm() / r.norm()) < 3e-6, name


@pytest.mark.parametrize("dtype", DTYPES)
def test_without_parameters_and_partial_gradients(dtype):
    x, w, b, dy = data((3, 50, 24), dtype)
    near(trnfft.group_norm(x, 4), norm_ref(x.double(), 4, None, None, 1e-5, None), dtype, "bare")
    near(trnfft.group_norm(x, 4, bias=b, activation="silu"), norm_ref(x.double(), 4, None, b.double(), 1e-5, "silu"), dtype, "bias")
    near(trnfft.group_norm(x, 4, w, eps=0.5), norm_ref(x.double(), 4, w.double(), None, 0.5, None), dtype, "weight")
    leaves = [p.requires_grad_() for p in (x, w, b)]
    full = torch.autograd.grad(trnfft.group_norm(x, 4, w, b, activation="gelu"), leaves, dy)
    for i in range(3):
        args = [p if j == i else p.detach() for j, p in enumerate(leaves)]
        (one,) = torch.autograd.grad(trnfft.group_norm(args[0], 4, args[1], args[2], activation="gelu"), leaves[i], dy)
        assert torch.equal(one, full[i])
    half = [p.detach().to(torch.bfloat16).requires_grad_() for p in (w, b)]
    g = torch.autograd.grad(trnfft.group_norm(x.detach(), 4, *half), half, dy)
    assert all(p.dtype == torch.bfloat16 for p in g)


@pytest.mark.parametrize("shape,groups", [((2, 300, 64), 4), ((64, 512), 8), ((1, 60000, 32), 2)])
def test_far_mean(shape, groups):
    """A mean a thousand times the spread: differences of squares would lose the variance."""
    x, w, b, _ = data(shape, torch.float32, shift=1500.0)
    want = norm_ref(x.double(), groups, w.double(), b.double(), 1e-5, None)
    # the values themselves are rounded to 2^-24 * 1500 against a spread of 1.5, and so is the mean
    assert float((trnfft.group_norm(x, groups, w, b).double() - want).abs().max()) < 1e-3


def test_gradients_against_differences():
    x, w, b, dy = data((2, 40, 12), torch.float32)
    leaves = [p.requires_grad_() for p in (x, w, b)]
    grads = torch.autograd.grad(trnfft.group_norm(x, 3, w, b, activation="silu"), leaves, dy)
    gen = torch.Generator(device="cuda").manual_seed(3)
    for i, g in enumerate(grads):
        d = torch.randn(leaves[i].shape, device="cuda", generator=gen)
        h = 1e-4
        at = [norm_ref(*(([p.detach().double() + (e * d.double() if j == i else 0) for j, p in enumerate(leaves)])[:1]), 3,
                       *([p.detach().double() + (e * d.double() if j == i else 0) for j, p in enumerate(leaves)])[1:], 1e-5, "silu")
              for e in (h, -h)]
        want = float(((at[0] - at[1]) / (2 * h) * dy.double()).sum())
        assert abs(float((g.double() * d.double()).sum()) - want) < 1e-4 * (1 + abs(want))


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    x, w, b, dy = data((2, 31, 17, 40), dtype)
    want = trnfft.group_norm(x, 5, w, b, activation="silu")
    nchw = x.permute(0, 3, 1, 2).contiguous()
    assert torch.equal(trnfft.group_norm(nchw.permute(0, 2, 3, 1), 5, w, b, activation="silu"), want)
    odd = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape).copy_(x)
    got = trnfft.group_norm(odd, 5, w, b, activation="silu")
    near(got, norm_ref(x.double(), 5, w.double(), b.double(), 1e-5, "silu"), dtype, "off the 16-byte grid")
    x.requires_grad_()
    y = trnfft.group_norm(x, 5, w, b, activation="silu")
    (a,) = torch.autograd.grad(y.sum(), x, retain_graph=True)  # a gradient broadcast from one value
    assert torch.equal(a, torch.autograd.grad(y, x, torch.ones_like(y))[0])


def test_empty_and_bad_values():
    w = torch.ones(8, device="cuda", requires_grad=True)
    for shape in ((0, 4, 8), (3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        y = trnfft.group_norm(x, 2, w)
        assert y.shape == x.shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == x.shape and float(dw.abs().sum()) == 0
    for shape in ((4, 600, 16), (4, 16)):
        x = data(shape, torch.float32)[0]
        want = trnfft.group_norm(x, 4)
        for bad in (float("nan"), float("inf")):
            x2 = x.clone()
            x2[(1,) + (0,) * (len(shape) - 2) + (5,)] = bad
            y = trnfft.group_norm(x2, 4)
            assert bool(torch.isnan(y[1, ..., 4:8]).any())
            rest = torch.ones_like(x, dtype=torch.bool)
            rest[1, ..., 4:8] = False
            assert torch.equal(y[rest], want[rest]), "other groups and samples are untouched"
    x = torch.full((2, 50, 8), 3.25, device="cuda")
    assert float(trnfft.group_norm(x, 2).abs().max()) == 0, "a constant group"
    y = trnfft.group_norm(torch.full((2, 8), -80.0, device="cuda"), 2, bias=torch.full((8,), -200.0, device="cuda"), activation="silu")
    assert float(y.abs().max()) == 0 and bool(torch.isfinite(y).all()), "silu far below zero"


def test_repeatable_and_captured():
    x, w, b, dy = data((4, 5000, 96), torch.bfloat16)
    leaves = [p.requires_grad_() for p in (x, w, b)]

    def step():
        y = trnfft.group_norm(x, 12, w, b, activation="gelu")
        return (y.detach(), *torch.autograd.grad(y, leaves, dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first, step())), "sums in a fixed order"
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(kept, first))
    with torch.no_grad():
        x.copy_(data((4, 5000, 96), torch.bfloat16, seed=5)[0])
    graph.replay()
    assert all(torch.equal(p, q) for p, q in zip(kept, step()))


def test_cpu_tensors():
    x, w, b, _ = data((2, 10, 8), torch.float32)
    y = trnfft.group_norm(x.cpu(), 2, w.cpu(), b.cpu(), activation="gelu")
    assert not y.is_cuda and torch.equal(y, trnfft.group_norm(x, 2, w, b, activation="gelu").cpu())


def test_offsets_past_32_bits():
    n, c = (1 << 31) // 4096 + 5, 4096
    x = torch.zeros(n, c, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(c, device="cuda").bfloat16()
    y = trnfft.group_norm(x, 2)
    near(y[-1:], norm_ref(x[-1:].double(), 2, None, None, 1e-5, None), torch.bfloat16, "last row")
    assert float(y[:-1].abs().max()) == 0


@pytest.mark.parametrize("shape,groups", [
    ((64, 128), 1), ((64, 256), 1), ((64, 512), 1), ((40, 4096), 8), ((3, 20, 12), 1),  # in registers
    ((300, 30, 40), 2), ((200, 10, 1024), 1), ((5, 3, 8192), 2),                        # whole samples
    ((2, 300, 1024), 1), ((1, 5000, 1024), 4), ((2, 20000, 36), 3),                     # samples in parts
])
@pytest.mark.parametrize("what", ["value", "channel", "row"])
def test_statistics_with_one_far_start(shape, groups, what):
    """The first value, channel or row of a group far from the others: the sums of squares that start there
    lose no more than a few roundings of the variance, which is made of nothing else.

    Its relative error of e moves the result by e / 2.  Estimates of the mean up to 4 deviations off lose
    17 roundings of 2^-24 at most, and a thread's own rows their number of them, but these only of the part
    of the variance that is theirs: 2e-6, as for values without a far start."""
    x = data(shape, torch.float32, seed=4)[0].clone()
    rows = x.view(shape[0], -1, groups, shape[-1] // groups)
    {"value": rows[:, 0, :, 0], "channel": rows[..., 0], "row": rows[:, 0]}[what].add_(1000.0)
    want = norm_ref(x.double(), groups, None, None, 1e-5, None)
    off = trnfft.group_norm(x, groups).double() - want
    assert float(off.norm() / want.norm()) < 2e-6
    x.requires_grad_()
    dy = data(shape, torch.float32, seed=5)[3]
    xd = x.detach().double().requires_grad_()
    (dx,) = torch.autograd.grad(trnfft.group_norm(x, groups), x, dy)
    (wd,) = torch.autograd.grad(norm_ref(xd, groups, None, None, 1e-5, None), xd, dy.double())
    assert float((dx.double() - wd).norm() / wd.norm()) < 4e-6


def test_far_starts_leave_other_groups_as_they_are():
    """A group's result depends on its own values alone, to the last bit."""
    for shape, groups in (((64, 128), 8), ((300, 30, 40), 2), ((2, 5000, 64), 8)):
        x = data(shape, torch.float32, seed=6)[0]
        want = trnfft.group_norm(x, groups)
        y = x.clone().view(shape[0], -1, groups, shape[-1] // groups)
        y[0, 0, 1, 0] += 1e4
        got = trnfft.group_norm(y.view(shape), groups).view(y.shape)
        rest = torch.ones_like(y, dtype=torch.bool)
        rest[0, :, 1] = False
        assert torch.equal(got[rest], want.view(y.shape)[rest])


WIDE = [((2, 3, 30000), 1), ((1, 300, 26000), 26000), ((2, 7, 25700), 5), ((1, 1, 40000), 16), ((3, 40, 25800), 2)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape,groups", WIDE)
@pytest.mark.parametrize("act", ACTS)
def test_more_channels_than_shared_memory_holds(shape, groups, dtype, act):
    """The general form, forward and backward: a block's sets of the channels and groups would take more
    than 200 KB in the forward pass too."""
    assert 8 * (shape[-1] + groups) > 200 * 1024
    test_forward_and_gradients(shape, groups, dtype, act)


@pytest.mark.parametrize("shape,groups", [((2, 3, 30000), 1), ((1, 5000, 13000), 13000)])
def test_general_form_with_many_terms_and_a_far_mean(shape, groups):
    """Sums of thousands of terms by one thread, and a mean twenty times the spread, as exact as the other
    forms': the mean is kept in more than 32 bits, so what remains is the rounding of a few operations."""
    assert 8 * (shape[-1] + groups) > 200 * 1024
    x = data(shape, torch.float32, shift=30.0)[0]
    want = norm_ref(x.double(), groups, None, None, 1e-5, None)
    off = trnfft.group_norm(x, groups).double() - want
    assert float(off.norm() / want.norm()) < 3e-7
