"""Decayed linear attention (whole sequences, gradients, single tokens) against the recurrence in 64 bits."""

import math

import pytest
import torch

import trnfft_b200 as trnfft
from tests.layer_refs import decay_bound, decay_ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def rates(h, kind="mixed"):
    """log_decay of h heads: memories from 2 tokens to a thousand, or the ends of the range."""
    if kind == "mixed":
        return torch.log1p(-1.0 / torch.logspace(0.3, 3.0, h, dtype=torch.float64)).float().cuda()
    ends = {"none": 0.0, "all": -math.inf, "strong": -60.0}
    return torch.full((h,), ends[kind]).cuda()


def inputs(b, t, h, hk, dk, dv, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s, scale=1.0):
        return (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)

    return normal(b, t, h, dk), normal(b, t, hk, dk, scale=dk ** -0.5), normal(b, t, hk, dv), normal(b, t, h, dv)


def check(got, want, total, dtype, terms, what, fp32_out=False):
    off = (got.double() - want).abs()
    lim = decay_bound(dtype, terms, total, want, fp32_out)
    assert got.shape == want.shape, what
    assert bool((off <= lim).all()), f"{what}: {float((off / lim).max()):.3g} times the bound"
    norm = float(want.norm())
    # Far tighter than the worst case: roundings do not line up.  A rounding is relative to a value's
    # terms (`total`), so this holds for a norm over many values, where sums of n terms of either sign
    # have n^(1/2) of them, and not for a single value, whose terms may cancel to any degree.
    if norm and want.numel() >= 256:
        rel = {torch.float32: 1e-5, torch.bfloat16: 5e-3, torch.float16: 1e-3}[torch.float32 if fp32_out else dtype]
        assert float((got.detach().double() - want).norm()) <= rel * norm, what


def terms_of(t, dk, dv):
    return 2 * max(dk, dv) + 128 + t // 32


SIZES = [  # batch, time, heads, kv heads, dk, dv
    (1, 1, 1, 1, 1, 1),
    (2, 2, 2, 1, 5, 3),
    (1, 31, 3, 3, 16, 48),
    (2, 63, 2, 2, 32, 32),
    (1, 64, 4, 2, 64, 64),
    (2, 65, 2, 1, 40, 72),
    (1, 127, 2, 2, 128, 128),
    (1, 129, 3, 1, 128, 64),
    (1, 300, 2, 2, 64, 128),
    (3, 257, 2, 2, 33, 127),
    (1, 1500, 2, 1, 64, 64),
    (1, 700, 2, 2, 96, 100),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("carried", [False, True])
def test_prompt(size, dtype, carried):
    b, t, h, hk, dk, dv = size
    q, k, v, _ = inputs(*size, dtype)
    g = rates(h)
    first = torch.randn(b, h, dk, dv, device="cuda") if carried else None
    o, s = trnfft.decay_attention(q, k, v, g, initial_state=first, return_state=True)
    want, ws = decay_ref(q, k, v, g, dk ** -0.5, first)
    total, ts = decay_ref(q, k, v, g, dk ** -0.5, first, absolute=True)
    check(o, want, total, dtype, terms_of(t, dk, dv), "o")
    check(s, ws, ts, dtype, terms_of(t, dk, dv), "state", fp32_out=True)
    assert torch.equal(o, trnfft.decay_attention(q, k, v, g, initial_state=first)), "the state is wanted or not"


@pytest.mark.parametrize("kind", ["none", "all", "strong"])
@pytest.mark.parametrize("dtype", DTYPES)
def test_ends_of_the_decay(kind, dtype):
    size = (1, 200, 2, 2, 64, 64)
    q, k, v, do = inputs(*size, dtype)
    g = rates(2, kind)
    first = torch.randn(1, 2, 64, 64, device="cuda")
    o, s = trnfft.decay_attention(q, k, v, g, scale=0.5, initial_state=first, return_state=True)
    want, ws = decay_ref(q, k, v, g, 0.5, first)
    total, ts = decay_ref(q, k, v, g, 0.5, first, absolute=True)
    check(o, want, total, dtype, 400, "o")
    check(s, ws, ts, dtype, 400, "state", fp32_out=True)
    q.requires_grad_()
    (dq,) = torch.autograd.grad(trnfft.decay_attention(q, k, v, g), q, do)
    assert bool(torch.isfinite(dq).all())


def test_very_slow_decay_over_many_tokens():
    """The factor of a chunk is kept to more than 32 bits: thousands of them must not add up."""
    t = 20000
    q, k, v, _ = inputs(1, t, 1, 1, 32, 32, torch.float32)
    g = torch.tensor([-1.0 / 3e5]).cuda()
    o, s = trnfft.decay_attention(q, k, v, g, return_state=True)
    pos = torch.arange(t, device="cuda", dtype=torch.float64)
    w = torch.exp(g.double() * (t - 1 - pos))[:, None]
    want = (k[0, :, 0].double() * w).mT @ v[0, :, 0].double()
    assert float((s[0, 0].double() - want).norm() / want.norm()) < 2e-6
    last = q[0, -1, 0].double() @ want * 32 ** -0.5
    assert float((o[0, -1, 0].double() - last).norm() / last.norm()) < 5e-6


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("carried", [False, True])
def test_gradients(size, dtype, carried):
    b, t, h, hk, dk, dv = size
    q, k, v, do = inputs(*size, dtype, seed=1)
    g, scale = rates(h), 0.3
    first = torch.randn(b, h, dk, dv, device="cuda") if carried else None
    dlast = torch.randn(b, h, dk, dv, device="cuda") if carried else None
    leaves = [x.requires_grad_() for x in ([q, k, v, first] if carried else [q, k, v])]
    o, s = trnfft.decay_attention(q, k, v, g, scale=scale, initial_state=first, return_state=True)
    got = torch.autograd.grad((o, s) if carried else o, leaves, (do, dlast) if carried else do)

    def ref(absolute):
        f = (lambda x: x.detach().double().abs()) if absolute else (lambda x: x.detach().double())
        xs = [f(x).requires_grad_() for x in leaves]
        o, s = decay_ref(*xs[:3], g, scale, xs[3] if carried else None)
        return torch.autograd.grad((o, s) if carried else o, xs, (f(do), f(dlast)) if carried else f(do))

    for name, x, w, tot in zip(("dq", "dk", "dv", "dinitial"), got, ref(False), ref(True)):
        check(x, w, tot, dtype, terms_of(t, dk, dv) * (h // hk), name, fp32_out=name == "dinitial")


def test_gradients_against_differences():
    """o is linear in each operand, so central differences of any width are exact but for rounding."""
    q, k, v, do = inputs(1, 90, 2, 1, 16, 24, torch.float32, seed=2)
    first = torch.randn(1, 2, 16, 24, device="cuda")
    g = rates(2)
    leaves = [q, k, v, first]
    for x in leaves:
        x.requires_grad_()
    o = trnfft.decay_attention(q, k, v, g, initial_state=first)
    grads = torch.autograd.grad(o, leaves, do)
    gen = torch.Generator(device="cuda").manual_seed(5)
    for i, (x, dx) in enumerate(zip(leaves, grads)):
        d = torch.randn(x.shape, device="cuda", generator=gen)
        with torch.no_grad():
            ends = [trnfft.decay_attention(*(y + e * d if j == i else y for j, y in enumerate(leaves[:3])), g,
                                           initial_state=first + e * d if i == 3 else first) for e in (1.0, -1.0)]
        want = ((ends[0].double() - ends[1].double()) / 2 * do.double()).sum()
        size = float(do.double().norm() * ends[0].double().norm())
        assert abs(float((dx.double() * d.double()).sum() - want)) < 1e-5 * size


def test_gradients_of_some_inputs_and_of_the_state_alone():
    q, k, v, do = inputs(2, 70, 4, 2, 32, 40, torch.bfloat16)
    g = rates(4)
    for x in (q, k, v):
        x.requires_grad_()
    o, s = trnfft.decay_attention(q, k, v, g, return_state=True)
    full = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    for i, x in enumerate((q, k, v)):
        args = [y if j == i else y.detach() for j, y in enumerate((q, k, v))]
        (one,) = torch.autograd.grad(trnfft.decay_attention(*args, g), x, do)
        assert torch.equal(one, full[i])
    first = torch.zeros(2, 4, 32, 40, device="cuda", requires_grad=True)
    (di,) = torch.autograd.grad(trnfft.decay_attention(q.detach(), k.detach(), v.detach(), g, initial_state=first), first, do)
    assert float(di.abs().max()) > 0
    ds = torch.randn_like(s)
    dq, dk, dv = torch.autograd.grad(s, (q, k, v), ds)
    kd, vd = (x.detach().double().requires_grad_() for x in (k, v))
    _, sd = decay_ref(q.detach(), kd, vd, g, 1.0)
    wk, wv = torch.autograd.grad(sd, (kd, vd), ds.double())
    assert float(dq.abs().max()) == 0
    assert float((dk.double() - wk).norm() / wk.norm()) < 5e-3 and float((dv.double() - wv).norm() / wv.norm()) < 5e-3
    # a gradient that is one value broadcast
    o = trnfft.decay_attention(q, k, v, g)
    a = torch.autograd.grad(o.sum(), q, retain_graph=True)[0]
    assert torch.equal(a, torch.autograd.grad(o, q, torch.ones_like(o))[0])
    with pytest.raises(RuntimeError):  # differentiable once only
        o = trnfft.decay_attention(q, k, v, g)
        d1 = torch.autograd.grad(o.sum(), q, create_graph=True)[0]
        torch.autograd.grad(d1.sum(), k)


LENGTHS = [
    ([5], 0, 0),
    ([0], 0, 0),
    ([1, 0, 64, 63, 65, 0, 300, 2], 0, 3),
    ([128, 128, 1], 4, 0),
    ([700, 1, 90], 7, 9),
    ([0, 0, 0], 3, 2),
    ([0, 0], 0, 0),          # no rows at all
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lengths,before,behind", LENGTHS)
def test_packed(lengths, before, behind, dtype):
    h, hk, dk, dv = 4, 2, 48, 64
    total = before + sum(lengths) + behind
    q, k, v, do = inputs(1, total, h, hk, dk, dv, dtype, seed=3)
    g, n = rates(h), len(lengths)
    cu = torch.tensor([before, *lengths]).cumsum(0).cuda()
    first, dlast = (torch.randn(n, h, dk, dv, device="cuda") for _ in range(2))
    leaves = [x.requires_grad_() for x in (q, k, v, first)]
    for c in (cu, cu.int()):
        o, s = trnfft.decay_attention(q, k, v, g, initial_state=first, cu_seqlens=c, return_state=True)
    got = torch.autograd.grad((o, s), leaves, (do, dlast))
    outside = torch.ones(total, dtype=torch.bool, device="cuda")
    for i, (x, y) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        outside[x:y] = False
        xs = [z.detach()[:, x:y].double().requires_grad_() for z in (q, k, v)] + [first.detach()[i:i + 1].double().requires_grad_()]
        wo, ws = decay_ref(*xs[:3], g, dk ** -0.5, xs[3])
        ab = [z.detach().abs().requires_grad_() for z in xs]
        to, ts = decay_ref(*ab[:3], g, dk ** -0.5, ab[3])
        terms = terms_of(y - x, dk, dv)
        check(o[:, x:y], wo.detach(), to.detach(), dtype, terms, f"o of {i}")
        check(s[i:i + 1], ws.detach(), ts.detach(), dtype, terms, f"state of {i}", fp32_out=True)
        if x == y:
            assert torch.equal(got[3][i], dlast[i])
            continue
        wg = torch.autograd.grad((wo, ws), xs, (do[:, x:y].double(), dlast[i:i + 1].double()))
        tg = torch.autograd.grad((to, ts), ab, (do[:, x:y].double().abs(), dlast[i:i + 1].double().abs()))
        for name, z, w, t in zip(("dq", "dk", "dv"), got, wg, tg):
            check(z[:, x:y], w, t, dtype, 2 * terms, f"{name} of {i}")
        check(got[3][i:i + 1], wg[3], tg[3], dtype, terms, f"dinitial of {i}", fp32_out=True)
    for z in (o.detach(), *got[:3]):
        assert float(z[:, outside].abs().sum()) == 0, "rows of no sequence are zero"


@pytest.mark.parametrize("dtype", DTYPES)
def test_packed_graph_follows_the_lengths(dtype):
    """A captured call reads the lengths where they are: a buffer of many rows, few of them used, others each time."""
    rows, h, d = 1500, 2, 64
    q, k, v, _ = inputs(1, rows, h, h, d, d, dtype, seed=12)
    g = rates(h)
    cu = torch.tensor([0, 700, 701, 1400], device="cuda", dtype=torch.int32)
    first = torch.randn(3, h, d, d, device="cuda")

    def call(c):
        with torch.no_grad():
            return trnfft.decay_attention(q, k, v, g, initial_state=first, cu_seqlens=c, return_state=True)

    call(cu)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, s = call(cu)
    for ends in ([0, 700, 701, 1400], [0, 3, 3, 10], [0, 0, 1500, 1500], [5, 64, 128, 1000]):
        cu.copy_(torch.tensor(ends, dtype=torch.int32))
        graph.replay()
        wo, ws = call(torch.tensor(ends, device="cuda"))
        assert torch.equal(o, wo) and torch.equal(s, ws), ends


def test_two_streams_and_inference_mode():
    """Calls that run at once, each with workspaces of its own; states made in inference mode."""
    g = rates(4)
    sets = [inputs(1, 6000, 4, 4, 64, 64, t, seed=13)[:3] for t in DTYPES]
    want = [trnfft.decay_attention(*x, g, return_state=True) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[] for _ in sets]
    for _ in range(5):
        for s, x, keep in zip(streams, sets, got):
            with torch.cuda.stream(s):
                keep.append(trnfft.decay_attention(*x, g, return_state=True))
    torch.cuda.synchronize()
    for keep, w in zip(got, want):
        assert all(torch.equal(o, w[0]) and torch.equal(s, w[1]) for o, s in keep)
    with torch.inference_mode():
        q, k, v = (x[:, -1] for x in sets[0])
        state = torch.zeros(1, 4, 64, 64, device="cuda")
        o, new = trnfft.decay_attention_step(q, k, v, g, state)
    assert new is state and bool(torch.isfinite(o).all()) and float(state.abs().max()) > 0


def test_packed_of_no_sequence():
    q, k, v, _ = inputs(1, 9, 2, 2, 16, 16, torch.float32)
    cu = torch.tensor([4], dtype=torch.int32, device="cuda")
    o, s = trnfft.decay_attention(q, k, v, rates(2), cu_seqlens=cu, return_state=True)
    assert s.shape == (0, 2, 16, 16) and float(o.abs().sum()) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts_and_alignment(dtype):
    """Any order of the dimensions, gaps, broadcast heads and addresses off the 16-byte grid."""
    b, t, h, hk, dk, dv = 2, 130, 4, 2, 64, 64
    q, k, v, do = inputs(b, t, h, hk, dk, dv, dtype, seed=4)
    g = rates(h)
    want = trnfft.decay_attention(q, k, v, g)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    assert torch.equal(trnfft.decay_attention(*heads_first, g), want)
    joined = torch.cat([q, k, v], 2)
    assert torch.equal(trnfft.decay_attention(joined[:, :, :h], joined[:, :, h:h + hk], joined[:, :, h + hk:], g), want)
    shifted = []
    for x in (q, k, v):
        y = torch.empty(x.numel() + 1, dtype=dtype, device="cuda")[1:].view(x.shape)
        shifted.append(y.copy_(x))
    exact, _ = decay_ref(q, k, v, g, dk ** -0.5)
    total, _ = decay_ref(q, k, v, g, dk ** -0.5, absolute=True)
    check(trnfft.decay_attention(*shifted, g), exact, total, dtype, terms_of(t, dk, dv), "off the 16-byte grid")
    gaps = [torch.nn.functional.pad(x, (1, 2))[..., 1:-2] for x in (q, k, v)]
    check(trnfft.decay_attention(*gaps, g), exact, total, dtype, terms_of(t, dk, dv), "rows at odd distances")
    inner = [x.transpose(-1, -2).contiguous().transpose(-1, -2) for x in (q, k, v)]
    assert torch.equal(trnfft.decay_attention(*inner, g), want)
    k1, v1 = k[:, :, :1].expand(-1, -1, hk, -1), v[:, :1].expand(-1, t, -1, -1)
    assert torch.equal(trnfft.decay_attention(q, k1, v1, g), trnfft.decay_attention(q, k1.contiguous(), v1.contiguous(), g))
    q.requires_grad_()
    o = trnfft.decay_attention(q, k, v, g)
    do2 = do.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(torch.autograd.grad(o, q, do2, retain_graph=True)[0], torch.autograd.grad(o, q, do)[0])


@pytest.mark.parametrize("dtype", DTYPES)
def test_continued_sequences_and_single_tokens(dtype):
    """A sequence in one call, in two, and token by token."""
    b, t, h, hk, dk, dv = 2, 150, 4, 2, 40, 56
    q, k, v, _ = inputs(b, t, h, hk, dk, dv, dtype, seed=6)
    g = rates(h)
    want, ws = decay_ref(q, k, v, g, dk ** -0.5)
    total, ts = decay_ref(q, k, v, g, dk ** -0.5, absolute=True)
    o1, s = trnfft.decay_attention(q[:, :77], k[:, :77], v[:, :77], g, return_state=True)
    o2, s = trnfft.decay_attention(q[:, 77:], k[:, 77:], v[:, 77:], g, initial_state=s, return_state=True)
    terms = 2 * terms_of(t, dk, dv)
    check(torch.cat([o1, o2], 1), want, total, dtype, terms, "two calls")
    check(s, ws, ts, dtype, terms, "state of two calls", fp32_out=True)
    pool = torch.randn(b, 3, h, dk, dv, device="cuda")
    state = pool[:, 1].zero_()
    others = pool[:, ::2].clone()
    rows = []
    for i in range(t):
        o, got = trnfft.decay_attention_step(q[:, i], k[:, i], v[:, i], g, state)
        assert got is state
        rows.append(o)
    check(torch.stack(rows, 1), want, total, dtype, terms + t, "token by token")
    check(state, ws, ts, dtype, terms + t, "state token by token", fp32_out=True)
    assert torch.equal(pool[:, ::2], others)


@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (3, 4, 2, 5, 7), (2, 2, 1, 64, 64), (5, 8, 4, 40, 72), (70, 2, 2, 128, 128),
                                  (2, 3, 3, 127, 33), (300, 4, 1, 32, 96), (1, 2, 2, 128, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step(size, dtype):
    b, h, hk, dk, dv = size
    q, k, v, _ = (x[:, 0] for x in inputs(b, 1, h, hk, dk, dv, dtype, seed=7))
    g = rates(h)
    state = torch.randn(b, h, dk, dv, device="cuda")
    want, ws = decay_ref(q[:, None], k[:, None], v[:, None], g, 0.7, state)
    total, ts = decay_ref(q[:, None], k[:, None], v[:, None], g, 0.7, state, absolute=True)
    kept, new = state.clone(), torch.full_like(state, float("nan"))
    o, got = trnfft.decay_attention_step(q, k, v, g, state, scale=0.7, new_state=new)
    assert got is new and torch.equal(state, kept)
    check(o, want[:, 0], total[:, 0], dtype, dk + 8, "o")
    check(new, ws, ts, dtype, 4, "state", fp32_out=True)
    o2, _ = trnfft.decay_attention_step(q, k, v, g, state, scale=0.7)
    assert torch.equal(o, o2) and torch.equal(state, new)
    wide = torch.empty(b, 2 * h * dk * dv + 1, device="cuda")[:, 1:1 + h * dk * dv].view(b, h, dk, dv)  # off the 16-byte grid
    wide.copy_(kept)
    o3, _ = trnfft.decay_attention_step(q, k, v, g, wide, scale=0.7)
    assert float((o3.double() - o.double()).abs().max()) <= float(decay_bound(dtype, dk + 8, total[:, 0], want[:, 0]).max())
    check(wide, ws, ts, dtype, 4, "state", fp32_out=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("t,b,h", [(5000, 1, 1), (9001, 1, 3), (3000, 2, 5)])
def test_long_sequences_in_segments(t, b, h, dtype):
    """Few heads and a long axis: the sequences are cut, forwards and backwards."""
    d = 32
    q, k, v, do = inputs(b, t, h, h, d, d, dtype, seed=11)
    g = rates(h)
    first, dlast = (torch.randn(b, h, d, d, device="cuda") for _ in range(2))
    leaves = [x.requires_grad_() for x in (q, k, v, first)]
    o, s = trnfft.decay_attention(q, k, v, g, initial_state=first, return_state=True)
    got = torch.autograd.grad((o, s), leaves, (do, dlast))
    xs = [x.detach().double().requires_grad_() for x in leaves]
    pos = torch.arange(t, device="cuda", dtype=torch.float64)
    behind = pos[:, None] - pos
    w = torch.exp(g.double()[:, None, None] * behind.clamp_min(0)) * (behind >= 0)
    qd, kd, vd = (x.transpose(1, 2) for x in xs[:3])
    ahead = torch.exp(g.double()[:, None] * (pos + 1))[None, :, :, None]
    wo = ((qd @ kd.mT * w) @ vd + (qd @ xs[3]) * ahead) * d ** -0.5
    left = torch.exp(g.double()[:, None] * (t - 1 - pos))[None, :, :, None]
    ws = (kd * left).mT @ vd + xs[3] * torch.exp(g.double() * t)[:, None, None]
    wg = torch.autograd.grad((wo.transpose(1, 2), ws), xs, (do.double(), dlast.double()))
    rel = {torch.float32: 3e-6, torch.bfloat16: 5e-3, torch.float16: 1e-3}
    for name, x, y in zip(("o", "state", "dq", "dk", "dv", "dinitial"), (o, s, *got), (wo.transpose(1, 2), ws, *wg)):
        off = float((x.detach().double() - y).norm() / y.norm())
        assert off < rel[torch.float32 if name in ("state", "dinitial") else dtype], (name, off)


def test_step_refuses_overlap():
    s = torch.zeros(3, 2, 8, 8, device="cuda")
    q = torch.zeros(2, 2, 8, device="cuda")
    with pytest.raises(ValueError, match="overlaps"):
        trnfft.decay_attention_step(q, q, q, torch.zeros(2).cuda(), s[:2], new_state=s[1:])
    kept = torch.ones(2, 2, 8, 8, device="cuda", requires_grad=True) * 1.0
    loss = (kept * kept).sum()
    with torch.no_grad():
        trnfft.decay_attention_step(q, q, q, torch.zeros(2).cuda(), kept)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        loss.backward()


def test_empty_calls():
    q, k, v, _ = inputs(2, 0, 2, 2, 8, 8, torch.float32)
    first = torch.randn(2, 2, 8, 8, device="cuda", requires_grad=True)
    o, s = trnfft.decay_attention(q, k, v, rates(2), initial_state=first, return_state=True)
    assert o.shape == (2, 0, 2, 8) and torch.equal(s, first)
    (d,) = torch.autograd.grad(s, first, torch.ones_like(s))
    assert torch.equal(d, torch.ones_like(s))
    _, s = trnfft.decay_attention(q, k, v, rates(2), return_state=True)
    assert float(s.abs().sum()) == 0
    q, k, v, _ = inputs(0, 5, 2, 2, 8, 8, torch.float32)
    o, s = trnfft.decay_attention(q, k, v, rates(2), return_state=True)
    assert o.shape == (0, 5, 2, 8) and s.shape == (0, 2, 8, 8)
    o, s = trnfft.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], rates(2), s)
    assert o.shape == (0, 2, 8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 40])
def test_other_values_stay_in_their_rows(dtype, d):
    """NaN and infinity at one token reach that token and later ones of its head and sequence, nothing else."""
    q, k, v, _ = inputs(2, 200, 2, 2, d, d, dtype)
    g = rates(2)
    want = trnfft.decay_attention(q, k, v, g)
    for bad in (float("nan"), float("inf")):
        v2 = v.clone()
        v2[1, 100, 0] = bad
        o = trnfft.decay_attention(q, k, v2, g)
        assert torch.equal(o[0], want[0]) and torch.equal(o[1, :, 1], want[1, :, 1])
        assert not bool(torch.isfinite(o[1, 100:, 0]).any()), "the state keeps it"
        assert bool(torch.isfinite(o[1, :100, 0]).all()), "a token's value reaches no row before it"
        assert float((o[1, :100, 0].float() - want[1, :100, 0].float()).abs().max()) <= 0.02 * float(want.float().abs().max())
        packed = trnfft.decay_attention(*(x.reshape(1, 400, 2, d) for x in (q, k, v2)), g,
                                        cu_seqlens=torch.tensor([0, 150, 290, 310, 400], device="cuda"))
        assert bool(torch.isfinite(packed[0, :290]).all()) and bool(torch.isfinite(packed[0, 310:]).all())


def test_cpu_tensors_and_devices():
    q, k, v, _ = inputs(1, 20, 2, 2, 16, 16, torch.float32)
    g = rates(2)
    want, ws = trnfft.decay_attention(q, k, v, g, return_state=True)
    o, s = trnfft.decay_attention(q.cpu(), k.cpu(), v.cpu(), g.cpu(), return_state=True)
    assert not o.is_cuda and not s.is_cuda and torch.equal(o, want.cpu()) and torch.equal(s, ws.cpu())
    state = ws.cpu()
    o, got = trnfft.decay_attention_step(q[:, 0].cpu(), k[:, 0].cpu(), v[:, 0].cpu(), g.cpu(), state)
    o2, s2 = trnfft.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, ws)
    assert got is state and torch.equal(o, o2.cpu()) and torch.equal(state, s2.cpu())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_streams_and_graphs(dtype):
    """A captured training step, replayed on new values, beside eager ones on another stream."""
    size = (2, 400, 4, 2, 64, 64)
    q, k, v, do = inputs(*size, dtype, seed=8)
    g = rates(4)
    for x in (q, k, v):
        x.requires_grad_()

    def step():
        o, s = trnfft.decay_attention(q, k, v, g, return_state=True)
        return (o.detach(), s.detach(), *torch.autograd.grad(o, (q, k, v), do))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = step()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(kept, eager))
    with torch.no_grad():
        for x, y in zip((q, k, v, do), inputs(*size, dtype, seed=9)):
            x.copy_(y)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(kept, step()))


def test_two_graphs_do_not_share_workspaces():
    g = rates(2)
    sets = [inputs(1, 3000, 2, 2, 64, 64, torch.float32, seed=s)[:3] for s in (1, 2)]
    want = [trnfft.decay_attention(*x, g, return_state=True) for x in sets]
    graphs, got = [], []
    for x in sets:
        trnfft.decay_attention(*x, g)
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(trnfft.decay_attention(*x, g, return_state=True))
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, x in zip(streams, graphs):
            with torch.cuda.stream(s):
                x.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_offsets_past_32_bits():
    """Strides that lead more than 2^31 elements away."""
    t, far = 70, (1 << 31) + 64
    q, k, v, _ = inputs(2, t, 1, 1, 64, 64, torch.bfloat16, seed=10)
    want = trnfft.decay_attention(q, k, v, rates(1))
    pool = torch.empty(far + t * 64, dtype=torch.bfloat16, device="cuda")
    views = []
    y = torch.as_strided(pool, q.shape, (far, 64, 64, 1))
    y.copy_(q)
    views.append(y)
    assert torch.equal(trnfft.decay_attention(y, k, v, rates(1)), want)
    y.copy_(v)
    assert torch.equal(trnfft.decay_attention(q, k, y, rates(1)), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [(1, 1500, 2, 1, 64, 64), (2, 300, 2, 2, 128, 128), (2, 257, 4, 2, 40, 72), (1, 4096, 1, 1, 33, 30)])
def test_sixteen_bit_results_lose_their_own_rounding_alone(size, dtype):
    """o and the gradients are as far from 64 bits as those rounded to the type are.

    P and C enter the products in two parts (2^-16 of them at worst) and sums are of 32 bits, so an error
    of some 2^-16 of the result joins the rounding's, which is at least 2^-13 of it in the mean: less than
    1 % more in the root of the sum of squares.  P and C in the type's own 11 bits would give 41 % more."""
    b, t, h, hk, dk, dv = size
    q, k, v, do = inputs(*size, dtype, seed=20)
    g = rates(h)
    first = torch.randn(b, h, dk, dv, device="cuda")
    leaves = [x.requires_grad_() for x in (q, k, v)]
    o = trnfft.decay_attention(q, k, v, g, initial_state=first)
    got = (o, *torch.autograd.grad(o, leaves, do))
    xs = [x.detach().double().requires_grad_() for x in leaves]
    wo, _ = decay_ref(*xs, g, dk ** -0.5, first)
    for name, x, w in zip(("o", "dq", "dk", "dv"), got, (wo, *torch.autograd.grad(wo, xs, do.double()))):
        w = w.detach()
        rounding = float((w.to(dtype).double() - w).norm())
        assert float((x.detach().double() - w).norm()) < 1.02 * rounding, name


def same_infinities(got, want, rel, what):
    """Infinite where the 64-bit form is, with its sign; near it elsewhere; nowhere NaN."""
    got, inf = got.detach().double(), want.isinf()
    assert not bool(want.isnan().any()), "the case has no NaN"
    assert torch.equal(got.isinf(), inf) and not bool(got.isnan().any()), what
    assert torch.equal(got[inf], want[inf]), what
    assert float((got[~inf] - want[~inf]).norm()) <= rel * float(want[~inf].norm()), what


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [33, 40, 64, 128])
@pytest.mark.parametrize("t", [1, 200, 3000])
def test_infinite_states_stay_infinite(dtype, d, t):
    """An infinite element of a state, or one that an infinite key makes, stays infinite however it decays."""
    q, k, v, do = inputs(1, t, 3, 3, d, d, dtype, seed=25)
    g = torch.tensor([-0.1, 0.0, -60.0]).cuda()
    rel = {torch.float32: 1e-5, torch.bfloat16: 5e-3, torch.float16: 1e-3}[dtype]
    first = torch.randn(1, 3, d, d, device="cuda")
    first[0, :, 1, 2] = math.inf
    first[0, :, 4, 0] = -math.inf
    o, s = trnfft.decay_attention(q, k, v, g, initial_state=first, return_state=True)
    want, ws = decay_ref(q, k, v, g, d ** -0.5, first)
    same_infinities(s, ws, 1e-5, "state of an infinite state")
    same_infinities(o, want, rel, "o of an infinite state")
    state = first.clone()
    o1, _ = trnfft.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)
    w1, ws1 = decay_ref(q[:, :1], k[:, :1], v[:, :1], g, d ** -0.5, first)
    same_infinities(state, ws1, 1e-5, "state of a step")
    same_infinities(o1, w1[:, 0], rel, "o of a step")
    k2 = k.clone()
    k2[0, t // 2, 0, 3], k2[0, t // 2, 1:, 5] = math.inf, -math.inf
    o, s = trnfft.decay_attention(q, k2, v, g, return_state=True)
    want, ws = decay_ref(q, k2, v, g, d ** -0.5)
    same_infinities(s, ws, 1e-5, "state of an infinite key")
    same_infinities(o, want, rel, "o of an infinite key")
    one = torch.zeros(1, 3, d, d, device="cuda", requires_grad=True)
    dlast = torch.randn_like(one)
    dlast[0, :, 2, 3] = math.inf
    _, s = trnfft.decay_attention(q, k, v, g, initial_state=one, return_state=True)
    (di,) = torch.autograd.grad(s, one, dlast)
    same_infinities(di, dlast.double() * torch.exp(g.double() * t).clamp_min(1e-300)[:, None, None], 1e-5, "gradient of the state")


def test_step_between_two_buffers_of_one_pool():
    """Old and new states of the streams side by side, each stream's in turn: they interleave, and do not overlap."""
    b, h, dk, dv = 5, 2, 8, 12
    q, k, v, _ = (x[:, 0] for x in inputs(b, 1, h, h, dk, dv, torch.float32, seed=26))
    g = rates(h)
    pool = torch.randn(b, 3, h, dk, dv, device="cuda")
    kept = pool.clone()
    want, ws = trnfft.decay_attention_step(q, k, v, g, pool[:, 0].contiguous())
    for old, new in ((0, 1), (0, 2), (1, 0), (2, 1)):
        pool.copy_(kept)
        pool[:, old] = kept[:, 0]
        o, got = trnfft.decay_attention_step(q, k, v, g, pool[:, old], new_state=pool[:, new])
        assert torch.equal(o, want) and torch.equal(got, ws) and torch.equal(pool[:, old], kept[:, 0])
        third = 3 - old - new
        assert torch.equal(pool[:, third], kept[:, third])
    one = h * dk * dv
    flat = pool.view(-1)
    for off in (1, one - 1, 2 * one + 1, 3 * one - 1, 3 * one):
        shifted = torch.as_strided(flat, (b - 1, h, dk, dv), (3 * one, dk * dv, dv, 1), off)
        with pytest.raises(ValueError, match="overlaps"):
            trnfft.decay_attention_step(q[:-1], k[:-1], v[:-1], g, pool[:-1, 0], new_state=shifted)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_nan_decay_is_not_hidden(dtype):
    """A head whose log_decay is NaN has no number in its state or, from a carried state, in its outputs."""
    q, k, v, _ = inputs(1, 70, 3, 3, 64, 64, dtype, seed=27)
    g = rates(3)
    first = torch.randn(1, 3, 64, 64, device="cuda")
    want, ws = trnfft.decay_attention(q, k, v, g, initial_state=first, return_state=True)
    g[1] = math.nan
    o, s = trnfft.decay_attention(q, k, v, g, initial_state=first, return_state=True)
    assert bool(s[:, 1].isnan().all()) and bool(o[:, :, 1].isnan().all())
    assert torch.equal(o[:, :, ::2], want[:, :, ::2]) and torch.equal(s[:, ::2], ws[:, ::2])
    state = first.clone()
    o, _ = trnfft.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)
    assert bool(state[:, 1].isnan().all()) and bool(o[:, 1].isnan().all())
    assert bool(torch.isfinite(state[:, ::2]).all()) and bool(torch.isfinite(o[:, ::2]).all())
