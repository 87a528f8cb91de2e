"""The bfloat16 walk on the tensor cores at every width: segments, packed rows, rows that no tensor map
describes, and values that are not finite, each with its gradients."""

import math

import pytest
import torch

import trnfft_b200 as trnfft
from trnfft_b200 import _attention, _lib
from tests.layer_refs import decay_ref
from tests.test_gpu_decay_attention import check, inputs, rates, terms_of

pytestmark = pytest.mark.gpu

WIDTHS = [(64, 64), (128, 128), (64, 128), (128, 72), (96, 40)]


def segmented(q, k, v, cu=None, nseq=None, backward=0):
    """Whether the call cuts its sequences: the work area then holds a state for each of several segments."""
    nseq = q.shape[0] if nseq is None else nseq
    shape = _attention._shape(q, k, v, (0, 0, 0), cu, nseq, 1.0)
    bytes_ = _lib.load().trnfft_decay_attention_work_bytes(shape, backward)
    return bytes_ > 4 * nseq * q.shape[2] * q.shape[3] * v.shape[3]


def gradients(q, k, v, g, do, first=None, dlast=None, **kw):
    leaves = [x.detach().requires_grad_() for x in ((q, k, v) if first is None else (q, k, v, first))]
    o, s = trnfft.decay_attention(*leaves[:3], g, initial_state=leaves[3] if first is not None else None, return_state=True, **kw)
    outs, grads = ((o, s), (do, dlast)) if dlast is not None else ((o,), (do,))
    return (o.detach(), s.detach(), *torch.autograd.grad(outs, leaves, grads))


def by_definition(q, k, v, g, do, first, dlast, absolute=False):
    """The same in 64 bits by sums over all pairs of tokens."""
    f = (lambda x: x.detach().double().abs()) if absolute else (lambda x: x.detach().double())
    xs = [f(x).requires_grad_() for x in (q, k, v, first)]
    t, group = q.shape[1], q.shape[2] // k.shape[2]
    pos = torch.arange(t, device="cuda", dtype=torch.float64)
    behind, rate = pos[:, None] - pos, g.double()
    w = torch.exp(rate[:, None, None] * behind.clamp_min(0)) * (behind >= 0)
    qd, kd, vd = xs[0].transpose(1, 2), *(x.transpose(1, 2).repeat_interleave(group, 1) for x in xs[1:3])
    ahead = torch.exp(rate[:, None] * (pos + 1))[None, :, :, None]
    o = (((qd @ kd.mT * w) @ vd + (qd @ xs[3]) * ahead) * q.shape[3] ** -0.5).transpose(1, 2)
    left = torch.exp(rate[:, None] * (t - 1 - pos))[None, :, :, None]
    s = (kd * left).mT @ vd + xs[3] * torch.exp(rate * t)[:, None, None]
    return (o.detach(), s.detach(), *torch.autograd.grad((o, s), xs, (f(do), f(dlast))))


NAMES = ("o", "state", "dq", "dk", "dv", "dinitial")


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("b,t,h,hk", [(1, 6001, 1, 1), (1, 3000, 4, 2), (2, 2500, 3, 3)])
def test_segments(b, t, h, hk, dk, dv):
    q, k, v, do = inputs(b, t, h, hk, dk, dv, torch.bfloat16, seed=21)
    g = rates(h)
    assert segmented(q, k, v) and (h != hk or segmented(q, k, v, backward=1))
    first, dlast = (torch.randn(b, h, dk, dv, device="cuda") for _ in range(2))
    got = gradients(q, k, v, g, do, first, dlast)
    args = (q, k, v, g, do, first, dlast)
    for name, x, w, total in zip(NAMES, got, by_definition(*args), by_definition(*args, absolute=True)):
        check(x, w, total, torch.bfloat16, terms_of(t, dk, dv) * (h // hk), name, fp32_out=name in ("state", "dinitial"))


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("lengths,before,behind,cut", [
    ([1, 0, 64, 127, 128, 129, 0, 300, 2], 0, 3, False),
    ([700, 1, 90], 7, 9, False),
    ([4000, 0, 129, 700], 5, 2, True),
])
def test_packed(lengths, before, behind, cut, dk, dv):
    h, hk = (1, 1) if cut else (4, 2)
    total, n = before + sum(lengths) + behind, len(lengths)
    q, k, v, do = inputs(1, total, h, hk, dk, dv, torch.bfloat16, seed=22)
    g = rates(h)
    cu = torch.tensor([before, *lengths]).cumsum(0).cuda()
    assert not cut or segmented(q, k, v, cu, n)
    first, dlast = (torch.randn(n, h, dk, dv, device="cuda") for _ in range(2))
    got = gradients(q, k, v, g, do, first, dlast, cu_seqlens=cu)
    outside = torch.ones(total, dtype=torch.bool, device="cuda")
    for i, (x, y) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        outside[x:y] = False
        if x == y:
            assert torch.equal(got[5][i], dlast[i]) and torch.equal(got[1][i], first[i])
            continue
        args = (q[:, x:y], k[:, x:y], v[:, x:y], g, do[:, x:y], first[i:i + 1], dlast[i:i + 1])
        for name, z, w, tot in zip(NAMES, got, by_definition(*args), by_definition(*args, absolute=True)):
            z = z[i:i + 1] if name in ("state", "dinitial") else z[:, x:y]
            check(z, w, tot, torch.bfloat16, terms_of(y - x, dk, dv) * (h // hk), f"{name} of {i}",
                  fp32_out=name in ("state", "dinitial"))
    for z in (got[0], *got[2:5]):
        assert float(z[:, outside].abs().sum()) == 0, "rows of no sequence are zero"


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("t", [300, 5000])
def test_rows_that_no_tensor_map_describes(t, dk, dv):
    """Heads, tokens or sequences that share their rows: loaded row by row, with the values of the copy."""
    b, h, hk = 2, 2, 2
    q, k, v, do = inputs(b, t, h, hk, dk, dv, torch.bfloat16, seed=23)
    g = rates(h)
    k, v = k[:, :, :1].expand(-1, -1, hk, -1), v[:1, :1].expand(b, t, -1, -1)
    want = gradients(q, k.contiguous(), v.contiguous(), g, do)
    got = gradients(q, k, v, g, do)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dk,dv", WIDTHS)
@pytest.mark.parametrize("t", [200, 4000])
@pytest.mark.parametrize("where", ["q", "k", "v", "first"])
def test_bad_values_reach_their_own_rows_alone(where, t, dk, dv):
    """NaN and infinity in one operand, in one call and in segments: outputs and gradients that the sums
    do not lead to stay as they were, to a rounding (their rows are taken by the other walk)."""
    q, k, v, do = inputs(1, t, 2, 2, dk, dv, torch.bfloat16, seed=24)
    g = rates(2)
    first, dlast = (torch.randn(1, 2, dk, dv, device="cuda") for _ in range(2))
    want = dict(zip(NAMES, gradients(q, k, v, g, do, first, dlast)))
    at = t * 5 // 8
    for bad in (math.nan, math.inf):
        args = dict(q=q.clone(), k=k.clone(), v=v.clone(), first=first.clone())
        if where == "first":
            args["first"][0, 0, 1] = bad
        else:
            args[where][0, at, 0] = bad
        got = dict(zip(NAMES, gradients(args["q"], args["k"], args["v"], g, do, args["first"], dlast)))
        # what stays: (name, tokens) of head 0
        stay = {"q": [("o", slice(0, at)), ("o", slice(at + 1, t)), ("dk", slice(at + 1, t)), ("dv", slice(at + 1, t)),
                      ("dq", slice(0, t))],
                "k": [("o", slice(0, at)), ("dq", slice(0, at)), ("dk", slice(0, t)), ("dv", slice(0, at)),
                      ("dv", slice(at + 1, t))],
                "v": [("o", slice(0, at)), ("dq", slice(0, at)), ("dv", slice(0, t)), ("dk", slice(0, at)),
                      ("dk", slice(at + 1, t))],
                "first": [("dk", slice(0, t)), ("dv", slice(0, t))]}[where]
        for name in NAMES:
            x, y = got[name], want[name]
            other = (slice(None), 1) if name in ("state", "dinitial") else (slice(None), slice(None), 1)
            assert torch.equal(x[other], y[other]), f"{name}: the other head"
        for name, rows in stay:
            x, y = got[name][:, rows, 0].double(), want[name][:, rows, 0].double()
            assert bool(torch.isfinite(x).all()), (name, rows)
            assert float((x - y).norm()) <= 5e-3 * float(y.norm()), (name, rows)
        reach = {"q": ("o", at), "k": ("o", t - 1), "v": ("o", t - 1), "first": ("o", 0)}[where]
        assert not bool(torch.isfinite(got[reach[0]][:, reach[1], 0]).any()), "the rows that it does reach"
