"""Argument checks of the sequence and normalisation operators, without a GPU."""

import ctypes
import pathlib
import re

import pytest
import torch

import trnfft_b200 as trnfft
from trnfft_b200 import _lib
from trnfft_b200.nn import ComplexDecayAttention, ComplexGroupNorm, GroupNorm


def qkv(b=2, t=3, h=4, hk=2, dk=8, dv=6, dtype=torch.float32):
    return (torch.zeros(b, t, h, dk, dtype=dtype), torch.zeros(b, t, hk, dk, dtype=dtype),
            torch.zeros(b, t, hk, dv, dtype=dtype), torch.zeros(h))


@pytest.mark.parametrize("change,match", [
    (lambda q, k, v, g: (q[0], k, v, g), "must be"),
    (lambda q, k, v, g: (q.double(), k.double(), v.double(), g), "share one of"),
    (lambda q, k, v, g: (q, k.bfloat16(), v, g), "share one of"),
    (lambda q, k, v, g: (q, k[:, :2], v, g), "belong together"),
    (lambda q, k, v, g: (q, k[..., :7], v, g), "belong together"),
    (lambda q, k, v, g: (q[:1], k, v, g), "belong together"),
    (lambda q, k, v, g: (q[:, :, :3], k, v, g), "multiple"),
    (lambda q, k, v, g: (q, k[:, :, :0], v[:, :, :0], g), "multiple"),
    (lambda q, k, v, g: (q[..., :0], k[..., :0], v, g), "positive"),
    (lambda q, k, v, g: (q, k, v, g[:3]), "log_decay"),
    (lambda q, k, v, g: (q, k, v, g.long()), "log_decay"),
    (lambda q, k, v, g: (q, k, v, g.requires_grad_()), "no gradient"),
])
def test_attention_refuses(change, match):
    with pytest.raises(ValueError, match=match):
        trnfft.decay_attention(*change(*qkv()))


@pytest.mark.parametrize("more,match", [
    (dict(initial_state=torch.zeros(2, 4, 8, 5)), "initial_state"),
    (dict(initial_state=torch.zeros(2, 4, 8, 6).bfloat16()), "initial_state"),
    (dict(cu_seqlens=torch.zeros(3, dtype=torch.int32)), "batch 1"),
    (dict(cu_seqlens=torch.zeros(3)), "int32 or int64"),
    (dict(cu_seqlens=torch.zeros(0, dtype=torch.int32)), "int32 or int64"),
])
def test_attention_refuses_states_and_lengths(more, match):
    with pytest.raises(ValueError, match=match):
        trnfft.decay_attention(*qkv(), **more)


def test_step_refuses():
    q, k, v, g = qkv()
    q, k, v = q[:, 0], k[:, 0], v[:, 0]
    s = torch.zeros(2, 4, 8, 6)
    for bad in (torch.zeros(2, 4, 8, 5), s.bfloat16(), s[:1], s.transpose(2, 3).contiguous().transpose(2, 3)):
        with pytest.raises(ValueError, match="state"):
            trnfft.decay_attention_step(q, k, v, g, bad)
    with pytest.raises(ValueError, match="its own"):
        trnfft.decay_attention_step(q, k, v, g, s[:1].expand(2, 4, 8, 6))
    with pytest.raises(ValueError, match="no gradient"):
        trnfft.decay_attention_step(q.requires_grad_(), k, v, g, s)


def test_step_refuses_to_write_into_a_leaf_of_a_graph():
    q, k, v, g = qkv()
    s = torch.zeros(2, 4, 8, 6)
    with pytest.raises(ValueError, match="no gradient"):
        trnfft.decay_attention_step(q[:, 0], k[:, 0], v[:, 0], g, s, new_state=s.clone().requires_grad_())


def test_group_norm_refuses():
    x = torch.zeros(2, 5, 12)
    for args, kw, match in [((x[0, 0], 3), {}, "batch"), ((x.double(), 3), {}, "float32"), ((x, 5), {}, "fall into"),
                            ((x, 0), {}, "fall into"), ((x, 3, torch.ones(11)), {}, "weight"),
                            ((x, 3, None, torch.ones(12).double()), {}, "bias"), ((x, 3), {"activation": "tanh"}, "activation"),
                            ((x, 3), {"eps": -1.0}, "eps"), ((x, 3), {"eps": float("nan")}, "eps")]:
        with pytest.raises(ValueError, match=match):
            trnfft.group_norm(*args, **kw)


def test_forward_mode_is_refused():
    """A tangent would be lost: no kernel carries it.  Without one, an open level of forward mode changes nothing."""
    fwd = torch.autograd.forward_ad
    q, k, v, g = qkv()
    s = torch.zeros(2, 4, 8, 6)
    x, w = torch.zeros(2, 5, 12), torch.ones(12)
    calls = [(trnfft.decay_attention, [q, k, v, g], (0, 1, 2, 3)),
             (lambda q, k, v, g, s: trnfft.decay_attention(q, k, v, g, initial_state=s), [q, k, v, g, s], (4,)),
             (trnfft.decay_attention_step, [q[:, 0], k[:, 0], v[:, 0], g, s], (0, 1, 2, 3, 4)),
             (lambda x, w, b: trnfft.group_norm(x, 3, w, b), [x, w, w], (0, 1, 2))]
    for call, args, places in calls:
        for i in places:
            with fwd.dual_level():
                dual = fwd.make_dual(args[i], torch.ones_like(args[i]))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(*args[:i], dual, *args[i + 1:])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(lambda y: call(y, *args[1:]), (args[0],), (torch.ones_like(args[0]),))
    with fwd.dual_level():
        with pytest.raises(ValueError, match="fall into"):
            trnfft.group_norm(x, 5)


def test_no_cpu_fallback():
    if torch.cuda.is_available():
        pytest.skip("a CUDA device is visible")
    for call in (lambda: trnfft.decay_attention(*qkv()), lambda: trnfft.group_norm(torch.zeros(2, 4), 2)):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()


# -- the C boundary, whose checks run before any GPU work --------------------------------------


def shape(**kw):
    s = {**dict(batch=2, tokens=3, heads=4, kv_heads=2, key_width=8, value_width=6, cu_seqlens=0, num_seqs=0, dtype=0), **kw}
    return _lib.DECAY_SHAPE.pack(*(s[x] for x in ("batch", "tokens", "heads", "kv_heads", "key_width", "value_width")),
                                 *[1] * 12, s["cu_seqlens"], s["num_seqs"], 0, s["dtype"], 1.0)


def test_packed_shapes_have_c_layout():
    class Decay(ctypes.Structure):
        _fields_ = [(str(i), ctypes.c_int64) for i in range(18)] + [
            ("cu", ctypes.c_void_p), ("n", ctypes.c_int64), ("is64", ctypes.c_int32), ("t", ctypes.c_int32), ("s", ctypes.c_float)]

    class Step(ctypes.Structure):
        _fields_ = [(str(i), ctypes.c_int64) for i in range(13)] + [("t", ctypes.c_int32), ("s", ctypes.c_float)]

    assert _lib.DECAY_SHAPE.size == ctypes.sizeof(Decay)
    assert _lib.DECAY_STEP_SHAPE.size == ctypes.sizeof(Step)
    d = Decay.from_buffer_copy(_lib.DECAY_SHAPE.pack(*range(18), 77, 78, 1, 2, 0.5))
    assert [getattr(d, str(i)) for i in range(18)] == list(range(18))
    assert (d.cu, d.n, d.is64, d.t, d.s) == (77, 78, 1, 2, 0.5)


@pytest.mark.parametrize("kw,error", [
    (dict(dtype=3), ValueError), (dict(batch=-1), ValueError), (dict(kv_heads=3), ValueError), (dict(kv_heads=0), ValueError),
    (dict(key_width=0), ValueError), (dict(key_width=129), NotImplementedError), (dict(value_width=200), NotImplementedError),
    (dict(cu_seqlens=64, num_seqs=2), ValueError), (dict(cu_seqlens=66, num_seqs=2, batch=1), ValueError),
    (dict(tokens=1 << 31), NotImplementedError), (dict(heads=65536, kv_heads=65536), NotImplementedError), ({}, ValueError),
])
def test_attention_entry_refuses(kw, error):
    s = shape(**kw)
    with pytest.raises(error):
        _lib.call("trnfft_decay_attention", s, *[None] * 8, 0, None)
    with pytest.raises(error):
        _lib.call("trnfft_decay_attention_backward", s, *[None] * 12, 0, None)
    if kw:
        assert _lib.load().trnfft_decay_attention_work_bytes(s, 1) == -1
    with pytest.raises(ValueError, match="null shape"):
        _lib.call("trnfft_decay_attention", None, *[None] * 8, 0, None)


def test_attention_entry_of_nothing():
    for kw in (dict(batch=0), dict(tokens=0)):
        _lib.call("trnfft_decay_attention", shape(**kw), *[None] * 8, 0, None)
        _lib.call("trnfft_decay_attention_backward", shape(**kw), *[None] * 12, 0, None)


def test_step_entry_refuses():
    one = 4 * 8 * 6

    def step(state=4096, new=4096, **kw):
        s = {**dict(batch=2, heads=4, kv_heads=2, key_width=8, value_width=6, state_stride=one, new_state_stride=one, dtype=0),
             **kw}
        s = _lib.DECAY_STEP_SHAPE.pack(*(s[x] for x in ("batch", "heads", "kv_heads", "key_width", "value_width")), *[1] * 6,
                                       s["state_stride"], s["new_state_stride"], s["dtype"], 1.0)
        _lib.call("trnfft_decay_attention_step", s, 64, 64, 64, 64, state, new, 64, 0, None)

    for kw in (dict(dtype=7), dict(kv_heads=3), dict(key_width=0), dict(state=0), dict(state=4098),
               dict(new=4096 + 4 * one), dict(state_stride=one - 1), dict(new_state_stride=2 * one)):
        with pytest.raises(ValueError):
            step(**kw)
    with pytest.raises(NotImplementedError):
        step(key_width=129, state_stride=1 << 20, new_state_stride=1 << 20)
    step(batch=0)


def test_norm_entry_refuses():
    def norm(x=64, y=64, mean=None, rstd=None, n=2, s=3, c=12, g=3, act=0, dtype=0):
        _lib.call("trnfft_group_norm", x, None, None, y, mean, rstd, n, s, c, g, 1e-5, act, dtype, 4096, 0, None)

    for kw in (dict(g=5), dict(g=0), dict(c=0), dict(n=-1), dict(act=4), dict(dtype=3), dict(x=None), dict(x=66), dict(mean=64)):
        with pytest.raises(ValueError):
            norm(**kw)
    for kw in (dict(c=1 << 25, g=1), dict(n=1 << 31), dict(s=1 << 32)):
        with pytest.raises(NotImplementedError):
            norm(**kw)
    norm(n=0)
    assert _lib.load().trnfft_group_norm_work_bytes(2, 3, 12, 5, 0, 0) == -1
    with pytest.raises(ValueError):
        _lib.call("trnfft_group_norm_backward", 64, 64, None, None, None, None, 64, None, None, 2, 3, 12, 5, 0, 0, 4096, 0,
                  None)


@pytest.mark.parametrize("work", [4097, 4100, 4104])
def test_norm_entry_refuses_a_misaligned_work_area(work):
    """Its sums are stored 8 and 16 bytes at a time."""
    with pytest.raises(ValueError, match="misaligned work"):
        _lib.call("trnfft_group_norm", 64, None, None, 64, None, None, 2, 300, 12, 3, 1e-5, 0, 0, work, 0, None)
    with pytest.raises(ValueError, match="misaligned work"):
        _lib.call("trnfft_group_norm_backward", 64, 64, None, None, 64, 64, 64, None, None, 2, 300, 12, 3, 0, 0, work, 0, None)


def test_layers_have_their_parameters():
    assert set(GroupNorm(2, 8).state_dict()) == {"weight", "bias"}
    assert not GroupNorm(2, 8, affine=False).state_dict()
    assert set(ComplexGroupNorm(2, 8).state_dict()) == {"gn_re.weight", "gn_re.bias", "gn_im.weight", "gn_im.bias"}
    m = ComplexDecayAttention(6, 3, 4)
    assert m.log_decay.shape == (3,) and (m.log_decay < 0).all() and (m.log_decay.diff() > 0).all()
    assert m.initial_state(5).shape == (5, 3, 8, 8)


@pytest.mark.parametrize("heads,width", [(2, 65), (2, 128), (2, 0), (0, 8), (-1, 8)])
def test_layer_refuses_heads_that_it_cannot_run(heads, width):
    """When it is made, not at its first call."""
    with pytest.raises(ValueError, match="width"):
        ComplexDecayAttention(12, heads, width)


def test_widest_layer():
    assert ComplexDecayAttention(12, 2, 64).initial_state(1).shape == (1, 2, 128, 128)


@pytest.mark.parametrize("default", [torch.float64, torch.bfloat16])
def test_states_are_float32_whatever_the_default_type(default):
    m = ComplexDecayAttention(6, 3, 4)
    kept = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        assert m.initial_state(5).dtype == torch.float32
    finally:
        torch.set_default_dtype(kept)


# -- waits that give up ------------------------------------------------------------------------


def source(name):
    return (pathlib.Path(_lib.__file__).parent / "csrc" / name).read_text()


def test_roles_of_a_block_meet_at_bounded_waits_alone():
    """A warp whose wait ran out leaves its loop.  A barrier of a given number of threads inside the loops
    would wait for it without a limit: the roles of the tensor-core walk meet at bounded waits alone."""
    text = source("decay_tc.cu")
    assert not re.search(r"\b(bar|barrier)(\.cta)?\.(sync|red|arrive)\b", text)
    roles = text[text.index("if (warp > kMmaWarp)"):text.index("tcgen05.dealloc")]
    assert "__syncthreads" not in roles[:roles.rindex("fence_before();")], "no barrier of the block inside a role"


def test_streams_of_buffers_give_up_with_the_whole_block():
    """A thread whose wait for a buffer ran out goes through the same barriers as the others, to the end."""
    for name in ("group_norm.cu", "group_norm_bwd.cu"):
        text = source(name)
        waits = re.findall(r"[^\n]*\b(?:rows|samples)\.wait\([^\n]*", text)
        assert waits and all(w.strip() in ("rows.wait(i);", "samples.wait(i);") for w in waits), "no thread leaves by itself"
        assert len(re.findall(r"\b(?:rows|samples)\.finish\(\);", text)) == len(waits)
