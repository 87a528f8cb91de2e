"""Linear attention with a decay for each head: whole sequences, training and single tokens.

Every head keeps a matrix state that decays by a constant factor per token::

    S_t = exp(log_decay) S_{t-1} + k_t v_t^T        o_t = scale * q_t S_t

``decay_attention`` runs whole sequences (trnfft_decay_attention) with its
gradients (trnfft_decay_attention_backward), ``decay_attention_step`` one
token of each stream (trnfft_decay_attention_step).  Operands are float32,
bfloat16 or float16; states are float32.
"""

from __future__ import annotations

import torch
import torch.autograd.forward_ad as fwd

from . import _lib
from ._device import place_layer, refuse_tangents

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _unit_inner(t: torch.Tensor) -> torch.Tensor:
    """The tensor itself where its last dimension is dense, else a contiguous copy."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _shape(q, k, v, o_stride, cu, nseq, scale) -> bytes:
    b, t, h, dk = q.shape
    return _lib.DECAY_SHAPE.pack(b, t, h, k.shape[2], dk, v.shape[3], *q.stride()[:3], *k.stride()[:3], *v.stride()[:3],
                                 *o_stride, 0 if cu is None else cu.data_ptr(), nseq,
                                 cu is not None and cu.dtype == torch.int64, DTYPES[q.dtype], scale)


def _addr(t):
    return None if t is None else t.data_ptr()


def _work(shape, backward, device):
    n = _lib.load().trnfft_decay_attention_work_bytes(shape, backward)
    if n < 0:
        _lib.raise_last("trnfft_decay_attention_work_bytes")
    return torch.empty(n, dtype=torch.uint8, device=device) if n else None


def once(run):
    """The backward of a Function whose gradients are no graph.  torch's once_differentiable says so to
    whoever differentiates them, at a tenth of a small step's time, and is needed only where a graph of
    the gradients is made at all."""
    careful = torch.autograd.function.once_differentiable(run)

    def backward(ctx, *grads):
        return (careful if torch.is_grad_enabled() else run)(ctx, *grads)

    return backward


def _forward(q, k, v, log_decay, initial, cu, nseq, scale, want_state):
    o = torch.empty(q.shape[:3] + v.shape[3:], dtype=q.dtype, device=q.device)
    last = None
    if want_state:
        last = torch.empty(nseq, q.shape[2], q.shape[3], v.shape[3], dtype=torch.float32, device=q.device)
    shape = _shape(q, k, v, (0, 0, 0), cu, nseq, scale)
    work = _work(shape, 0, q.device)
    _lib.call("trnfft_decay_attention", shape, q.data_ptr(), k.data_ptr(), v.data_ptr(),
              log_decay.data_ptr(), _addr(initial), o.data_ptr(), _addr(last), _addr(work), q.get_device(),
              _lib.raw_stream(q.get_device()))
    return o, last


class _DecayFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, log_decay, initial, cu, nseq, scale, want_state):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(q, k, v, log_decay, initial, cu)
        ctx.nseq, ctx.scale = nseq, scale
        return _forward(q, k, v, log_decay, initial, cu, nseq, scale, want_state)

    @staticmethod
    @once
    def backward(ctx, do, dlast):
        q, k, v, log_decay, initial, cu = ctx.saved_tensors
        if do is None and dlast is None:
            return (None,) * 9
        do = torch.zeros(q.shape[:3] + v.shape[3:], dtype=q.dtype, device=q.device) if do is None else _unit_inner(do)
        dlast = None if dlast is None else dlast.contiguous()
        need = ctx.needs_input_grad
        dq = torch.empty(q.shape, dtype=q.dtype, device=q.device) if need[0] else None
        dk = torch.empty(k.shape, dtype=q.dtype, device=q.device) if need[1] else None
        dv = torch.empty(v.shape, dtype=q.dtype, device=q.device) if need[2] else None
        dinitial = torch.empty(initial.shape, dtype=torch.float32, device=q.device) if need[4] else None
        shape = _shape(q, k, v, do.stride()[:3], cu, ctx.nseq, ctx.scale)
        work = _work(shape, 1, q.device)
        _lib.call("trnfft_decay_attention_backward", shape, q.data_ptr(), k.data_ptr(), v.data_ptr(),
                  log_decay.data_ptr(), _addr(initial), do.data_ptr(), _addr(dlast), _addr(dq), _addr(dk), _addr(dv),
                  _addr(dinitial), _addr(work), q.get_device(), _lib.raw_stream(q.get_device()))
        return dq, dk, dv, None, dinitial, None, None, None, None


def _check_heads(fn, q, k, v, log_decay, dims):
    names = "(batch, time, heads, width)" if dims == 4 else "(batch, heads, width)"
    if not q.dim() == k.dim() == v.dim() == dims:
        raise ValueError(f"{fn}: q, k and v must be {names}, got {tuple(q.shape)}, {tuple(k.shape)}, {tuple(v.shape)}")
    if q.dtype not in DTYPES or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"{fn}: q, k and v must share one of float32, bfloat16 and float16, got {q.dtype}, {k.dtype}, "
                         f"{v.dtype}")
    if k.shape[:-1] != v.shape[:-1] or q.shape[:-2] != k.shape[:-2] or q.shape[-1] != k.shape[-1]:
        raise ValueError(f"{fn}: the shapes {tuple(q.shape)}, {tuple(k.shape)} and {tuple(v.shape)} of q, k and v do not "
                         "belong together")
    h, hk = q.shape[-2], k.shape[-2]
    if h < 1 or hk < 1 or h % hk:
        raise ValueError(f"{fn}: {h} heads are not a multiple of {hk} key/value heads")
    if q.shape[-1] < 1 or v.shape[-1] < 1:
        raise ValueError(f"{fn}: head widths must be positive")
    if log_decay.shape != (h,) or not log_decay.is_floating_point():
        raise ValueError(f"{fn}: log_decay must be a floating tensor of {h} values, got {tuple(log_decay.shape)}")


def decay_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, *,
                    scale: float | None = None, initial_state: torch.Tensor | None = None,
                    cu_seqlens: torch.Tensor | None = None, return_state: bool = False):
    """Causal linear attention with a decay for each head, over whole sequences.

    For every head, S_t = exp(log_decay) S_{t-1} + k_t v_t^T and o_t = scale * q_t S_t.

    q is (batch, time, heads, width), k and v are (batch, time, kv_heads, width) and
    (batch, time, kv_heads, value width), all float32, bfloat16 or float16, any strides;
    query head h reads key/value head h // (heads // kv_heads).  Widths go up to 128.
    log_decay (heads) holds the logarithm of each head's factor, at most 0 (0: no decay, -inf:
    the token alone); it is a constant, not differentiated.  scale defaults to width ** -0.5.

    initial_state (sequences, heads, width, value width), float32, is the state before the
    first token (zero by default).  With return_state the result is (o, state): the state
    after each sequence's last token, from which the sequence can be continued.

    With cu_seqlens (int32 or int64, ascending, one more value than there are sequences),
    batch is 1 and sequence i is the rows cu_seqlens[i] to cu_seqlens[i+1]; it may be empty.
    Rows of no sequence get zeros.  The values stay on the device and are not checked: of
    values that are not ascending or not in range, no output is defined.

    A NaN or an infinite value in an operand reaches the results that its sums lead to and no
    others; an infinite state stays infinite however it decays (but NaN under log_decay -inf).

    Differentiable once in q, k, v and initial_state, from o and from the state; forward-mode tangents are
    refused.
    """
    _check_heads("decay_attention", q, k, v, log_decay, 4)
    b, t, h, dk = q.shape
    dv = v.shape[3]
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise ValueError("decay_attention: log_decay has no gradient here; pass log_decay.detach()")
    nseq = b
    if cu_seqlens is not None:
        if cu_seqlens.dim() != 1 or cu_seqlens.dtype not in (torch.int32, torch.int64) or cu_seqlens.shape[0] < 1:
            raise ValueError("decay_attention: cu_seqlens must be a vector of int32 or int64")
        if b != 1:
            raise ValueError(f"decay_attention: packed sequences need batch 1, got {b}")
        nseq = cu_seqlens.shape[0] - 1
    if initial_state is not None and (initial_state.shape != (nseq, h, dk, dv) or initial_state.dtype != torch.float32):
        raise ValueError(f"decay_attention: initial_state must be float32 {(nseq, h, dk, dv)}, got {initial_state.dtype} "
                         f"{tuple(initial_state.shape)}")
    if fwd._current_level >= 0:
        refuse_tangents("decay_attention", q, k, v, log_decay, initial_state)
    (q, k, v, log_decay, initial, cu), restore = place_layer("decay_attention", q, k, v, log_decay, initial_state, cu_seqlens)
    q, k, v = _unit_inner(q), _unit_inner(k), _unit_inner(v)
    log_decay = log_decay.detach().float().contiguous()
    initial = None if initial is None else initial.contiguous()
    cu = None if cu is None else cu.contiguous()
    scale = dk ** -0.5 if scale is None else float(scale)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or
                                    (initial is not None and initial.requires_grad)):
        o, last = _DecayFn.apply(q, k, v, log_decay, initial, cu, nseq, scale, return_state)
    else:
        o, last = _forward(q, k, v, log_decay, initial, cu, nseq, scale, return_state)
    return (restore(o), restore(last)) if return_state else restore(o)


def decay_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, state: torch.Tensor, *,
                         scale: float | None = None, new_state: torch.Tensor | None = None):
    """One new token of each stream: the recurrent form of ``decay_attention``.

    q is (batch, heads, width), k and v are (batch, kv_heads, width) and (batch, kv_heads,
    value width); state (batch, heads, width, value width), float32, holds the streams'
    states, each dense, at any distance.  The state is updated in place, or, where
    new_state is given, left as it is and the new one written there.  Returns (o, new
    state), o (batch, heads, value width).  No gradient: train with ``decay_attention``.
    """
    fn = "decay_attention_step"
    qs, ks, vs = q.shape, k.shape, v.shape
    # (the checks of _check_heads in one expression: a single token's call takes no longer than its kernel)
    if not (len(qs) == len(ks) == len(vs) == 3 and q.dtype in DTYPES and k.dtype == q.dtype and v.dtype == q.dtype
            and ks[:2] == vs[:2] and qs[0] == ks[0] and qs[2] == ks[2] and ks[1] > 0 and qs[1] > 0 and qs[1] % ks[1] == 0
            and qs[2] > 0 and vs[2] > 0 and log_decay.shape == qs[1:2] and log_decay.dtype == torch.float32):
        _check_heads(fn, q, k, v, log_decay, 3)
    b, h, dk = qs
    dv = vs[2]
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, log_decay, state, new_state)):
        raise ValueError(f"{fn}: has no gradient; use decay_attention, or torch.no_grad()")
    if fwd._current_level >= 0:
        refuse_tangents(fn, q, k, v, log_decay, state, new_state)
    one = h * dk * dv
    for s in (state,) if new_state is None else (state, new_state):
        if s.shape != (b, h, dk, dv) or s.dtype != torch.float32 or s.device != state.device:
            raise ValueError(f"{fn}: states must be float32 {(b, h, dk, dv)} on one device, got {s.dtype} {tuple(s.shape)}")
        stride = s.stride()
        if stride[1:] != (dk * dv, dv, 1) and b and not s[0].is_contiguous() or b > 1 and stride[0] < one:
            raise ValueError(f"{fn}: the state of each stream must be dense and its own, got strides {stride}")
    new_state = state if new_state is None else new_state
    if not state.is_cuda:  # states in host memory: update a copy on the device
        (q, k, v, log_decay, dev_state), restore = place_layer(fn, q, k, v, log_decay, state)
        o, got = decay_attention_step(q, k, v, log_decay, dev_state, scale=scale)
        new_state.copy_(got)
        return restore(o), new_state
    device = state.get_device()
    restore = None
    if not (q.get_device() == k.get_device() == v.get_device() == log_decay.get_device() == device):
        (q, k, v, log_decay, _), restore = place_layer(fn, q, k, v, log_decay, state)
    q, k, v = _unit_inner(q), _unit_inner(k), _unit_inner(v)
    if log_decay.dtype != torch.float32 or not log_decay.is_contiguous():
        log_decay = log_decay.float().contiguous()
    o = torch.empty(b, h, dv, dtype=q.dtype, device=q.device)
    shape = _lib.DECAY_STEP_SHAPE.pack(b, h, k.shape[1], dk, dv, *q.stride()[:2], *k.stride()[:2], *v.stride()[:2],
                                       state.stride(0) if b > 1 else one, new_state.stride(0) if b > 1 else one,
                                       DTYPES[q.dtype], dk ** -0.5 if scale is None else scale)
    _lib.call("trnfft_decay_attention_step", shape, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(),
              state.data_ptr(), new_state.data_ptr(), o.data_ptr(), device, _lib.raw_stream(device))
    torch.autograd.graph.increment_version(new_state)
    return (o if restore is None else restore(o)), new_state
