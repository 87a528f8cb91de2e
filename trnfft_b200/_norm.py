"""Group normalisation with an activation over channels-last features (trnfft_group_norm)."""

from __future__ import annotations

import functools

import torch
import torch.autograd.forward_ad as fwd

from . import _lib
from ._attention import DTYPES, _addr, once
from ._device import place_layer, refuse_tangents

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3}


@functools.lru_cache(maxsize=4096)
def _work_bytes(n, s, c, groups, dtype, backward):
    size = _lib.load().trnfft_group_norm_work_bytes(n, s, c, groups, dtype, backward)
    if size < 0:
        _lib.raise_last("trnfft_group_norm_work_bytes")
    return size


def _work(n, s, c, groups, dtype, backward, device):
    size = _work_bytes(n, s, c, groups, dtype, backward)
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _float(p):
    return p if p is None or p.dtype == torch.float32 else p.float()


def _forward(x, groups, weight, bias, eps, act, keep):
    n, c = x.shape[0], x.shape[-1]
    s = x.numel() // (n * c) if n else 0
    y = torch.empty_like(x)
    stats = torch.empty(2, n, groups, dtype=torch.float32, device=x.device) if keep else None
    dt = DTYPES[x.dtype]
    work = _work(n, s, c, groups, dt, 0, x.device)
    at = stats.data_ptr() if keep else None
    _lib.call("trnfft_group_norm", x.data_ptr(), _addr(weight), _addr(bias), y.data_ptr(), at,
              at + 4 * n * groups if keep else None, n, s, c, groups, eps, act, dt, _addr(work), x.get_device(),
              _lib.raw_stream(x.get_device()))
    return y, stats


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, act):
        w, b = _float(weight), _float(bias)
        y, stats = _forward(x, groups, w, b, eps, act, True)
        ctx.save_for_backward(x, w, b, stats)
        ctx.groups, ctx.act = groups, act
        ctx.types = (weight.dtype if weight is not None else None, bias.dtype if bias is not None else None)
        return y

    @staticmethod
    @once
    def backward(ctx, dy):
        x, w, b, stats = ctx.saved_tensors
        groups, need = ctx.groups, ctx.needs_input_grad
        n, c = x.shape[0], x.shape[-1]
        s = x.numel() // (n * c) if n else 0
        dy = dy.contiguous()
        dx = torch.empty_like(x) if need[0] else None
        dw = torch.empty(c, dtype=torch.float32, device=x.device) if need[1] else None
        db = torch.empty(c, dtype=torch.float32, device=x.device) if need[2] else None
        dt = DTYPES[x.dtype]
        work = _work(n, s, c, groups, dt, 1, x.device)
        at = stats.data_ptr()
        _lib.call("trnfft_group_norm_backward", x.data_ptr(), dy.data_ptr(), _addr(w), _addr(b), at, at + 4 * n * groups,
                  _addr(dx), _addr(dw), _addr(db), n, s, c, groups, ctx.act, dt, _addr(work), x.get_device(),
                  _lib.raw_stream(x.get_device()))
        if dw is not None and ctx.types[0] != torch.float32:
            dw = dw.to(ctx.types[0])
        if db is not None and ctx.types[1] != torch.float32:
            db = db.to(ctx.types[1])
        return dx, dw, db, None, None, None


def _fits(p, c):
    return p is None or (p.dim() == 1 and p.shape[0] == c and p.dtype in DTYPES)


def _refuse(x, num_groups, weight, bias, eps, activation):
    """Says what is wrong with the arguments; the number of groups as an int if nothing is."""
    if x.dim() < 2:
        raise ValueError(f"group_norm: x must be (batch, ..., channels), got {tuple(x.shape)}")
    if x.dtype not in DTYPES:
        raise ValueError(f"group_norm: x must be float32, bfloat16 or float16, got {x.dtype}")
    c, num_groups = x.shape[-1], int(num_groups)
    if c < 1 or num_groups < 1 or c % num_groups:
        raise ValueError(f"group_norm: {c} channels do not fall into {num_groups} groups")
    if activation not in ACTIVATIONS:
        raise ValueError(f"group_norm: activation must be one of {tuple(ACTIVATIONS)}, got {activation!r}")
    if not eps >= 0:
        raise ValueError(f"group_norm: eps must not be negative, got {eps}")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None and (p.shape != (c,) or p.dtype not in DTYPES):
            raise ValueError(f"group_norm: {name} must hold {c} values in float32, bfloat16 or float16, got {p.dtype} "
                             f"{tuple(p.shape)}")
    return num_groups


def group_norm(x: torch.Tensor, num_groups: int, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None,
               eps: float = 1e-5, activation: str | None = None) -> torch.Tensor:
    """act(group_norm(x)) over channels-last features, in one operator.

    x is (batch, ..., channels), float32, bfloat16 or float16.  The channels fall into
    num_groups groups; each group of each sample is normalised by its mean and variance
    over all positions (statistics in float32), then scaled by weight and shifted by bias
    (channels each, optional) and put through the activation: None, "relu", "silu" or
    "gelu" (z times the normal distribution function, to 1e-7).  Differentiable once in x, weight and bias;
    forward-mode tangents are refused.
    """
    c = x.shape[-1] if x.dim() else 0
    if not (x.dim() >= 2 and x.dtype in DTYPES and c > 0 and type(num_groups) is int and num_groups > 0 and c % num_groups == 0
            and activation in ACTIVATIONS and eps >= 0 and _fits(weight, c) and _fits(bias, c)):
        num_groups = _refuse(x, num_groups, weight, bias, eps, activation)
    if fwd._current_level >= 0:
        refuse_tangents("group_norm", x, weight, bias)
    restore = None
    device = x.get_device()
    if device < 0 or (weight is not None and weight.get_device() != device) or (bias is not None and
                                                                               bias.get_device() != device):
        (x, weight, bias), restore = place_layer("group_norm", x, weight, bias)
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and any(p is not None and p.requires_grad for p in (x, weight, bias)):
        y = _GroupNormFn.apply(x, weight, bias, num_groups, eps, act)
    else:
        y = _forward(x, num_groups, _float(weight), _float(bias), eps, act, False)[0]
    return y if restore is None else restore(y)
