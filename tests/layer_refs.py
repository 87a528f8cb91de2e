"""Plain 64-bit forms of the layer operators, for the tests, and the bounds that their roundings give."""

import torch

UNIT = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def decay_ref(q, k, v, log_decay, scale, first=None, absolute=False):
    """The recurrence, token by token, of one batch in 64 bits: (o, last state).  With `absolute`, of the
    absolute values: the sum that bounds every rounding's effect."""
    q, k, v = (x.double() for x in (q, k, v))
    g = torch.exp(log_decay.double())[None, :, None, None]
    k, v = (x.repeat_interleave(q.shape[2] // k.shape[2], 2) for x in (k, v))
    s = q.new_zeros(q.shape[0], q.shape[2], q.shape[3], v.shape[3]) if first is None else first.double()
    if absolute:
        q, k, v, s = q.abs(), k.abs(), v.abs(), s.abs()
    rows = []
    for t in range(q.shape[1]):
        s = g * s + k[:, t, :, :, None] * v[:, t, :, None, :]
        rows.append(torch.einsum("bhk,bhkv->bhv", q[:, t], s) * scale)
    o = torch.stack(rows, 1) if rows else q.new_zeros(q.shape[0], 0, q.shape[2], v.shape[3])
    return o, s


def decay_bound(dtype, terms, total, want, fp32_out=False):
    """How far a value may be from `want`, where `total` is the sum of its terms' absolute values.

    Products of two factors split into two 11-bit parts lose at most 3 * 2^-22 each, of at most four on
    a path with the factors of the decay (2^-23 each): 16 * 2^-22.  `terms` additions round by 2^-23 at
    most.  A 16-bit type may round the weights and the state that it multiplies once more, half a step
    each, and its result is rounded by half a step."""
    b = (16 * 2.0 ** -22 + terms * 2.0 ** -23) * total
    if dtype != torch.float32 and not fp32_out:
        b = b + 2 * UNIT[dtype] * total
    out = 2.0 ** -24 if fp32_out else UNIT[dtype]
    tiny = 2.0 ** -24 if dtype == torch.float16 and not fp32_out else 1e-30  # half the smallest fp16 step is 2^-25
    return b + out * want.abs() + tiny


def act_ref(z, act):
    if act == "relu":
        return torch.relu(z)
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(-z * 0.5 ** 0.5)
    return z


def norm_ref(x, groups, weight, bias, eps, act):
    """Group norm with an activation in 64 bits, differentiable."""
    n, c = x.shape[0], x.shape[-1]
    rows = x.reshape(n, -1, groups, c // groups)
    mean = rows.mean((1, 3), keepdim=True)
    var = ((rows - mean) ** 2).mean((1, 3), keepdim=True)
    z = ((rows - mean) / torch.sqrt(var + eps)).reshape(x.shape)
    if weight is not None:
        z = z * weight
    if bias is not None:
        z = z + bias
    return act_ref(z, act)
