"""The sequence and normalisation operators as a user's program calls them, over the sizes that such programs have.

Each case is one pass through one operator: decayed linear attention over whole sequences
(``prompt``), its training step (``train``), its single-frame form (``step``), group normalisation
with an activation over channels-last features (``norm``) and its training step (``norm_train``).
``run`` computes a pass in elementary torch operations, or through ``trnfft_b200`` where ``own`` is
true; ``exact`` gives the definition's value in 64 bits.
"""

import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZES = {"fp32": 4, "bf16": 2, "fp16": 2}
CHUNK = 128  # tokens that the plain form handles with one matrix of weights


def listed():
    return [
        # one live stream, one new frame: the smallest call, latency counts
        dict(name="step_one", op="step", batch=1, heads=8, kv_heads=8, dk=64, dv=64, type="bf16"),
        # a server's batch of streams, one new frame each
        dict(name="step_batch", op="step", batch=128, heads=16, kv_heads=4, dk=128, dv=128, type="bf16"),
        # utterances of different lengths packed together, continued from kept states, in the framework's own type
        dict(name="prompt_packed", op="prompt", batch=1, tokens=2517, seqs=9, heads=8, kv_heads=8, dk=64, dv=64, type="fp32"),
        # a batch of long prompts with shared key and value heads
        dict(name="prompt_batch", op="prompt", batch=8, tokens=4096, seqs=0, heads=16, kv_heads=4, dk=128, dv=128, type="bf16"),
        # one recording of half an hour, an odd number of frames: few heads, a long axis
        dict(name="prompt_long", op="prompt", batch=1, tokens=112501, seqs=0, heads=8, kv_heads=8, dk=64, dv=64, type="fp16"),
        # a training step of a wide model
        dict(name="train_wide", op="train", batch=8, tokens=2048, heads=16, kv_heads=16, dk=128, dv=128, type="bf16", carry=False),
        # a training step on ten-second spectrograms (626 frames), odd widths, shared heads, state carried over
        dict(name="train_frames", op="train", batch=6, tokens=626, heads=8, kv_heads=4, dk=40, dv=72, type="fp32", carry=True),
        # one frame's features: latency counts
        dict(name="norm_one", op="norm", batch=1, spots=1, channels=512, groups=8, type="fp32", act="silu"),
        # the heads of an attention's output, each normalised for itself
        dict(name="norm_heads", op="norm", batch=32768, spots=1, channels=2048, groups=16, type="bf16", act="none"),
        # features over whole spectrograms (257 bins, 626 frames)
        dict(name="norm_spectrogram", op="norm", batch=8, spots=257 * 626, channels=48, groups=6, type="fp32", act="gelu"),
        # a training step on 64 x 64 features
        dict(name="norm_train_square", op="norm_train", batch=32, spots=4096, channels=320, groups=32, type="bf16", act="silu"),
        # a training step on parts of spectrograms, odd sizes
        dict(name="norm_train_odd", op="norm_train", batch=5, spots=257 * 41, channels=84, groups=12, type="fp32", act="gelu"),
    ]


def _between(rng, lo, hi):
    """A whole number from lo to hi, spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["step", "prompt", "train", "norm", "norm_train"])
    kind = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if op.startswith("norm"):
        width, groups = _between(rng, 4, 128), _between(rng, 1, 32)
        spots = rng.choice([1, _between(rng, 2, 200000)])
        most = 16_000_000 // (width * groups * spots)
        batch = _between(rng, 1, max(1, min(40000, most)))
        if width * groups * spots > 64_000_000:
            spots = 64_000_000 // (width * groups)
        return dict(op=op, batch=batch, spots=spots, channels=width * groups, groups=groups, type=kind,
                    act=rng.choice(["none", "silu", "gelu"]))
    kv_heads, shared = _between(rng, 1, 16), rng.choice([1, 1, 2, 4])
    heads = min(32, kv_heads * shared) // kv_heads * kv_heads
    width = rng.choice([32, 64, 64, 128, 128])
    dk, dv = rng.choice([(width, width), (width, width), (rng.randint(5, 128), rng.randint(5, 128))])
    case = dict(op=op, heads=heads, kv_heads=kv_heads, dk=dk, dv=dv, type=kind)
    if op == "step":
        return dict(case, batch=_between(rng, 1, max(1, min(512, 32_000_000 // (heads * dk * dv)))))
    most = 20_000_000 // (heads * max(dk, dv))
    tokens = _between(rng, 1, min(32768, most))
    if op == "prompt" and rng.random() < 0.4:
        return dict(case, batch=1, tokens=min(tokens, 8192) + 3, seqs=_between(rng, 1, 24))
    batch = _between(rng, 1, min(64, max(1, most // tokens)))
    if op == "prompt":
        return dict(case, batch=batch, tokens=tokens, seqs=0)
    return dict(case, batch=batch, tokens=min(tokens, 4096), carry=rng.random() < 0.5)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = TYPES[case["type"]]

    def normal(*shape, scale=1.0, shift=0.0, type=t):
        return (torch.randn(*shape, device="cuda", generator=g) * scale + shift).to(type)

    if case["op"].startswith("norm"):
        n, s, c = case["batch"], case["spots"], case["channels"]
        state = dict(case=case, x=normal(n, s, c, scale=1.5, shift=0.7), weight=normal(c, scale=0.2, shift=1.0, type=torch.float32),
                     bias=normal(c, scale=0.2, type=torch.float32))
        if case["op"] == "norm_train":
            state["dy"] = normal(n, s, c)
            for name in ("x", "weight", "bias"):
                state[name].requires_grad_()
        return state
    b, h, hk, dk, dv = (case[k] for k in ("batch", "heads", "kv_heads", "dk", "dv"))
    # rates as such layers have them: a head's memory is from a few tokens to thousands of them
    memory = torch.logspace(math.log10(8.0), math.log10(4096.0), h, device="cuda", dtype=torch.float64)
    state = dict(case=case, log_decay=torch.log1p(-1.0 / memory).float())
    if case["op"] == "step":
        state |= dict(q=normal(b, h, dk), k=normal(b, hk, dk, scale=dk ** -0.5), v=normal(b, hk, dv),
                      state=normal(b, h, dk, dv, type=torch.float32))
        state["next"] = torch.empty_like(state["state"])
        return state
    n = case["tokens"]
    state |= dict(q=normal(b, n, h, dk), k=normal(b, n, hk, dk, scale=dk ** -0.5), v=normal(b, n, hk, dv))
    if case.get("seqs"):
        # sequences of any length, none among them, and three rows behind the last one
        cuts = torch.randint(0, n - 2, (case["seqs"] - 1,), generator=torch.Generator().manual_seed(seed)).sort().values.tolist()
        ends = [0, *cuts, n - 3]
        state["cu_seqlens"] = torch.tensor(ends, dtype=torch.int32, device="cuda")
        state["longest"] = max(1, max(y - x for x, y in zip(ends, ends[1:])))
        state["initial"] = normal(case["seqs"], h, dk, dv, type=torch.float32)
    if case["op"] == "train":
        state["do"] = normal(b, n, h, dv)
        if case["carry"]:
            state |= dict(initial=normal(b, h, dk, dv, type=torch.float32), dlast=normal(b, h, dk, dv, type=torch.float32))
        for name in ("q", "k", "v", "initial"):
            if name in state:
                state[name].requires_grad_()
    return state


def run(state):
    return (_own if own else _plain)(state)


def work(case):
    size = SIZES[case["type"]]
    if case["op"].startswith("norm"):
        n, c = case["batch"] * case["spots"] * case["channels"], case["channels"]
        if case["op"] == "norm":
            return {"bytes": 2 * n * size + 8 * c, "flops": 12 * n}
        return {"bytes": 4 * n * size + 16 * c, "flops": 40 * n}
    b, h, hk, dk, dv = (case[k] for k in ("batch", "heads", "kv_heads", "dk", "dv"))
    if case["op"] == "step":
        return {"bytes": 8 * b * h * dk * dv + size * b * (h * (dk + dv) + hk * (dk + dv)), "flops": 5 * b * h * dk * dv}
    rows = b * case["tokens"]
    once = size * rows * (h + hk) * (dk + dv)  # q, k, v and o (or their gradients)
    last = case["seqs"] or b if case["op"] == "prompt" else b
    if case["op"] == "prompt":
        return {"bytes": once + 4 * last * h * dk * dv * (2 if case["seqs"] else 1), "flops": 4 * rows * h * dk * dv}
    return {"bytes": 2 * once + 4 * last * h * dk * dv * (4 if case["carry"] else 0), "flops": 12 * rows * h * dk * dv}


# ---------------------------------------------------------------- through the framework


def _own(state):
    import trnfft_b200 as trnfft

    case = state["case"]
    op = case["op"]
    act = None if case.get("act") == "none" else case.get("act")
    if op == "norm":
        return trnfft.group_norm(state["x"], case["groups"], state["weight"], state["bias"], activation=act)
    if op == "norm_train":
        leaves = [state["x"], state["weight"], state["bias"]]
        y = trnfft.group_norm(state["x"], case["groups"], state["weight"], state["bias"], activation=act)
        dx, dw, db = torch.autograd.grad(y, leaves, state["dy"])
        return {"y": y, "dx": dx, "dw": dw, "db": db}
    if op == "step":
        o, last = trnfft.decay_attention_step(state["q"], state["k"], state["v"], state["log_decay"], state["state"],
                                              new_state=state["next"])
        return {"o": o, "state": last}
    o, last = trnfft.decay_attention(state["q"], state["k"], state["v"], state["log_decay"],
                                     initial_state=state.get("initial"), cu_seqlens=state.get("cu_seqlens"), return_state=True)
    if op == "prompt":
        return {"o": o, "state": last}
    if case["carry"]:
        got = torch.autograd.grad((o, last), (state["q"], state["k"], state["v"], state["initial"]), (state["do"], state["dlast"]))
        return {"o": o, "state": last, "dq": got[0], "dk": got[1], "dv": got[2], "dinitial": got[3]}
    got = torch.autograd.grad(o, (state["q"], state["k"], state["v"]), state["do"])
    return {"o": o, "dq": got[0], "dk": got[1], "dv": got[2]}


# ---------------------------------------------------------------- in elementary operations


def _activate(z, act):
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return z * (0.5 + 0.5 * torch.erf(z * math.sqrt(0.5)))
    return z


def _slope(z, act):
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 + 0.5 * torch.erf(z * math.sqrt(0.5)) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _plain_norm(state, eps=1e-5):
    case, x = state["case"], state["x"].detach()
    n, s, c = x.shape
    grouped = (n, s, case["groups"], c // case["groups"])
    xf, w, b = x.float().view(grouped), state["weight"].detach().view(grouped[2:]), state["bias"].detach().view(grouped[2:])
    mean = xf.mean((1, 3), keepdim=True)
    rest = xf - mean
    rstd = 1 / torch.sqrt((rest * rest).mean((1, 3), keepdim=True) + eps)
    hat = rest * rstd
    z = hat * w + b
    y = _activate(z, case["act"]).view(x.shape).to(x.dtype)
    if case["op"] == "norm":
        return y
    dz = state["dy"].float().view(grouped) * _slope(z, case["act"])
    dw, db = (dz * hat).sum((0, 1)).view(c), dz.sum((0, 1)).view(c)
    dhat = dz * w
    dx = rstd * (dhat - dhat.mean((1, 3), keepdim=True) - hat * (dhat * hat).mean((1, 3), keepdim=True))
    return {"y": y, "dx": dx.view(x.shape).to(x.dtype), "dw": dw, "db": db}


def _power(log_decay, n):
    """The decay of each head to the power n, for whole n >= 0: (heads, *n.shape)."""
    rate = log_decay.double().view(-1, *[1] * n.dim())
    return torch.exp(rate * n).float()


def _attend(q, k, v, log_decay):
    """o_t = sum over s <= t of decay^(t-s) (q_t . k_s) v_s and S = sum over s of decay^(T-1-s) k_s v_s^T,
    for (batch, time, heads, width) in 32 bits, in chunks of CHUNK tokens."""
    b, n, h, dk = q.shape
    chunks = -(-n // CHUNK)
    front = chunks * CHUNK - n  # zero rows before the first token change nothing

    def split(x):
        x = torch.cat([x.new_zeros(b, front, *x.shape[2:]), x], 1) if front else x
        return x.view(b, chunks, CHUNK, h, -1).permute(0, 3, 1, 2, 4)

    q, k, v = split(q), split(k), split(v)
    i = torch.arange(CHUNK, device=q.device)
    behind = i[:, None] - i[None, :]
    weight = torch.where(behind >= 0, _power(log_decay, behind.clamp_min(0)), 0.0)
    o = (q @ k.transpose(-1, -2) * weight[:, None]) @ v
    gain = ((k * _power(log_decay, CHUNK - 1 - i)[:, None, :, None]).transpose(-1, -2) @ v).reshape(b, h, chunks, -1)
    c = torch.arange(chunks + 1, device=q.device)
    passed = c[:, None] - 1 - c[None, :-1]
    carry = torch.where(passed >= 0, _power(log_decay, passed.clamp_min(0) * CHUNK), 0.0)
    states = (carry @ gain).view(b, h, chunks + 1, dk, -1)
    o = o + (q @ states[:, :, :-1]) * _power(log_decay, i + 1)[:, None, :, None]
    return o.permute(0, 2, 3, 1, 4).reshape(b, chunks * CHUNK, h, -1)[:, front:], states[:, :, -1]


def _shared(x, heads):
    """Each key or value head once for each query head that reads it, in 32 bits."""
    return x.detach().float().repeat_interleave(heads // x.shape[-2], -2)


def _plain_step(state):
    case = state["case"]
    q, k, v = (_shared(state[x], case["heads"]) for x in "qkv")
    kept = state["state"] * _power(state["log_decay"], torch.ones((), device=q.device, dtype=torch.int64))[:, None, None]
    state["next"].copy_(kept + k[..., :, None] * v[..., None, :])
    o = (q[..., None, :] @ state["next"]).squeeze(-2) * case["dk"] ** -0.5
    return {"o": o.to(state["q"].dtype), "state": state["next"]}


def _plain_prompt(state):
    case = state["case"]
    q, k, v = (_shared(state[x], case["heads"]) for x in "qkv")
    g, scale, kind = state["log_decay"], case["dk"] ** -0.5, state["q"].dtype
    if "cu_seqlens" not in state:
        o, last = _attend(q, k, v, g)
        return {"o": (o * scale).to(kind), "state": last}
    # each sequence right-aligned in a row of its own, behind zeros
    cu, longest, first = state["cu_seqlens"].long(), state["longest"], state["initial"]
    at = cu[1:, None] - longest + torch.arange(longest, device=cu.device)
    there = at >= cu[:-1, None]
    at = at.clamp_min(0)
    q, k, v = (torch.where(there[..., None, None], x[0, at], 0.0) for x in (q, k, v))
    o, last = _attend(q, k, v, g)
    place = (at - cu[:-1, None] + 1).clamp_min(0)
    o = o + torch.einsum("bthk,bhkv->bthv", q, first) * _power(g, place).permute(1, 2, 0)[..., None]
    last = last + first * _power(g, cu[1:] - cu[:-1]).t()[..., None, None]
    out = o.new_zeros(state["v"].shape[1], *o.shape[2:])
    out[at[there]] = o[there]
    return {"o": (out * scale).to(kind)[None], "state": last}


def _plain_train(state):
    case = state["case"]
    b, n, h, hk = (case[x] for x in ("batch", "tokens", "heads", "kv_heads"))
    q, k, v = (_shared(state[x], h) for x in "qkv")
    do, g, scale, kind = state["do"].float() * case["dk"] ** -0.5, state["log_decay"], case["dk"] ** -0.5, state["q"].dtype
    o, last = _attend(q, k, v, g)
    dq, _ = _attend(do, v, k, g)
    back = lambda x: x.flip(1)  # noqa: E731
    dv, dfirst = _attend(back(k), back(q), back(do), g)
    dk, _ = _attend(back(v), back(do), back(q), g)
    dv, dk = back(dv), back(dk)
    o = o * scale
    got = {}
    if case["carry"]:
        first, dlast, t = state["initial"].detach(), state["dlast"], torch.arange(n, device=q.device)
        ahead, left = (_power(g, x).t()[None, :, :, None] for x in (t + 1, n - 1 - t))
        o = o + torch.einsum("bthk,bhkv->bthv", q, first) * ahead * scale
        dq = dq + torch.einsum("bthv,bhkv->bthk", do, first) * ahead
        dv = dv + torch.einsum("bthk,bhkv->bthv", k, dlast) * left
        dk = dk + torch.einsum("bthv,bhkv->bthk", v, dlast) * left
        whole, one = (_power(g, torch.tensor(x, device=q.device))[:, None, None] for x in (n, 1))
        got = {"state": last + first * whole, "dinitial": dlast * whole + dfirst * one}
    dk, dv = (x.view(b, n, hk, h // hk, -1).sum(3) for x in (dk, dv))
    return {"o": o.to(kind), "dq": dq.to(kind), "dk": dk.to(kind), "dv": dv.to(kind), **got}


def _plain(state):
    op = state["case"]["op"]
    with torch.no_grad():
        if op.startswith("norm"):
            return _plain_norm(state)
        return {"step": _plain_step, "prompt": _plain_prompt, "train": _plain_train}[op](state)


# ---------------------------------------------------------------- the definitions in 64 bits


def _sum_over_past(q, k, v, rate, first, scale, block=512):
    """One sequence's (heads, time, width) by the definition, each weight from its own exponential."""
    n = q.shape[1]
    t = torch.arange(n, device=q.device, dtype=torch.float64)
    rows = []
    for at in range(0, n, block):
        end = min(n, at + block)
        behind = t[at:end, None] - t[None, :end]
        w = torch.exp(rate[:, None, None] * behind.clamp_min(0)) * (behind >= 0)
        rows.append(torch.matmul(torch.matmul(q[:, at:end], k[:, :end].mT) * w, v[:, :end]))
    o = torch.cat(rows, 1) if rows else q.new_zeros(q.shape[0], 0, v.shape[2])
    last = torch.matmul((k * torch.exp(rate[:, None] * (n - 1 - t))[..., None]).mT, v)
    if first is not None:
        o = o + torch.matmul(q, first) * torch.exp(rate[:, None] * (t + 1))[..., None]
        last = last + first * torch.exp(rate * n)[:, None, None]
    return o * scale, last


def _exact_attention(case, state):
    h, hk, scale, rate = case["heads"], case["kv_heads"], case["dk"] ** -0.5, state["log_decay"].double()

    def heads(x):
        return x.double().transpose(0, 1).repeat_interleave(h // x.shape[1], 0)

    if case["op"] == "step":
        q, k, v, old = (state[x].double() for x in ("q", "k", "v", "state"))
        k, v = (x.repeat_interleave(h // hk, 1) for x in (k, v))
        new = torch.exp(rate)[:, None, None] * old + torch.einsum("bhk,bhv->bhkv", k, v)
        return {"o": torch.einsum("bhk,bhkv->bhv", q, new) * scale, "state": new}
    if case["op"] == "prompt":
        if case["seqs"]:
            cu = state["cu_seqlens"].tolist()
            o, last = torch.zeros(case["tokens"], h, case["dv"], device="cuda", dtype=torch.float64), []
            for i, (x, y) in enumerate(zip(cu, cu[1:])):
                q, k, v = (heads(state[name][0, x:y]) for name in "qkv")
                part, end = _sum_over_past(q, k, v, rate, state["initial"][i].double(), scale)
                o[x:y] = part.transpose(0, 1)
                last.append(end)
            return {"o": o[None], "state": torch.stack(last)}
        o, last = [], []
        for i in range(case["batch"]):
            part, end = _sum_over_past(*(heads(state[name][i]) for name in "qkv"), rate, None, scale)
            o.append(part.transpose(0, 1))
            last.append(end)
        return {"o": torch.stack(o), "state": torch.stack(last)}
    got = {x: [] for x in ("o", "dq", "dk", "dv") + (("state", "dinitial") if case["carry"] else ())}
    for i in range(case["batch"]):
        q, k, v = (state[name].detach()[i].double().requires_grad_() for name in "qkv")
        first = state["initial"].detach()[i].double().requires_grad_() if case["carry"] else None
        o, last = _sum_over_past(heads(q), heads(k), heads(v), rate, first, scale, block=1024)
        loss = (o.transpose(0, 1) * state["do"][i].double()).sum()
        if case["carry"]:
            loss = loss + (last * state["dlast"][i].double()).sum()
        grads = torch.autograd.grad(loss, [q, k, v] + ([first] if case["carry"] else []))
        got["o"].append(o.detach().transpose(0, 1))
        for name, x in zip(("dq", "dk", "dv", "dinitial"), grads):
            got[name].append(x)
        if case["carry"]:
            got["state"].append(last.detach())
    return {name: torch.stack(x) for name, x in got.items()}


def _exact_norm(case, state, eps=1e-5):
    g, act = case["groups"], case["act"]
    w, b = (state[x].detach().double().requires_grad_() for x in ("weight", "bias"))
    ys, dxs = [], []
    dw, db = torch.zeros_like(w), torch.zeros_like(b)
    train = case["op"] == "norm_train"
    part = max(1, 100_000_000 // (case["spots"] * case["channels"]))
    for at in range(0, case["batch"], part):
        x = state["x"].detach()[at:at + part].double().requires_grad_()
        rows = x.unflatten(-1, (g, -1)).transpose(1, 2).flatten(2)  # (batch, group, values)
        var, mean = torch.var_mean(rows, dim=-1, unbiased=False, keepdim=True)
        hat = ((rows - mean) / torch.sqrt(var + eps)).unflatten(-1, (case["spots"], -1)).transpose(1, 2).flatten(2)
        z = hat * w + b
        y = {"none": lambda: z, "silu": lambda: z * torch.sigmoid(z), "gelu": lambda: 0.5 * z * torch.erfc(-z / math.sqrt(2.0))}[act]()
        ys.append(y.detach())
        if train:
            dx, pw, pb = torch.autograd.grad(y, (x, w, b), state["dy"][at:at + part].double())
            dxs.append(dx)
            dw, db = dw + pw, db + pb
    y = torch.cat(ys)
    return {"y": y, "dx": torch.cat(dxs), "dw": dw.detach(), "db": db.detach()} if train else y


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"].startswith("norm"):
        return _exact_norm(case, state)
    return _exact_attention(case, state)
