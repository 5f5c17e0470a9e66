"""The operators over image and video tokens (``bndm_amd.tokens``) as cases that can be timed: their plain forms in elementary
torch operations, the same calls through the framework's kernels, and their values in 64 bits.

    linear                   y = act(x W^T + b) + r                                    forward, and with its gradients
    rotary                   rotation of query / key heads by positions on several axes forward, and with its gradients
    differential_attention   (softmax(q1 k1^T s) - lam softmax(q2 k2^T s)) v            forward, single tokens, gradients
"""
import math

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # the time embedding's hidden layer at the sampler's batch: one small launch inside a step, latency is what counts
        {"name": "linear time embedding", "op": "linear", "rows": 64, "k": 512, "n": 512, "act": "silu", "bias": True,
         "residual": False, "train": False, "type": "f16"},
        # one time step through the projections of every block at once: a single row against 10 MB of weights
        {"name": "linear one row", "op": "linear", "rows": 1, "k": 512, "n": 9984, "act": "", "bias": True,
         "residual": False, "train": False, "type": "bf16"},
        # an attention layer's output projection over eight 64 x 64 latents, added to the stream it came from
        {"name": "linear projection", "op": "linear", "rows": 32768, "k": 512, "n": 512, "act": "", "bias": True,
         "residual": True, "train": False, "type": "bf16"},
        # a training step through the wide layer of a block over sixteen 32 x 32 latents
        {"name": "linear training", "op": "linear", "rows": 16384, "k": 1024, "n": 4096, "act": "gelu", "bias": True,
         "residual": False, "train": True, "type": "bf16"},
        # sizes that no tile divides and rows that no wide load is aligned to
        {"name": "linear odd training", "op": "linear", "rows": 1237, "k": 515, "n": 771, "act": "silu", "bias": True,
         "residual": True, "train": True, "type": "f16"},
        # one new token for each of 64 sequences: latency
        {"name": "rotary one token", "op": "rotary", "batch": 64, "grid": "1x1x1", "heads": 16, "kv_heads": 4, "dim": 64,
         "interleaved": False, "packed": True, "first": 4097, "train": False, "type": "bf16"},
        # queries and keys of eight 64 x 64 latents, both read out of the projection's packed rows
        {"name": "rotary image", "op": "rotary", "batch": 8, "grid": "64x64", "heads": 32, "kv_heads": 32, "dim": 64,
         "interleaved": False, "packed": True, "first": 0, "train": False, "type": "f16"},
        # a training step of a clip late in a long video: odd sides, a head size that is no power of two, far positions
        {"name": "rotary video training", "op": "rotary", "batch": 2, "grid": "15x30x45", "heads": 24, "kv_heads": 8, "dim": 96,
         "interleaved": True, "packed": False, "first": 100000, "train": True, "type": "f32"},
        # the 4 x 4 level of the network: 512 channels in heads of 8, 16 tokens, the sampler's batch
        {"name": "attention 4x4 level", "op": "attention", "batch": 64, "nq": 16, "nk": 16, "heads": 32, "kv_heads": 32,
         "dim": 8, "causal": False, "ragged": False, "packed": False, "train": False, "type": "f16"},
        # sampling: 64 x 64 latents, every token sees every token
        {"name": "attention image", "op": "attention", "batch": 4, "nq": 4096, "nk": 4096, "heads": 8, "kv_heads": 8,
         "dim": 64, "causal": False, "ragged": False, "packed": True, "train": False, "type": "bf16"},
        # a training step over padded token sequences in raster order, shared key heads
        {"name": "attention training", "op": "attention", "batch": 4, "nq": 2047, "nk": 2047, "heads": 8, "kv_heads": 4,
         "dim": 64, "causal": True, "ragged": True, "packed": False, "train": True, "type": "f16"},
        # serving: one new token for each of eight sequences over its stored keys, four query heads to a key head
        {"name": "attention one token", "op": "attention", "batch": 8, "nq": 1, "nk": 16384, "heads": 16, "kv_heads": 4,
         "dim": 64, "causal": True, "ragged": True, "packed": False, "train": False, "type": "bf16"},
    ]


def draw(rng):
    def spread(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(["linear", "rotary", "attention"])
    train = rng.random() < 0.5
    if kind == "linear":
        rows, k, n = spread(1, 32768), spread(64, 4096), spread(64, 10000)
        if rng.random() < 0.6:  # most widths are multiples of eight, as channel counts are
            k, n = (k + 7) // 8 * 8, (n + 7) // 8 * 8
        rows = max(1, min(rows, 68_000_000_000 // (k * n)))
        return {"op": "linear", "rows": rows, "k": k, "n": n, "act": rng.choice(["", "silu", "gelu"]), "bias": rng.random() < 0.7,
                "residual": rng.random() < 0.4, "train": train, "type": rng.choice(["f16", "bf16"])}
    if kind == "rotary":
        sides = [spread(1, 64) for _ in range(rng.choice([2, 3]))]
        heads = rng.choice([1, 2, 4, 6])
        per = rng.choice([1, 2, 4])
        dim = 2 * rng.choice([8, 15, 16, 20, 32, 48, 64])
        tokens = math.prod(sides)
        batch = max(1, min(spread(1, 64), 240_000_000 // (tokens * heads * (per + 1) * dim * (2 if train else 1))))
        while tokens * heads * (per + 1) * dim * (2 if train else 1) > 240_000_000:
            sides[0] = max(1, sides[0] // 2)
            tokens = math.prod(sides)
        return {"op": "rotary", "batch": batch, "grid": "x".join(map(str, sides)), "heads": heads * per, "kv_heads": heads, "dim": dim,
                "interleaved": rng.random() < 0.5, "packed": rng.random() < 0.5, "first": rng.choice([0, spread(1, 1_000_000)]),
                "train": train, "type": rng.choice(["f16", "bf16", "f32"])}
    dim = rng.choice([8, 16, 24, 32, 40, 64, 64, 64, 72, 96, 128])
    heads, per = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 4])
    one = not train and rng.random() < 0.4
    nk = spread(16, 16384) if one else spread(1, 4096)
    nq = rng.choice([1, 1, 2, 5]) if one else (nk if rng.random() < 0.6 else spread(1, 4096))
    most = min((100_000_000_000 if train else 200_000_000_000) // (12 * dim), 500_000_000)  # products of a query and a key
    while heads * per * nq * nk > most:
        nq, nk = max(1, nq // 2), max(1, nk // 2)
    batch = max(1, min(spread(1, 32), most // (heads * per * nq * nk)))
    return {"op": "attention", "batch": batch, "nq": nq, "nk": nk, "heads": heads * per, "kv_heads": heads, "dim": dim,
            "causal": rng.random() < 0.5, "ragged": rng.random() < 0.5, "packed": rng.random() < 0.4 and nq == nk, "train": train,
            "type": rng.choice(["f16", "bf16"])}


# ------------------------------------------------------------------------------------------------ what a program has in hand
def _sides(case):
    return [int(s) for s in case["grid"].split("x")]


def _sections(case):
    """Rotated pairs of each axis: shared out evenly, the first axes take what is left over."""
    axes, pairs = len(_sides(case)), case["dim"] // 2
    return [pairs // axes + (1 if a < pairs % axes else 0) for a in range(axes)]


def _kv_lengths(case):
    """Stored keys of each sequence: from all of them down to about a half; the second of three or more has none yet."""
    batch, nk = case["batch"], case["nk"]
    lengths = [nk - (nk // 2) * b // max(1, batch) for b in range(batch)]
    if batch > 2:
        lengths[1] = 0
    return lengths


def _q_start(case):
    """Where the first query stands among the keys: at the end of what is stored (serving), or at the start (whole sequences)."""
    if case["nq"] == case["nk"]:
        return [0] * case["batch"]
    lengths = _kv_lengths(case) if case["ragged"] else [case["nk"]] * case["batch"]
    return [n - case["nq"] for n in lengths]


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dtype = TYPES[case["type"]]

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * std).to(dtype)

    state = {"case": case, "grad": None}
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        leaves = {"x": normal(rows, k), "weight": normal(n, k, std=k ** -0.5)}
        if case["bias"]:
            leaves["bias"] = normal(n, std=0.1)
        if case["residual"]:
            leaves["residual"] = normal(rows, n)
        out = (rows, n)
    elif case["op"] == "rotary":
        b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["dim"]
        sides = _sides(case)
        tokens = math.prod(sides)
        rows = torch.arange(tokens, device="cuda")
        axes = []
        for side in reversed(sides):  # the last axis runs fastest
            axes.insert(0, rows % side)
            rows = rows // side
        axes[0] = axes[0] + case["first"]
        state["positions"] = torch.stack(axes, -1).to(torch.int32)
        state["sections"] = _sections(case)
        if case["packed"]:
            both = normal(b, tokens, (h + 2 * hk) * d)  # as a projection leaves queries, keys and values
            q = both[..., : h * d].unflatten(-1, (h, d))
            leaves = {"q": q, "k": both[..., h * d : (h + hk) * d].unflatten(-1, (hk, d))}
        else:
            leaves = {"q": normal(b, tokens, h, d), "k": normal(b, tokens, hk, d)}
        out = None
        state["grad"] = (normal(b, tokens, h, d), normal(b, tokens, hk, d))
    else:
        b, nq, nk, h, hk, d = (case[x] for x in ("batch", "nq", "nk", "heads", "kv_heads", "dim"))
        if case["packed"]:
            both = normal(b, nq, 2 * (h + 2 * hk) * d)
            q, k, v = both.split([2 * h * d, 2 * hk * d, 2 * hk * d], -1)
            leaves = {"q": q.unflatten(-1, (2 * h, d)), "k": k.unflatten(-1, (2 * hk, d)), "v": v.unflatten(-1, (hk, 2 * d))}
        else:
            leaves = {"q": normal(b, nq, 2 * h, d), "k": normal(b, nk, 2 * hk, d), "v": normal(b, nk, hk, 2 * d)}
        leaves["lam"] = (0.5 + 0.2 * torch.rand(h, device="cuda", generator=gen)).to(dtype)
        state["kv_lengths"] = torch.tensor(_kv_lengths(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        state["q_start"] = torch.tensor(_q_start(case), dtype=torch.int32, device="cuda") if case["causal"] else None
        out = (b, nq, h, 2 * d)
    if case["train"]:
        leaves = {name: t.detach().requires_grad_() for name, t in leaves.items()}
        if out is not None:
            state["grad"] = normal(*out)
    state["leaves"] = leaves
    return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    op = state["case"]["op"]
    if own:
        return {"linear": _own_linear, "rotary": _own_rotary, "attention": _own_attention}[op](state)
    with torch.no_grad():
        return {"linear": _plain_linear, "rotary": _plain_rotary, "attention": _plain_attention}[op](state)


def _with_gradients(state, out, grad):
    if not state["case"]["train"]:
        return {"out": out}
    leaves = state["leaves"]
    grads = torch.autograd.grad(out, list(leaves.values()), grad)
    return {"out": out, "grads": dict(zip(leaves, grads))}


def _own_linear(state):
    from bndm_amd import tokens

    leaves = state["leaves"]
    out = tokens.linear(leaves["x"], leaves["weight"], leaves.get("bias"), activation=state["case"]["act"] or None,
                        residual=leaves.get("residual"))
    return _with_gradients(state, out, state["grad"])


def _own_rotary(state):
    from bndm_amd import tokens

    out = tokens.rotary(state["leaves"]["q"], state["leaves"]["k"], state["positions"], state["sections"],
                        interleaved=state["case"]["interleaved"])
    return _with_gradients(state, out, state["grad"])


def _own_attention(state):
    from bndm_amd import tokens

    leaves = state["leaves"]
    out = tokens.differential_attention(leaves["q"], leaves["k"], leaves["v"], leaves["lam"], causal=state["case"]["causal"],
                                        q_start=state["q_start"], kv_lengths=state["kv_lengths"])
    return _with_gradients(state, out, state["grad"])


def _plain_linear(state):
    case, leaves = state["case"], state["leaves"]
    x, w = leaves["x"].float(), leaves["weight"].float()
    dtype = leaves["x"].dtype
    z = x @ w.t()
    if case["bias"]:
        z = z + leaves["bias"].float()
    if case["act"] == "silu":
        s = 1 / (1 + torch.exp(-z))
        y, slope = z * s, s * (1 + z * (1 - s))
    elif case["act"] == "gelu":
        c = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        y, slope = z * c, c + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    else:
        y, slope = z, None
    if case["residual"]:
        y = y + leaves["residual"].float()
    out = {"out": y.to(dtype)}
    if case["train"]:
        dy = state["grad"].float()
        dz = dy if slope is None else dy * slope
        grads = {"x": (dz @ w).to(dtype), "weight": (dz.t() @ x).to(dtype)}
        if case["bias"]:
            grads["bias"] = dz.sum(0).to(dtype)
        if case["residual"]:
            grads["residual"] = state["grad"]
        out["grads"] = grads
    return out


def _angles(case, positions):
    """Angle of every token and rotated pair [tokens, pairs], 64 bits: far positions times a frequency lose it in 32."""
    sections = torch.tensor(_sections(case), device=positions.device)
    axis = torch.repeat_interleave(torch.arange(len(sections), device=positions.device), sections)
    start = torch.cumsum(sections, 0) - sections
    within = torch.arange(len(axis), device=positions.device) - start[axis]
    frequency = 10000.0 ** (-within.double() / sections[axis].double())
    return positions.double()[:, axis] * frequency


def _plain_rotary(state):
    case = state["case"]
    angle = _angles(case, state["positions"])[:, None, :]
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()

    def turn(x, sin):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0::2], y[..., 1::2]
            return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2).to(x.dtype)
        a, b = y.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1).to(x.dtype)

    out = {"out": (turn(state["leaves"]["q"], sin), turn(state["leaves"]["k"], sin))}
    if case["train"]:
        out["grads"] = {"q": turn(state["grad"][0], -sin), "k": turn(state["grad"][1], -sin)}
    return out


def _visible(state, device):
    """[batch or 1, 1, nq, nk]: which keys a query sees."""
    case = state["case"]
    j = torch.arange(case["nk"], device=device)
    seen = torch.ones(1, 1, case["nq"], case["nk"], dtype=torch.bool, device=device)
    if case["ragged"]:
        seen = seen & (j < state["kv_lengths"][:, None, None, None])
    if case["causal"]:
        last = state["q_start"][:, None] + torch.arange(case["nq"], device=device)
        seen = seen & (j <= last[:, None, :, None])
    return seen


def _plain_attention(state):
    case, leaves = state["case"], state["leaves"]
    per, scale, dtype = case["heads"] // case["kv_heads"], case["dim"] ** -0.5, leaves["q"].dtype
    q = leaves["q"].float().transpose(1, 2)
    k = leaves["k"].float().unflatten(2, (-1, 2)).repeat_interleave(per, 2).flatten(2, 3).transpose(1, 2).contiguous()
    v = leaves["v"].float().repeat_interleave(per, 2).transpose(1, 2).contiguous()
    lam = leaves["lam"].float()[:, None, None]
    seen = _visible(state, q.device)
    s = (torch.matmul(q.contiguous(), k.transpose(-1, -2).contiguous()) * scale).masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    del s
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    del e
    p1, p2 = p[:, 0::2], p[:, 1::2]
    weights = p1 - lam * p2
    out = {"out": torch.matmul(weights, v).transpose(1, 2).to(dtype).contiguous()}
    if case["train"]:
        do = state["grad"].float().transpose(1, 2).contiguous()
        dv = torch.matmul(weights.transpose(-1, -2).contiguous(), do)
        dw = torch.matmul(do, v.transpose(-1, -2).contiguous())
        ds1 = p1 * (dw - (p1 * dw).sum(-1, keepdim=True))
        ds2 = -lam * p2 * (dw - (p2 * dw).sum(-1, keepdim=True))
        ds = torch.stack((ds1, ds2), 2).flatten(1, 2)
        dq = torch.matmul(ds, k) * scale
        dk = torch.matmul(ds.transpose(-1, -2).contiguous(), q.contiguous()) * scale
        b, nk = case["batch"], case["nk"]
        dk = dk.reshape(b, case["kv_heads"], per, 2, nk, -1).sum(2).flatten(1, 2)
        dv = dv.reshape(b, case["kv_heads"], per, nk, -1).sum(2)
        dlam = -(p2 * dw).sum((0, 2, 3))
        out["grads"] = {"q": dq.transpose(1, 2).to(dtype).contiguous(), "k": dk.transpose(1, 2).to(dtype).contiguous(),
                        "v": dv.transpose(1, 2).to(dtype).contiguous(), "lam": dlam.to(dtype)}
    return out


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "linear":
        rows, k, n = case["rows"], case["k"], case["n"]
        values = rows * k + n * k + rows * n + (n if case["bias"] else 0) + (rows * n if case["residual"] else 0)
        flops = 2 * rows * k * n
        if case["train"]:  # the output's gradient in; the input's, the weight's, the bias's out (the residual's is the output's)
            values += rows * n + rows * k + n * k + (n if case["bias"] else 0)
            flops *= 3
        return {"bytes": values * size, "flops": flops}
    if case["op"] == "rotary":
        tokens = math.prod(_sides(case))
        values = case["batch"] * tokens * (case["heads"] + case["kv_heads"]) * case["dim"] * (2 if case["train"] else 1)
        return {"bytes": 2 * values * size + tokens * 4 * len(_sides(case)), "flops": 3 * values}
    b, nq, nk, h, hk, d = (case[x] for x in ("batch", "nq", "nk", "heads", "kv_heads", "dim"))
    lengths = _kv_lengths(case) if case["ragged"] else [nk] * b
    pairs = 0
    for length, start in zip(lengths, _q_start(case)):
        pairs += sum(max(0, min(length, start + i + 1)) for i in range(nq)) if case["causal"] else nq * length
    keys = sum(lengths)
    values = b * nq * h * 4 * d + keys * hk * 4 * d + h
    flops = pairs * h * (4 * d + 4 * d)  # both maps' products of queries and keys, one product of their difference with the values
    if case["train"]:
        values += b * nq * h * 4 * d + b * nk * hk * 4 * d + h
        flops += pairs * h * 16 * d
    return {"bytes": values * size, "flops": flops}


# ------------------------------------------------------------------------------------------------ the values in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    leaves = {name: t.detach().double().requires_grad_(case["train"]) for name, t in state["leaves"].items()}
    grad = state["grad"]
    if case["op"] == "linear":
        out = torch.nn.functional.linear(leaves["x"], leaves["weight"], leaves.get("bias"))
        if case["act"] == "silu":
            out = out * torch.sigmoid(out)
        elif case["act"] == "gelu":
            out = out * 0.5 * torch.special.erfc(-out / math.sqrt(2.0))
        if case["residual"]:
            out = out + leaves["residual"]
        grad = grad.double() if case["train"] else None
    elif case["op"] == "rotary":
        start, turns = 0, []
        for axis, pairs in enumerate(state["sections"]):
            frequency = torch.exp(torch.arange(pairs, device="cuda").double() * (-math.log(10000.0) / pairs))
            turns.append(torch.polar(torch.ones(1, pairs, device="cuda").double(),
                                     torch.outer(state["positions"][:, axis].double(), frequency)))
        turns = torch.cat(turns, -1)[None, :, None, :]
        out = []
        for x in (leaves["q"], leaves["k"]):
            half = case["dim"] // 2
            pairs = x.unflatten(-1, (half, 2)) if case["interleaved"] else x.unflatten(-1, (2, half)).transpose(-1, -2)
            y = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turns)
            out.append((y if case["interleaved"] else y.transpose(-1, -2)).flatten(-2))
        out = tuple(out)
        grad = tuple(g.double() for g in grad)
    else:
        per, rows = case["heads"] // case["kv_heads"], []
        lengths = _kv_lengths(case) if case["ragged"] else [case["nk"]] * case["batch"]
        for b, (length, start) in enumerate(zip(lengths, _q_start(case))):
            heads = []
            for h in range(case["heads"]):
                maps = []
                for m in range(2):
                    q, k = leaves["q"][b, :, 2 * h + m], leaves["k"][b, :length, 2 * (h // per) + m]
                    s = q @ k.t() / math.sqrt(case["dim"])
                    if case["causal"]:
                        i = torch.arange(case["nq"], device="cuda")[:, None]
                        hidden = torch.arange(length, device="cuda") > start + i
                        s = s.masked_fill(hidden, -math.inf)
                        nothing = hidden.all(-1, keepdim=True)
                        s = torch.softmax(s.masked_fill(nothing, 0.0), -1).masked_fill(nothing, 0.0)
                    else:
                        s = torch.softmax(s, -1)
                    maps.append(s)
                heads.append((maps[0] - leaves["lam"][h] * maps[1]) @ leaves["v"][b, :length, h // per])
            rows.append(torch.stack(heads, 1))
        out = torch.stack(rows)
        grad = grad.double() if case["train"] else None
    if not case["train"]:
        return {"out": out}
    grads = torch.autograd.grad(out, list(leaves.values()), grad)
    return {"out": out, "grads": dict(zip(leaves, grads))}
