"""The work that the transformer operators of this framework are measured on: layer norm with its gradients, rotary positions
of several axes, cross attention to an encoder's states, and AdamW over many tensors.

`run` computes a case in elementary torch operations where `own` is false and through the framework's entry points
where it is true; `exact` gives the same from the definition in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BLOCK = 256          # values that share a scale in AdamW's 8-bit states; every tensor starts on a block of its own
TOP = 448.0          # largest e4m3 value
FLOOR = 2.0 ** -9    # smallest positive e4m3 value
TINY = 2.0 ** -100   # blocks whose largest value is below this are stored as zeros
BETAS, EPS, LR, DECAY = (0.9, 0.99), 1e-8, 1e-4, 1e-2


def listed():
    return [
        # normalising the tokens of one small request: latency
        {"name": "norm, one request", "op": "norm", "train": False, "rows": 16, "width": 512, "type": "bf16", "affine": True},
        # a training batch: 64 feature maps of 16 x 16 tokens
        {"name": "norm, training batch", "op": "norm", "train": True, "rows": 16384, "width": 1024, "type": "bf16", "affine": True},
        # full-precision rows of an odd width that no vector load fits
        {"name": "norm, odd rows in fp32", "op": "norm", "train": True, "rows": 4099, "width": 777, "type": "fp32", "affine": True},
        # the next token of 64 requests, each somewhere else in its volume
        {"name": "rotary, next tokens", "op": "rotary", "batch": 64, "length": 1, "heads": 32, "dim": 128, "type": "bf16", "interleaved": False, "far": 4096},
        # all tokens of a volume of slices, (slice, row, column)
        {"name": "rotary, volume", "op": "rotary", "batch": 1, "length": 65536, "heads": 16, "dim": 64, "type": "bf16", "interleaved": False, "far": 512},
        # one query row over a short encoder output: latency
        {"name": "cross, smallest", "op": "cross", "train": False, "batch": 1, "queries": 1, "keys": 77, "groups": 8, "share": 1, "dim": 64, "type": "bf16", "pad": "none"},
        # serving: one token for each of 16 requests, over the long encoder states of each
        {"name": "cross, next tokens", "op": "cross", "train": False, "batch": 16, "queries": 1, "keys": 4096, "groups": 8, "share": 4, "dim": 128, "type": "bf16", "pad": "lengths"},
        # decoder tokens over an encoder's feature map, whole
        {"name": "cross, prompt", "op": "cross", "train": False, "batch": 2, "queries": 4096, "keys": 4096, "groups": 16, "share": 1, "dim": 128, "type": "bf16", "pad": "none"},
        # training with shared key heads and a padded batch of an odd length
        {"name": "cross, training batch", "op": "cross", "train": True, "batch": 4, "queries": 1024, "keys": 1500, "groups": 4, "share": 4, "dim": 64, "type": "bf16", "pad": "lengths"},
        # training, nothing a multiple of a tile, keys dropped by a mask
        {"name": "cross, odd training", "op": "cross", "train": True, "batch": 3, "queries": 333, "keys": 777, "groups": 5, "share": 1, "dim": 80, "type": "fp16", "pad": "mask"},
        # the update of a network of many small tensors, states in 32 bits
        {"name": "adamw, many tensors", "op": "adamw", "tensors": 222, "smallest": 16, "largest": 524288, "type": "fp32", "bits": 32},
        # the update of a large network, states in 8 bits
        {"name": "adamw, large in 8 bits", "op": "adamw", "tensors": 48, "smallest": 1024, "largest": 16777216, "type": "bf16", "bits": 8},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["norm", "rotary", "cross", "cross", "adamw"])
    if op == "norm":
        width = _log(rng, 8, 8192)
        if rng.random() < 0.5:
            width = max(8, width // 8 * 8)
        return {"op": op, "train": rng.random() < 0.6, "rows": _log(rng, 1, min(65536, 2 ** 24 // width)), "width": width,
                "type": rng.choice(["bf16", "fp16", "fp32"]), "affine": rng.random() < 0.8}
    if op == "rotary":
        dim = rng.choice([32, 48, 64, 80, 96, 128])
        heads = rng.choice([1, 2, 3, 4, 8, 16, 32])
        batch = _log(rng, 1, 64)
        length = _log(rng, 1, max(1, 2 ** 25 // (batch * heads * dim)))
        return {"op": op, "batch": batch, "length": length, "heads": heads, "dim": dim, "type": rng.choice(["bf16", "fp16", "fp32"]),
                "interleaved": rng.random() < 0.4, "far": _log(rng, 16, 1000000)}
    if op == "cross":
        train = rng.random() < 0.5
        batch, groups, share = _log(rng, 1, 16), rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([1, 1, 2, 4, 8])
        queries = 1 if not train and rng.random() < 0.3 else _log(rng, 1, 4096)
        keys = _log(rng, 1, 8192)
        most = 2 ** 27 if train else 2 ** 28                     # pairs of a query and a key: the listed cases have up to 2^29
        while batch * groups * share * queries * keys > most:
            queries, keys = max(1, queries // 2), max(1, keys - keys // 3)
        return {"op": op, "train": train, "batch": batch, "queries": queries, "keys": keys, "groups": groups, "share": share,
                "dim": rng.choice([32, 40, 64, 64, 80, 96, 128, 128]), "type": rng.choice(["bf16", "bf16", "fp16"]),
                "pad": rng.choice(["none", "lengths", "mask"])}
    return {"op": op, "tensors": _log(rng, 1, 256), "smallest": _log(rng, 1, 4096), "largest": _log(rng, 4096, 1048576),
            "type": rng.choice(["bf16", "fp32"]), "bits": rng.choice([32, 8])}


# ---------------------------------------------------------------------------------------------------------- the inputs
def _sections(dim):
    """Pairs of the slice, row and column axis: a quarter for the slices, the rest in two."""
    pairs = dim // 2
    slices = pairs // 4
    rows = (pairs - slices) // 2
    return (slices, rows, pairs - slices - rows)


def _frequencies(dim, base=10000.0):
    return torch.cat([base ** (-torch.arange(n, dtype=torch.float64) / n) for n in _sections(dim)])


def _sizes(case):
    """Sizes spread evenly over the logarithm between the smallest and the largest tensor, in a mixed order."""
    ratio = math.log(case["largest"] / case["smallest"])
    return [max(1, int(round(case["smallest"] * math.exp(ratio * ((i * 0.6180339887498949) % 1.0))))) for i in range(case["tensors"])]


def _lengths(case, seed):
    """Valid keys of each request: the same set for every seed, in another order."""
    batch, keys = case["batch"], case["keys"]
    lengths = [max(1, keys - (keys * 3 // 4) * i // max(1, batch)) for i in range(batch)]
    order = torch.randperm(batch, generator=torch.Generator().manual_seed(seed)).tolist()
    return [lengths[i] for i in order]


def _valid(state):
    """[batch][keys] truth values, or None where every key counts."""
    if state["lengths"] is not None:
        return torch.arange(state["k"].shape[1], device=DEV)[None, :] < state["lengths"][:, None]
    return state["key_mask"]


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    kind = TYPES[case["type"]]

    def normal(*shape, to=kind, scale=1.0, shift=0.0):
        return (torch.randn(*shape, generator=gen, device=DEV) * scale + shift).to(to)

    state = {"case": case}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        state["x"] = normal(rows, width, scale=1.5, shift=0.25)
        state["w"] = normal(width, to=torch.float32, scale=0.2, shift=1.0) if case["affine"] else None
        state["b"] = normal(width, to=torch.float32, scale=0.2) if case["affine"] else None
        if case["train"]:
            state["dy"] = normal(rows, width)
        if own and case["train"]:
            for name in ("x", "w", "b"):
                if state[name] is not None:
                    state[name].requires_grad_()
    elif case["op"] == "rotary":
        shape = (case["batch"], case["length"])
        state["x"] = normal(*shape, case["heads"], case["dim"])
        state["positions"] = torch.randint(0, case["far"], (*shape, 3), generator=gen, device=DEV, dtype=torch.int32)
        state["sections"] = _sections(case["dim"])
        state["freqs"] = _frequencies(case["dim"]).to(DEV)
    elif case["op"] == "cross":
        heads = case["groups"] * case["share"]
        state["q"] = normal(case["batch"], case["queries"], heads, case["dim"])
        state["k"] = normal(case["batch"], case["keys"], case["groups"], case["dim"])
        state["v"] = normal(case["batch"], case["keys"], case["groups"], case["dim"])
        state["lengths"] = state["key_mask"] = None
        if case["pad"] == "lengths":
            state["lengths"] = torch.tensor(_lengths(case, seed), dtype=torch.int32, device=DEV)
        elif case["pad"] == "mask":
            state["key_mask"] = torch.rand(case["batch"], case["keys"], generator=gen, device=DEV) < 0.8
        if case["train"]:
            state["dout"] = normal(case["batch"], case["queries"], heads, case["dim"])
            if own:
                for name in ("q", "k", "v"):
                    state[name].requires_grad_()
    else:
        sizes = _sizes(case)
        starts, blocks = [], 0
        for n in sizes:
            starts.append(blocks * BLOCK)
            blocks += -(-n // BLOCK)
        # one buffer holds the parameters, each tensor from a block's start on; what lies between them stays zero
        at = torch.zeros(blocks * BLOCK, dtype=torch.bool)
        for start, n in zip(starts, sizes):
            at[start:start + n] = True
        at = at.to(DEV)
        many = blocks * BLOCK
        state["p"] = normal(many, scale=0.05) * at.to(kind)
        flat = normal(many, scale=1e-3)
        state["grads"] = [flat[start:start + n].clone() for start, n in zip(starts, sizes)]
        state["gaps"] = [torch.zeros(-n % BLOCK, dtype=kind, device=DEV) for n in sizes]
        m = normal(many, to=torch.float32, scale=4e-4) * at
        r = (normal(many, to=torch.float32, scale=3e-4).abs() + 6e-4) * at
        state["step"] = torch.full((), 100, dtype=torch.int32, device=DEV)
        if case["bits"] == 32:
            state["m"], state["v"] = m, r * r
        else:
            state["m"], state["ms"] = _to_8(m, False)
            state["r"], state["rs"] = _to_8(r, True)
        if own:
            from reid_gan_amd import optim
            state["params"] = [torch.nn.Parameter(state["p"][start:start + n]) for start, n in zip(starts, sizes)]
            for p, g in zip(state["params"], state["grads"]):
                p.grad = g
            opt = optim.AdamW(state["params"], lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, state_bits=case["bits"])
            saved = {}
            for i, (start, n) in enumerate(zip(starts, sizes)):
                blk = slice(start // BLOCK, start // BLOCK + -(-n // BLOCK))
                saved[i] = {"step": state["step"]}
                if case["bits"] == 32:
                    saved[i].update(exp_avg=state["m"][start:start + n], exp_avg_sq=state["v"][start:start + n])
                else:
                    saved[i].update(exp_avg=state["m"][start:start + n], exp_avg_scale=state["ms"][blk],
                                    exp_avg_sq_root=state["r"][start:start + n], exp_avg_sq_root_scale=state["rs"][blk])
            opt.load_state_dict({"state": saved, "param_groups": opt.state_dict()["param_groups"]})
            state["opt"] = opt
    return state


# ------------------------------------------------------------------------------------------------------ the plain forms
def _norm(state):
    x, w, b = state["x"], state["w"], state["b"]
    f = x.float()
    centred = f - f.mean(-1, keepdim=True)
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    hat = centred * rstd
    y = (hat if w is None else hat * w + b).to(x.dtype)
    if "dy" not in state:
        return y
    dy = state["dy"].float()
    dhat = dy if w is None else dy * w
    dx = rstd * (dhat - dhat.mean(-1, keepdim=True) - hat * (dhat * hat).mean(-1, keepdim=True))
    out = [y, dx.to(x.dtype)]
    if w is not None:
        out += [(dy * hat).sum(0), dy.sum(0)]
    return out


def _rotary(state):
    x, pos, freqs = state["x"], state["positions"], state["freqs"]
    axis = torch.cat([torch.full((n,), a, dtype=torch.long, device=DEV) for a, n in enumerate(state["sections"])])
    angle = pos.double()[:, :, axis] * freqs                              # far positions: 64 bits
    cos, sin = torch.cos(angle).float()[:, :, None], torch.sin(angle).float()[:, :, None]
    f = x.float()
    if state["case"]["interleaved"]:
        a, b = f[..., 0::2], f[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2).to(x.dtype)
    a, b = f.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1).to(x.dtype)


def _cross(state):
    q, k, v = state["q"], state["k"], state["v"]
    batch, queries, heads, dim = q.shape
    keys, groups = k.shape[1], k.shape[2]
    rows = heads // groups * queries

    def fold(t):       # the heads that share a key head, one after the other
        return t.float().reshape(batch, queries, groups, heads // groups, dim).permute(0, 2, 3, 1, 4).reshape(batch * groups, rows, dim)

    def unfold(t):
        return t.reshape(batch, groups, heads // groups, queries, dim).permute(0, 3, 1, 2, 4).reshape(batch, queries, heads, dim)

    qf = fold(q)
    kf, vf = (t.float().permute(0, 2, 1, 3).reshape(batch * groups, keys, dim) for t in (k, v))
    scale = 1.0 / math.sqrt(dim)
    s = torch.bmm(qf, kf.transpose(1, 2).contiguous()) * scale
    valid = _valid(state)
    if valid is not None:
        hidden = ~valid[:, None, None, :].expand(batch, groups, 1, keys).reshape(batch * groups, 1, keys)
        s = s.masked_fill(hidden, -math.inf)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    e = torch.exp(s - top)
    total = e.sum(-1, keepdim=True)
    p = e / torch.where(total > 0, total, torch.ones_like(total))
    o = torch.bmm(p, vf)
    out = unfold(o).to(q.dtype)
    if "dout" not in state:
        return out
    do = fold(state["dout"])
    dv = torch.bmm(p.transpose(1, 2).contiguous(), do)
    ds = p * (torch.bmm(do, vf.transpose(1, 2).contiguous()) - (do * o).sum(-1, keepdim=True))
    dq = torch.bmm(ds, kf) * scale
    dk = torch.bmm(ds.transpose(1, 2).contiguous(), qf) * scale
    back = [t.reshape(batch, groups, keys, dim).permute(0, 2, 1, 3).contiguous().to(k.dtype) for t in (dk, dv)]
    return [out, unfold(dq).to(q.dtype), *back]


def _to_8(values, positive):
    """Codes and scales of values held in 8 bits, a scale for each block; a positive root never becomes zero."""
    rows = values.view(-1, BLOCK)
    top = rows.abs().amax(-1, keepdim=True)
    some = ~(top < TINY)                                                  # (NaN: the whole block says so)
    scale = torch.where(some, top * (1.0 / TOP), torch.zeros_like(top))
    coded = (rows * torch.where(some, torch.reciprocal(top) * TOP, torch.zeros_like(top))).to(torch.float8_e4m3fn).float()
    if positive:
        coded = torch.where(some & (rows > 0), coded.clamp(min=FLOOR), coded)
    return coded.to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _from_8(codes, scale):
    return (codes.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _adamw(state):
    g = torch.cat([t for pair in zip(state["grads"], state["gaps"]) for t in pair]).float()
    small = state["case"]["bits"] == 8
    state["step"] += 1
    t = state["step"].double()
    rate, root = (LR / (1.0 - BETAS[0] ** t)).float(), (1.0 / torch.sqrt(1.0 - BETAS[1] ** t)).float()
    if small:
        m, r = _from_8(state["m"], state["ms"]), _from_8(state["r"], state["rs"])
        v = r * r
    else:
        m, v = state["m"], state["v"]
    m = m * BETAS[0] + g * (1.0 - BETAS[0])
    v = v * BETAS[1] + g * g * (1.0 - BETAS[1])
    r = torch.sqrt(v)
    p = state["p"].float()
    state["p"].copy_(p * (1.0 - LR * DECAY) - rate * (m / (r * root + EPS)))
    if not small:
        state["m"].copy_(m)
        state["v"].copy_(v)
        return [state["p"], state["m"], state["v"]]
    for name, values in (("m", m), ("r", r)):
        codes, scale = _to_8(values, name == "r")
        state[name].copy_(codes)
        state[name + "s"].copy_(scale)
    return [state["p"], state["m"], state["ms"], state["r"], state["rs"]]


# ---------------------------------------------------------------------------------------- the framework's entry points
def _own(state):
    from reid_gan_amd import attention
    op = state["case"]["op"]
    if op == "norm":
        y = attention.layer_norm(state["x"], state["w"], state["b"], eps=1e-5)
        if "dy" not in state:
            return y
        leaves = [state[n] for n in ("x", "w", "b") if state[n] is not None]
        return [y, *torch.autograd.grad(y, leaves, state["dy"])]
    if op == "rotary":
        return attention.rotary(state["x"], state["positions"], state["freqs"], state["sections"], interleaved=state["case"]["interleaved"])
    if op == "cross":
        out = attention.cross_attention(state["q"], state["k"], state["v"], lengths=state["lengths"], key_mask=state["key_mask"])
        if "dout" not in state:
            return out
        return [out, *torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["dout"])]
    state["opt"].step()
    held = state["opt"].flat_state()[0]
    names = ("exp_avg", "exp_avg_sq") if state["case"]["bits"] == 32 else ("exp_avg", "exp_avg_scale", "exp_avg_sq_root", "exp_avg_sq_root_scale")
    return [state["p"], *(held[n] for n in names)]


def run(state):
    if own:
        return _own(state)
    return {"norm": _norm, "rotary": _rotary, "cross": _cross, "adamw": _adamw}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------------------------- what it costs
def work(case):
    size = 4 if case["type"] == "fp32" else 2
    if case["op"] == "norm":
        many = case["rows"] * case["width"]
        return {"bytes": many * size * (4 if case["train"] else 2) + case["width"] * 16, "flops": many * (20 if case["train"] else 8)}
    if case["op"] == "rotary":
        tokens = case["batch"] * case["length"]
        many = tokens * case["heads"] * case["dim"]
        return {"bytes": 2 * many * size + tokens * 12, "flops": 3 * many}
    if case["op"] == "cross":
        batch, heads = case["batch"], case["groups"] * case["share"]
        keys = {"none": batch * case["keys"], "lengths": sum(_lengths(case, 0)), "mask": int(0.8 * batch * case["keys"])}[case["pad"]]
        pairs = keys * heads * case["queries"]
        asked, held = batch * heads * case["queries"] * case["dim"], keys * case["groups"] * case["dim"]
        if case["train"]:
            return {"bytes": size * (4 * asked + 4 * held), "flops": 14 * pairs * case["dim"]}
        return {"bytes": size * (2 * asked + 2 * held), "flops": 4 * pairs * case["dim"]}
    many = sum(_sizes(case))
    return {"bytes": many * (3 * size + (16 if case["bits"] == 32 else 4)), "flops": many * 15}


# ------------------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    state = prepare({**case}, seed)
    op = case["op"]
    if op == "norm":
        x = state["x"].detach().double()
        width = x.shape[1]
        mu = x.sum(1, keepdim=True) / width
        spread = torch.sqrt(((x - mu) ** 2).sum(1, keepdim=True) / width + 1e-5)
        hat = (x - mu) / spread
        w = state["w"].detach().double() if case["affine"] else torch.ones(width, dtype=torch.float64, device=DEV)
        y = hat * w + state["b"].detach().double() if case["affine"] else hat
        if not case["train"]:
            return y
        dy = state["dy"].double()
        into = dy * w
        dx = (into - into.sum(1, keepdim=True) / width - hat * ((into * hat).sum(1, keepdim=True) / width)) / spread
        return [y, dx] + ([(dy * hat).sum(0), dy.sum(0)] if case["affine"] else [])
    if op == "rotary":
        x, pos, freqs = state["x"].double(), state["positions"].double(), state["freqs"]
        half = case["dim"] // 2
        out, at = torch.empty_like(x), 0
        for axis, n in enumerate(_sections(case["dim"])):
            for j in range(at, at + n):
                one, two = (2 * j, 2 * j + 1) if case["interleaved"] else (j, half + j)
                turn = torch.polar(torch.ones_like(pos[:, :, axis]), pos[:, :, axis] * freqs[j])[:, :, None]
                z = torch.complex(x[..., one], x[..., two]) * turn
                out[..., one], out[..., two] = z.real, z.imag
            at += n
        return out
    if op == "cross":
        q, k, v = (state[n].detach().double() for n in ("q", "k", "v"))
        share, scale = case["share"], case["dim"] ** -0.5
        grads = [torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
        out = torch.zeros_like(q)
        valid = _valid(state)
        for b in range(case["batch"]):
            keep = slice(None) if valid is None else valid[b].nonzero()[:, 0]
            for h in range(case["groups"] * share):
                kb, vb, qb = k[b, keep, h // share], v[b, keep, h // share], q[b, :, h]
                if kb.shape[0] == 0:
                    continue
                p = torch.softmax(qb @ kb.T * scale, -1)
                out[b, :, h] = p @ vb
                if case["train"]:
                    do = state["dout"][b, :, h].double()
                    dp = do @ vb.T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                    grads[0][b, :, h] = ds @ kb
                    grads[1][b, keep, h // share] += ds.T @ qb
                    grads[2][b, keep, h // share] += p.T @ do
        return [out, *grads] if case["train"] else out
    g = torch.zeros_like(state["p"], dtype=torch.float64)
    at = 0
    for t in state["grads"]:
        g[at:at + t.numel()] = t.double()
        at += -(-t.numel() // BLOCK) * BLOCK
    if case["bits"] == 32:
        m, v = state["m"].double(), state["v"].double()
    else:
        m = (state["m"].double().view(-1, BLOCK) * state["ms"].double()[:, None]).view(-1)
        v = (state["r"].double().view(-1, BLOCK) * state["rs"].double()[:, None]).view(-1) ** 2
    m = BETAS[0] * m + (1 - BETAS[0]) * g
    v = BETAS[1] * v + (1 - BETAS[1]) * g * g
    step = int(state["step"]) + 1
    m_hat, v_hat = m / (1 - BETAS[0] ** step), v / (1 - BETAS[1] ** step)
    p = state["p"].detach().double() * (1 - LR * DECAY) - LR * m_hat / (v_hat.sqrt() + EPS)
    if case["bits"] == 32:
        return [p, m, v]
    # the codes follow from the 32-bit values, roundings included: only their scales have a value of their own here
    tops = [t.abs().view(-1, BLOCK).amax(1) / TOP for t in (m, v.sqrt())]
    return [p, None, tops[0], None, tops[1]]
