"""Token operators (layer norm, rotary positions, cross attention, AdamW over many tensors) against plain formulas in 64
bits on the same inputs.

Tolerances are bounds, element by element, of what the kernels round: u is half a step of the type a value is stored in
(bf16 2^-8, fp16 2^-11, fp32 2^-24), e = 2^-24 bounds one fp32 operation, and a sum of n terms formed in any order is off
by at most n e times the sum of the terms' absolute values.  Each test states the sum it bounds."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu

from reid_gan_amd import attention, ops, optim

DEV = "cuda"
E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
GRAPHS = []            # captured graphs stay until the process ends
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38}      # below this a type has no relative precision
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def new_graph():
    GRAPHS.append(torch.cuda.CUDAGraph())
    return GRAPHS[-1]


def normal(g, *shape, to=F32, scale=1.0, shift=0.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale + shift).to(to)


def within(got, want, tol, what):
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~((got - want).abs() <= tol)
    if bool(bad.any()):
        i = int(bad.reshape(-1).nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} values off, the first at {i}: "
                             f"{got.reshape(-1)[i].item()} for {want.reshape(-1)[i].item()}, allowed {tol.expand_as(want).reshape(-1)[i].item():.3g}")


# --------------------------------------------------------------------------- layer norm
def ln_exact(x, w, b, eps=1e-5):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    sigma = ((x - mu).square().mean(-1, keepdim=True) + eps).sqrt()
    hat = (x - mu) / sigma
    y = hat if w is None else hat * w.double()
    return (y if b is None else y + b.double()), hat, sigma


def ln_check(x, w, b, dy, y, dx, dw, db, what):
    """The row sums run over at most 32 terms per lane and 10 steps across lanes and waves (wider rows: C / 1024 terms per
    thread): (42 + C / 1024) e relative to the mean of |x|, which sigma divides; the centred squares likewise, to hat."""
    C = x.shape[-1]
    n = 64 + C / 1024
    want, hat, sigma = ln_exact(x, w, b)
    wide = 1 + x.double().abs().amax(-1, keepdim=True) / sigma            # error of x - mean, in units of sigma, is n e wide
    wd = torch.ones(C, device=DEV, dtype=torch.float64) if w is None else w.double()
    u = U[x.dtype]
    hat_off = n * E * (hat.abs() + wide)
    within(y, want, u * want.abs() + 2 * hat_off * wd.abs() + 4 * E * (want.abs() + (0 if b is None else b.double().abs())) + TINY[x.dtype], what + " y")
    if dy is None:
        return
    g = dy.double() * wd
    m1, m2 = g.mean(-1, keepdim=True), (g * hat).mean(-1, keepdim=True)
    want = (g - m1 - hat * m2) / sigma
    ga, gh = g.abs().mean(-1, keepdim=True), (g * hat).abs().mean(-1, keepdim=True)
    off = (n * E * (g.abs() + ga + 2 * hat.abs() * gh) + hat_off * (m2.abs() + gh) + (hat.abs() + 1) * (g.abs() * hat_off).mean(-1, keepdim=True)) / sigma
    within(dx, want, u * want.abs() + 2 * off + 2 * n * E * wide * want.abs() + TINY[x.dtype], what + " dx")
    rows = x.numel() // C
    steps = 64 + rows / 128                                               # rows per block and per lane group, plus the joins
    flat = lambda t: t.reshape(-1, C)
    if dw is not None:
        want = flat(dy.double() * hat).sum(0)
        within(dw, want, U[dw.dtype] * want.abs() + flat(dy.double().abs() * (steps * E * hat.abs() + hat_off)).sum(0) + TINY[dw.dtype], what + " dw")
    if db is not None:
        want = flat(dy.double()).sum(0)
        within(db, want, U[db.dtype] * want.abs() + steps * E * flat(dy.double().abs()).sum(0) + TINY[db.dtype], what + " db")


@pytest.mark.parametrize("rows, C", [(1, 1), (1, 8), (3, 7), (5, 33), (7, 64), (33, 100), (4, 256), (129, 512), (3, 777), (260, 1024),
                                     (2, 2047), (9, 2048), (3, 4099), (5, 8192), (2, 16384), (2, 40001)])
@pytest.mark.parametrize("kind, wkind", [(BF16, F32), (F16, F16), (F32, F32), (BF16, BF16), (F16, F32)])
def test_layer_norm(rows, C, kind, wkind):
    g = gen(rows * 100003 + C)
    x, dy = normal(g, rows, C, to=kind, scale=2.0, shift=1.0), normal(g, rows, C, to=kind)
    w, b = normal(g, C, to=wkind, scale=0.3, shift=1.0), normal(g, C, to=wkind)
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    y = attention.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    ln_check(x.detach(), w.detach(), b.detach(), dy, y, dx, dw, db, f"{rows} x {C} {kind}")
    with torch.no_grad():
        assert torch.equal(y, attention.layer_norm(x, w, b))


@pytest.mark.parametrize("affine", ["none", "weight", "bias"])
def test_layer_norm_parts(affine):
    g = gen(3)
    x, dy = normal(g, 2, 3, 5, 96, to=BF16), normal(g, 2, 3, 5, 96, to=BF16)
    w = normal(g, 96).requires_grad_() if affine == "weight" else None
    b = normal(g, 96).requires_grad_() if affine == "bias" else None
    x.requires_grad_()
    y = attention.layer_norm(x, w, b)
    leaves = [t for t in (x, w, b) if t is not None]
    got = dict(zip((id(t) for t in leaves), torch.autograd.grad(y, leaves, dy)))
    ln_check(x.detach(), None if w is None else w.detach(), None if b is None else b.detach(), dy, y, got[id(x)], got.get(id(w)), got.get(id(b)), affine)


def test_layer_norm_large_mean_keeps_its_precision():
    g = gen(4)
    x = normal(g, 64, 1024, scale=1e-2, shift=100.0)
    ln_check(x, None, None, None, attention.layer_norm(x), None, None, None, "mean 1e4 sigma")


def test_layer_norm_views_and_rows_it_must_not_touch():
    g = gen(5)
    buf = normal(g, 9, 200, to=BF16)
    x = buf[:, 3:131]                                                     # unaligned rows inside a wider buffer
    assert torch.equal(attention.layer_norm(x), attention.layer_norm(x.contiguous()))
    t = normal(g, 16, 12, 64, to=BF16).transpose(0, 1)
    assert torch.equal(attention.layer_norm(t), attention.layer_norm(t.contiguous()))
    e = normal(g, 1, 64, to=BF16).expand(7, 64)
    assert torch.equal(attention.layer_norm(e), attention.layer_norm(e.contiguous()))
    s = normal(g, 8, 64, to=BF16)[:, ::2]
    assert torch.equal(attention.layer_norm(s), attention.layer_norm(s.contiguous()))
    one = normal(g, 64, to=BF16)
    assert torch.equal(attention.layer_norm(one), attention.layer_norm(one[None])[0])
    out = torch.full((12, 80), 7.0, dtype=BF16, device=DEV)
    ops.layer_norm_fwd(x[:, :64], None, None, out[2:11, 8:72], None, 1e-5)
    assert torch.equal(out[2:11, 8:72], attention.layer_norm(x[:, :64]))
    out[2:11, 8:72] = 7.0
    assert bool((out == 7.0).all())
    assert attention.layer_norm(torch.empty(0, 8, device=DEV)).shape == (0, 8)
    w = torch.ones(8, device=DEV, requires_grad=True)
    attention.layer_norm(torch.empty(0, 8, device=DEV), w).sum().backward()
    assert torch.equal(w.grad, torch.zeros(8, device=DEV))


def test_layer_norm_gradient_against_differences():
    """<gradient, d> against (L(x + h d) - L(x - h d)) / 2h of the formula in 64 bits: the difference is off by O(h^2)."""
    g = gen(6)
    x, w, b, dy = normal(g, 12, 40), normal(g, 40), normal(g, 40), normal(g, 12, 40)
    leaves = [t.requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(attention.layer_norm(x, w, b), leaves, dy)
    for i, grad in enumerate(grads):
        d = normal(g, *grad.shape).double()
        args = [t.detach().double() for t in leaves]
        loss = lambda t: (ln_exact(*[t if j == i else a for j, a in enumerate(args)])[0] * dy.double()).sum()
        want = (loss(args[i] + 1e-4 * d) - loss(args[i] - 1e-4 * d)) / 2e-4
        assert abs(((grad.double() * d).sum() - want).item()) <= 1e-5 * (grad.double() * d).abs().sum().item()


# --------------------------------------------------------------------------- rotary positions
def rot_exact(x, pos, freqs, sections, interleaved=False, inverse=False):
    x, pairs = x.double(), sum(sections)
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], device=x.device)
    t = pos.double()[..., axis] * freqs * (-1 if inverse else 1)
    c, s = t.cos().unsqueeze(-2), t.sin().unsqueeze(-2)
    y = x.clone()
    one = x[..., 0:2 * pairs:2] if interleaved else x[..., :pairs]
    two = x[..., 1:2 * pairs:2] if interleaved else x[..., pairs:2 * pairs]
    mag = x.abs().clone()
    a, b, m = one * c - two * s, two * c + one * s, one.abs() + two.abs()
    if interleaved:
        y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2] = a, b
        mag[..., 0:2 * pairs:2], mag[..., 1:2 * pairs:2] = m, m
    else:
        y[..., :pairs], y[..., pairs:2 * pairs] = a, b
        mag[..., :pairs], mag[..., pairs:2 * pairs] = m, m
    return y, mag


@pytest.mark.parametrize("shape, sections", [((1, 1, 1, 2), (1,)), ((2, 5, 3, 64), (8, 12, 12)), ((3, 17, 1, 128), (16, 24, 24)), ((1, 7, 4, 80), (10, 15, 15)),
                                             ((2, 3, 2, 96), (4, 4, 4, 4)), ((1, 9, 5, 22), (3, 0, 5)), ((2, 1, 32, 128), (64,)), ((1, 2000, 2, 48), (8, 16)),
                                             ((1, 3, 2, 512), (64, 96, 96))])
@pytest.mark.parametrize("kind", [BF16, F16, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("ptype", [torch.int32, torch.int64, F32])
def test_rotary(shape, sections, kind, interleaved, ptype):
    """A pair's result is two products and a sum (3 e of |x0| + |x1|) of cosines and sines that are off by at most pi 2^-25
    (the rounding of the half turns to fp32) plus 2 e: 8 e together."""
    g = gen(sum(shape))
    x = normal(g, *shape, to=kind).requires_grad_()
    pos = torch.randint(-50, 1000000, (*shape[:2], len(sections)), generator=g, device=DEV).to(ptype)
    if ptype is F32:
        pos = pos / 64
    freqs = attention.rotary_frequencies(sections)
    y = attention.rotary(x, pos, freqs, sections, interleaved)
    want, mag = rot_exact(x.detach(), pos, freqs, sections, interleaved)
    within(y, want, U[kind] * want.abs() + 8 * E * mag + TINY[kind], "forward")
    dy = normal(g, *shape, to=kind)
    dx, = torch.autograd.grad(y, x, dy)
    want, mag = rot_exact(dy, pos, freqs, sections, interleaved, True)
    within(dx, want, U[kind] * want.abs() + 8 * E * mag + TINY[kind], "backward")
    with torch.no_grad():
        z = x.detach().clone()
        assert attention.rotary(z, pos, freqs, sections, interleaved, out=z) is z
        assert torch.equal(z, y)


def test_rotary_views():
    g = gen(8)
    sections, freqs = (8, 12, 12), attention.rotary_frequencies((8, 12, 12))
    qkv = normal(g, 2, 6, 5, 3 * 64 + 1, to=BF16)
    grid = torch.stack(torch.meshgrid(torch.arange(1), torch.arange(2), torch.arange(3), indexing="ij"), -1).view(6, 3).to(DEV)
    x = qkv[..., 64:128]
    want = attention.rotary(x.contiguous(), grid.expand(2, 6, 3).contiguous(), freqs, sections)
    assert torch.equal(attention.rotary(x, grid, freqs, sections), want)               # positions shared by the batch
    odd = qkv[..., 65:129]                                                              # rows that start at odd elements
    assert torch.equal(attention.rotary(odd, grid, freqs, sections), attention.rotary(odd.contiguous(), grid, freqs, sections))
    heads_first = x.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(attention.rotary(heads_first, grid, freqs, sections), want)
    before = qkv.clone()
    attention.rotary(x, grid, freqs, sections, out=x)                                   # in place inside a wider buffer
    assert torch.equal(qkv[..., 64:128], want)
    assert torch.equal(qkv[..., :64], before[..., :64]) and torch.equal(qkv[..., 128:], before[..., 128:])
    reduced = normal(g, 2, 6, 64, 5, to=BF16).transpose(2, 3)
    assert torch.equal(attention.rotary(reduced, grid, freqs, sections), attention.rotary(reduced.contiguous(), grid, freqs, sections))
    assert attention.rotary(torch.empty(2, 0, 4, 64, device=DEV), torch.empty(2, 0, 3, device=DEV), freqs, sections).shape == (2, 0, 4, 64)


# --------------------------------------------------------------------------- cross attention
def hidden(B, Lk, lengths, mask):
    ok = torch.ones(B, Lk, dtype=torch.bool, device=DEV)
    if lengths is not None:
        ok &= torch.arange(Lk, device=DEV)[None] < lengths[:, None]
    if mask is not None:
        ok &= mask.bool()
    return ok


def cross_exact(q, k, v, lengths=None, mask=None, scale=None, dout=None):
    """Results in 64 bits (out, lse, dq, dk, dv), and bounds of what the kernels may be off by.

    Scores: D products and as many sums, off by (D + 8) e of the sum of |q||k| scale, which is the relative error of a
    weight; the row's sum of weights is off by as much and by n e more.  Weights enter the products rounded to the type
    (u); fp16 loses all relative precision below 2^-24 of the largest.  dS = P (dP - Dl), with Dl formed from the stored o
    (u of |dO||o|), is rounded to the type again."""
    B, Lq, H, D = q.shape
    G = H // k.shape[2]
    u, tiny = U[q.dtype], TINY[q.dtype]
    scale = D ** -0.5 if scale is None else scale
    ok = hidden(B, k.shape[1], lengths, mask)
    qd, kd, vd = (t.detach().double().transpose(1, 2) for t in (q, k, v))
    kd, vd = (torch.where(ok[:, None, :, None], t, 0.0).repeat_interleave(G, 1) for t in (kd, vd))
    s = (qd @ kd.transpose(-1, -2) * scale).masked_fill(~ok[:, None, None], -torch.inf)
    lse = s.logsumexp(-1)
    p = torch.where(torch.isinf(lse)[..., None], 0.0, (s - lse[..., None]).exp())
    o = p @ vd
    sabs = (qd.abs() @ kd.abs().transpose(-1, -2) * scale).amax(-1, keepdim=True) if k.shape[1] else torch.zeros_like(o[..., :1])
    n = k.shape[1]
    rel = 2 * (D + 8) * E * sabs + (n + 64) * E                                    # relative error of P
    tol_o = u * o.abs() + (u + 2 * rel) * (p @ vd.abs()) + 2 * tiny * (1 + vd.abs().sum(-2, keepdim=True))
    tol_lse = (D + 8) * E * sabs[..., 0] + (n + 64) * E + 4 * E * lse.abs().nan_to_num(posinf=0)
    out = {"out": (o, tol_o), "lse": (lse, tol_lse)}
    if dout is not None:
        do = dout.double().transpose(1, 2)
        dp, dl = do @ vd.transpose(-1, -2), (do * o).sum(-1, keepdim=True)
        ds = p * (dp - dl)
        dp_off = (D + 8) * E * (do.abs() @ vd.abs().transpose(-1, -2)) + (do.abs() * (tol_o + u * o.abs() + (D + 8) * E * o.abs())).sum(-1, keepdim=True)
        ds_off = (u + 2 * rel + 4 * E) * ds.abs() + p * dp_off + 2.0 ** -36 * ds.abs().amax()
        rows = Lq * G
        fold = lambda t: t.unflatten(1, (-1, G)).sum(2)
        dq = ds @ kd * scale
        dk, dv = fold(ds.transpose(-1, -2) @ qd) * scale, fold(p.transpose(-1, -2) @ do)
        acc = (n + rows + 64) * E
        tol_dq = u * dq.abs() + scale * ((ds_off + acc * ds.abs()) @ kd.abs()) + tiny
        tol_dk = u * dk.abs() + scale * fold((ds_off + acc * ds.abs()).transpose(-1, -2) @ qd.abs()) + tiny
        tol_dv = u * dv.abs() + fold(((u + 2 * rel + acc) * p + 2.0 ** -39).transpose(-1, -2) @ do.abs()) + tiny
        out.update(dq=(dq, tol_dq), dk=(dk, tol_dk), dv=(dv, tol_dv))
    return {key: (val if key == "lse" else tuple(t.transpose(1, 2) for t in val)) for key, val in out.items()}


def cross_check(q, k, v, lengths=None, mask=None, scale=None, train=True, seed=1):
    what = f"q {tuple(q.shape)} k {tuple(k.shape)} {q.dtype}"
    dout = normal(gen(seed), *q.shape, to=q.dtype) if train else None
    want = cross_exact(q, k, v, lengths, mask, scale, dout)
    if not train:
        with torch.no_grad():
            within(attention.cross_attention(q, k, v, lengths, mask, scale), *want["out"], what)
        return
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = attention.cross_attention(*leaves, lengths, mask, scale)
    grads = torch.autograd.grad(out, leaves, dout)
    within(out, *want["out"], what + " out")
    for name, got in zip(("dq", "dk", "dv"), grads):
        within(got, *want[name], f"{what} {name}")
    ok = hidden(q.shape[0], k.shape[1], lengths, mask)
    for t in grads[1:]:
        assert bool((t[~ok] == 0).all()), "gradients of hidden keys"


def qkv(seed, B, Lq, Lk, H, Hk, D, kind, scale=1.0):
    g = gen(seed)
    return normal(g, B, Lq, H, D, to=kind, scale=scale), normal(g, B, Lk, Hk, D, to=kind), normal(g, B, Lk, Hk, D, to=kind)


SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 77, 8, 8, 64), (1, 33, 1, 2, 1, 32), (2, 3, 5, 4, 2, 40), (1, 64, 64, 2, 2, 64), (2, 65, 63, 3, 3, 96),
          (1, 100, 129, 6, 2, 128), (3, 127, 200, 2, 1, 80), (1, 300, 257, 4, 4, 24), (2, 129, 640, 8, 1, 128), (1, 5, 1000, 16, 4, 56),
          (1, 700, 40, 2, 2, 72), (1, 1, 3001, 8, 2, 128), (4, 2, 2500, 4, 4, 64), (1, 1025, 513, 1, 1, 120), (1, 31, 700, 1, 1, 104)]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kind", [BF16, F16])
def test_cross_attention(shape, kind):
    cross_check(*qkv(sum(shape), *shape, kind))


@pytest.mark.parametrize("shape", SHAPES[1:])
@pytest.mark.parametrize("kind", [BF16, F16])
def test_cross_attention_without_gradients(shape, kind):
    cross_check(*qkv(sum(shape) + 1, *shape, kind), train=False)


@pytest.mark.parametrize("shape", [(4, 40, 130, 4, 2, 64), (4, 1, 130, 4, 2, 128), (4, 200, 64, 2, 2, 32), (4, 3, 1100, 6, 2, 96), (4, 257, 900, 2, 1, 128)])
@pytest.mark.parametrize("kind", [BF16, F16])
def test_cross_attention_lengths_and_masks(shape, kind):
    q, k, v = qkv(sum(shape), *shape, kind)
    Lk = shape[2]
    lengths = torch.tensor([Lk, 0, 1, Lk // 2 + 3], dtype=torch.int32, device=DEV)
    mask = torch.rand(4, Lk, generator=gen(9), device=DEV) < 0.7
    mask[2] = False                                                         # an entry that the mask leaves empty
    mask[3, :Lk // 3] = False                                               # left padding: whole tiles without a key
    bad_k, bad_v = k.clone(), v.clone()
    for lens, m in ((lengths, None), (None, mask), (lengths, mask.to(torch.uint8) * 255)):
        cross_check(q, k, v, lens, m)
        cross_check(q, k, v, lens, m, train=False)
        ok = hidden(4, Lk, lens, m)
        bad_k.copy_(k), bad_v.copy_(v)
        bad_k[~ok], bad_v[~ok] = float("nan"), float("inf")                # what hidden keys hold has no effect
        cross_check(q, bad_k, bad_v, lens, m)
    out = torch.autograd.grad(attention.cross_attention(q.requires_grad_(), k, v, lengths), q, torch.ones_like(q))[0]
    assert bool((out[1] == 0).all()) and bool((attention.cross_attention(q.detach(), k, v, lengths)[1] == 0).all())
    over = torch.tensor([Lk + 5, -3, 2 ** 31 - 1, Lk], dtype=torch.int32, device=DEV)       # lengths past the ends are cut
    like = torch.tensor([Lk, 0, Lk, Lk], dtype=torch.int32, device=DEV)
    assert torch.equal(attention.cross_attention(q.detach(), k, v, over), attention.cross_attention(q.detach(), k, v, like))


@pytest.mark.parametrize("keys", [8192, 16384 + 100, 40000])
def test_cross_attention_many_shares_of_the_keys(keys):
    """One row over enough keys that they are shared out to up to 64 blocks, some of them without a key that counts."""
    q, k, v = qkv(keys, 2, 1, keys, 4, 1, 64, BF16)
    cross_check(q, k, v, train=False)
    cross_check(q, k, v, torch.tensor([keys, 33], dtype=torch.int32, device=DEV), train=False)
    mask = torch.zeros(2, keys, dtype=torch.bool, device=DEV)
    mask[0, keys - 5:] = True
    mask[1, ::97] = True
    cross_check(q, k, v, None, mask, train=False)


@pytest.mark.parametrize("dim", [32, 64, 128])
@pytest.mark.parametrize("sizes", [(3, 700, 300, 4, 2), (5, 260, 1500, 2, 1), (1, 3000, 70, 4, 4), (2, 1100, 130, 12, 3),
                                   (300, 40, 65, 2, 2)])
def test_cross_attention_gradients_of_the_keys_in_shares(sizes, dim):
    """The keys' gradients where their rows are dealt out to blocks: few and many keys, entries without any between others,
    whole 64s without keys behind the last one, more entries than are counted."""
    B, Lq, Lk, H, G = sizes
    q, k, v = qkv(dim + B, B, Lq, Lk, H, G, dim, BF16)
    cross_check(q, k, v)
    lengths = torch.randint(0, Lk + 1, (B,), generator=gen(97), device=DEV, dtype=torch.int32)
    lengths[B // 2] = 0
    lengths[B - 1] = Lk if B > 1 else Lk // 2
    cross_check(q, k, v, lengths)
    lengths.zero_()
    cross_check(q, k, v, lengths)


@pytest.mark.parametrize("kind", [BF16, F16])
def test_cross_attention_one_key_has_no_score_gradient(kind):
    """With one key that counts the weight is 1 whatever the score: dq and dk are zeros but for the fp32 rounding of dP - Dl
    (2 D e of |dO||v|), and the key's dv is the sum of dO.  Also where the keys are shared out over several blocks."""
    for Lq, Lk in ((20, 1), (3, 1200), (200, 700)):
        q, k, v = (t.requires_grad_() for t in qkv(18, 2, Lq, Lk, 4, 2, 64, kind))
        lengths = torch.ones(2, dtype=torch.int32, device=DEV)
        d = normal(gen(19), *q.shape, to=kind)
        dq, dk, dv = torch.autograd.grad(attention.cross_attention(q, k, v, lengths), (q, k, v), d)
        size = (d.double().abs().sum(-1) * 5 * 5 * 128 * E).max().item() * 5 * 0.125
        assert dq.abs().max().item() <= size and dk[:, 0].abs().max().item() <= size * Lq * 2
        want = d.double().transpose(1, 2).unflatten(1, (2, 2)).sum((2, 3))
        within(dv[:, 0], want, U[kind] * want.abs() + 4 * Lq * E * d.double().abs().transpose(1, 2).unflatten(1, (2, 2)).sum((2, 3)), "dv")


def test_cross_attention_small_weights_add_up_in_half_precision():
    """40000 keys of weight 2^-25 beside one of weight 1: together 2^-10 of the result.  A weight's rounding is at most
    2^-25 of its scale, 2^7 here: 40000 * 2^-32 in all, beside the roundings of the scores (e of |s| < 32) and the result."""
    n = 40000
    for Lq in (2, 70):                                                        # (single tokens, tiles)
        q, k, v = (torch.zeros(1, m, 1, 64, dtype=F16, device=DEV) for m in (Lq, n, n))
        q[..., 0], k[:, 0, :, 0], v[:, 1:] = 1, 17.328, 1
        s = k[0, 0, 0, 0].double()
        w = (n - 1) * torch.exp(-s)
        want = (w / (1 + w)).expand(1, Lq, 1, 64)
        got = attention.cross_attention(q, k, v, scale=1.0)
        within(got, want, n * 2 ** -32 + want * (U[F16] + 64 * E + n * E), "small weights")


def test_cross_attention_no_keys_no_queries_no_batch():
    for B, Lq, Lk in ((2, 3, 0), (2, 0, 3), (0, 3, 3)):
        q, k, v = (t.requires_grad_() for t in qkv(1, B, Lq, Lk, 4, 2, 64, BF16))
        out = attention.cross_attention(q, k, v)
        assert out.shape == q.shape and bool((out == 0).all())
        for g, t in zip(torch.autograd.grad(out, (q, k, v), torch.ones_like(out)), (q, k, v)):
            assert g.shape == t.shape and bool((g == 0).all())


@pytest.mark.parametrize("kind", [BF16, F16])
@pytest.mark.parametrize("Lq", [1, 50])
def test_cross_attention_values_that_are_large_or_not_numbers(kind, Lq):
    q, k, v = qkv(5, 1, Lq, 300, 2, 2, 64, kind, scale=30.0)                # one key takes almost all the weight
    cross_check(q, k, v)
    k2 = k.clone()
    k2[0, 200:] *= 20                                                       # the maximum rises late
    cross_check(q, k2, v, train=False)
    cross_check(q * 0, k, v)                                                # all weights equal
    q2 = q.clone()
    q2[0, 0, 1, 3] = float("nan")
    out = attention.cross_attention(q2, k, v)
    assert bool(out[0, 0, 1].isnan().all()) and torch.equal(out[0, :, 0], attention.cross_attention(q, k, v)[0, :, 0])
    v2 = v.clone()
    v2[0, 17, 0, 5] = float("inf")
    out = attention.cross_attention(q * 0, k, v2)
    assert bool(out[0, :, 0, 5].isinf().all()) and bool(out[0, :, 0, :5].isfinite().all())
    cross_check(q / 30, k, v, scale=2.5)


@pytest.mark.parametrize("power", [-16, -8, 8])
def test_cross_attention_fp16_gradients_of_any_size(power):
    """dS spans more than fp16 does: many keys make it small, large gradients make it large.  Gradients that are exact at both
    sizes give results that differ by the power of two alone, up to what fp16 can store of them."""
    q, k, v = (t.requires_grad_() for t in qkv(6, 1, 40, 4000, 2, 2, 64, F16))
    dout = torch.randint(-3, 4, (1, 40, 2, 64), generator=gen(7), device=DEV).to(F16)
    a = torch.autograd.grad(attention.cross_attention(q, k, v), (q, k, v), dout)
    b = torch.autograd.grad(attention.cross_attention(q, k, v), (q, k, v), dout * 2.0 ** power)
    for x, y in zip(a, b):
        x, y = x.double(), y.double() * 2.0 ** -power
        assert bool(y.isfinite().all())
        assert bool(((x - y).abs() <= 2.0 ** -10 * x.abs() + 2.0 ** -24 * (1 + 2.0 ** -power)).all())


def test_cross_attention_layouts():
    g = gen(10)
    q = normal(g, 2, 4, 70, 64, to=BF16).transpose(1, 2)                    # [batch][heads][tokens] storage
    kv = normal(g, 2, 90, 2, 2, 64, to=BF16)
    k, v = kv[:, :, 0], kv[:, :, 1]                                         # interleaved keys and values
    want = attention.cross_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(attention.cross_attention(q, k, v), want)
    wide = normal(g, 2, 90, 2, 67, to=BF16)
    odd = wide[..., 1:65]                                                   # not aligned: copied
    assert torch.equal(attention.cross_attention(q, odd, odd), attention.cross_attention(q, odd.contiguous(), odd.contiguous()))
    one = k[:1].expand(2, -1, -1, -1)                                       # one encoder output for the whole batch
    assert torch.equal(attention.cross_attention(q, one, one), attention.cross_attention(q, one.contiguous(), one.contiguous()))
    leaf = k[:1].clone().requires_grad_()
    full = leaf.detach().expand(2, -1, -1, -1).contiguous().requires_grad_()
    d = normal(g, 2, 70, 4, 64, to=BF16)
    gl, = torch.autograd.grad(attention.cross_attention(q, leaf.expand(2, -1, -1, -1), v), leaf, d)
    gf, = torch.autograd.grad(attention.cross_attention(q, full, v), full, d)
    within(gl, gf.double().sum(0, keepdim=True), 2 * U[BF16] * gf.double().abs().sum(0, keepdim=True), "gradient of a broadcast input")
    m = (torch.rand(90, generator=g, device=DEV) < 0.5)[None].expand(2, 90)
    assert torch.equal(attention.cross_attention(q, k, v, key_mask=m), attention.cross_attention(q, k, v, key_mask=m.contiguous()))
    m2 = (torch.rand(90, 2, generator=g, device=DEV) < 0.5).t()
    assert torch.equal(attention.cross_attention(q, k, v, key_mask=m2), attention.cross_attention(q, k, v, key_mask=m2.contiguous()))
    same = attention.cross_attention(k, k, k)                               # the same tensor three times
    assert torch.equal(same, attention.cross_attention(k, k.clone(), k.clone()))


def test_cross_attention_results_and_log_sums_go_where_they_are_told():
    q, k, v = qkv(11, 2, 33, 300, 4, 2, 64, BF16)
    buf = torch.full((2, 35, 4, 72), 7.0, dtype=BF16, device=DEV)
    lse = torch.empty(2, 4, 33, dtype=F32, device=DEV)
    out = buf[:, 1:34, :, :64]
    n = ops.xattn_fwd_scratch_floats(2, 33, 300, 4, 2, 64)
    ops.xattn_fwd(q, k, v, out, lse, 0.125, scratch=torch.empty(max(n, 1), device=DEV))
    want = cross_exact(q, k, v, scale=0.125)
    within(out, *want["out"], "out")
    within(lse, *want["lse"], "lse")
    out.fill_(7.0)
    assert bool((buf == 7.0).all())
    empty = torch.zeros(2, dtype=torch.int32, device=DEV)
    ops.xattn_fwd(q, k, v, out, lse, 0.125, lengths=empty, scratch=torch.empty(max(n, 1), device=DEV))
    assert bool((lse == -torch.inf).all()) and bool((out == 0).all())


def test_cross_attention_offsets_past_32_bits():
    """Keys of one entry span over 2^32 bytes: token strides of 2^22 elements, 600 keys (5 GB)."""
    g = gen(12)
    big = torch.empty(600 * (1 << 22), dtype=BF16, device=DEV)
    k = big.as_strided((1, 600, 2, 64), (0, 1 << 22, 64, 1))
    v = big.as_strided((1, 600, 2, 64), (0, 1 << 22, 64, 1), 4096)
    k.copy_(normal(g, 1, 600, 2, 64)), v.copy_(normal(g, 1, 600, 2, 64))
    for Lq in (1, 70):
        q = normal(g, 1, Lq, 4, 64, to=BF16)
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        d = normal(g, 1, Lq, 4, 64, to=BF16)
        got = attention.cross_attention(*leaves)
        want = cross_exact(q, k, v, dout=d)
        within(got, *want["out"], "out")
        for name, t in zip(("dq", "dk", "dv"), torch.autograd.grad(got, leaves, d)):
            within(t, *want[name], name)


def test_cross_attention_gradient_against_differences():
    """<gradient, d> against differences of the formula in 64 bits, within the bounds of each gradient."""
    q, k, v = qkv(13, 2, 9, 21, 4, 2, 32, BF16)
    lengths = torch.tensor([21, 13], dtype=torch.int32, device=DEV)
    dout = normal(gen(14), *q.shape, to=BF16)
    leaves = [t.requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(attention.cross_attention(*leaves, lengths), leaves, dout)
    bounds = cross_exact(q, k, v, lengths, dout=dout)
    args = [t.detach().double() for t in leaves]

    def loss(*a):
        ok = hidden(2, 21, lengths, None)
        s = (a[0].transpose(1, 2) @ a[1].transpose(1, 2).repeat_interleave(2, 1).transpose(-1, -2) * 32 ** -0.5).masked_fill(~ok[:, None, None], -torch.inf)
        return ((s.softmax(-1) @ a[2].transpose(1, 2).repeat_interleave(2, 1)).transpose(1, 2) * dout.double()).sum()
    for i, (grad, name) in enumerate(zip(grads, ("dq", "dk", "dv"))):
        d = normal(gen(15 + i), *grad.shape).double()
        move = lambda h: loss(*[a + h * d if j == i else a for j, a in enumerate(args)])
        want = (move(1e-4) - move(-1e-4)) / 2e-4
        assert abs(((grad.double() * d).sum() - want).item()) <= (bounds[name][1] * d.abs()).sum().item() + 1e-5 * abs(want.item())


def test_cross_attention_is_the_same_every_time():
    q, k, v = (t.requires_grad_() for t in qkv(16, 2, 300, 700, 8, 2, 64, BF16))
    d = normal(gen(17), *q.shape, to=BF16)
    first = torch.autograd.grad(attention.cross_attention(q, k, v), (q, k, v), d)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(attention.cross_attention(q, k, v), (q, k, v), d)))


# --------------------------------------------------------------------------- streams, graphs, threads
class Sub(torch.Tensor):
    """A subclass keeps a call from going straight to the kernels: the checks and copies in Python see it."""


@pytest.mark.parametrize("plain", [True, False])
def test_calls_and_gradients_by_both_ways(plain):
    """The direct calls and the Python functions behind them give the same bits; neither has a second derivative."""
    g = gen(90)
    as_ = (lambda t: t) if plain else (lambda t: t.as_subclass(Sub))
    bare = lambda t: t.as_subclass(torch.Tensor)
    x, w, b, dy = normal(g, 40, 96, to=BF16), normal(g, 96), normal(g, 96), normal(g, 40, 96, to=BF16)
    r, pos, sections = normal(g, 2, 7, 4, 64, to=BF16), torch.randint(0, 99, (2, 7, 3), generator=g, device=DEV), (8, 12, 12)
    freqs = attention.rotary_frequencies(sections)
    q, k, v = qkv(91, 2, 50, 70, 4, 2, 64, BF16)
    d = normal(g, 2, 50, 4, 64, to=BF16)
    mask = torch.rand(2, 70, generator=g, device=DEV) < 0.5
    calls = [(lambda *t: attention.layer_norm(*t), (x, w, b), dy), (lambda t: attention.rotary(t, pos, freqs, sections), (r,), r.clone()),
             (lambda *t: attention.cross_attention(*t, key_mask=mask), (q, k, v), d)]
    for call, inputs, grad in calls:
        stats = []
        for other in (False, True):
            leaves = [(t if other else as_(t)).detach().clone().requires_grad_() for t in inputs]
            out = call(*leaves)
            grads = torch.autograd.grad(out, leaves, grad, retain_graph=True)
            with torch.no_grad():
                again = call(*leaves)
            assert torch.equal(bare(out.detach()), bare(again))
            stats.append([bare(out.detach()), *(bare(t) for t in grads)])
            some = torch.autograd.grad(out, leaves[:1], grad)                       # only one of the gradients
            assert torch.equal(bare(some[0]), stats[-1][1])
        assert all(torch.equal(a, c) for a, c in zip(*stats))
        leaves = [as_(t).detach().clone().requires_grad_() for t in inputs]
        first = torch.autograd.grad(call(*leaves), leaves, grad.detach().clone().requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError, match="twice"):
            first[0].float().sum().backward()


def test_two_streams_at_once():
    sets = [qkv(20 + i, 2, 1, 2000, 8, 2, 128, BF16) for i in range(2)]
    want = [attention.cross_attention(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(attention.cross_attention(*sets[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(want[i], t) for t in got[i])


def test_captured_forward_and_backward():
    """A captured step on the entry points of ops, replayed several times with eager work between, new inputs each time."""
    B, Lq, Lk, H, Hk, D, C = 2, 40, 700, 4, 2, 64, 256
    sections, freqs = (8, 12, 12), attention.rotary_frequencies((8, 12, 12))
    g = gen(30)
    x, w, b = normal(g, B * Lq, C, to=BF16), normal(g, C), normal(g, C)
    k, v = normal(g, B, Lk, Hk, D, to=BF16), normal(g, B, Lk, Hk, D, to=BF16)
    pos = torch.randint(0, 500, (B, Lq, 3), generator=g, device=DEV)
    dout = normal(g, B, Lq, H, D, to=BF16)
    like = lambda t: torch.empty_like(t)
    y, stats, q, out, dq, dk, dv, dy, dx = like(x), torch.empty(2, B * Lq, device=DEV), like(dout), like(dout), like(dout), like(k), like(v), like(x), like(x)
    lse, dw, db = torch.empty(B, H, Lq, device=DEV), like(w), like(b)
    s1 = torch.empty(max(1, ops.xattn_fwd_scratch_floats(B, Lq, Lk, H, Hk, D)), device=DEV)
    s2 = torch.empty(ops.xattn_bwd_scratch_floats(B, Lq, Lk, H, Hk, D), device=DEV)
    s3 = torch.empty(ops.layer_norm_bwd_scratch_floats(B * Lq, C, BF16), device=DEV)

    def step():
        ops.layer_norm_fwd(x, w, b, y, stats, 1e-5)
        ops.rotary(y.view(B, Lq, H, D), q, pos, freqs, sections, False, False)
        ops.xattn_fwd(q, k, v, out, lse, 0.125, scratch=s1)
        ops.xattn_bwd(dout, q, k, v, out, lse, dq, dk, dv, 0.125, s2)
        ops.rotary(dq, dy.view(B, Lq, H, D), pos, freqs, sections, False, True)
        ops.layer_norm_bwd(dy, x, w, stats, dx, dw, db, s3)
    results = (out, dx, dw, db, dk, dv)
    step()
    torch.cuda.synchronize()
    graph = new_graph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(normal(g, B * Lq, C)), k.copy_(normal(g, B, Lk, Hk, D)), dout.copy_(normal(g, B, Lq, H, D))
        for t in results:
            t.fill_(7.0)
        graph.replay()
        got = [t.clone() for t in results]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, t) for a, t in zip(got, results)), i


@pytest.mark.parametrize("Lq, Lk", [(1000, 700), (2, 1500), (300, 130)])
def test_captured_lengths_are_read_at_the_replay(Lq, Lk):
    """A replay takes the lengths and the mask as they are then - also those that leave an entry, or all, without keys."""
    B, H, Hk, D = 4, 8, 2, 64
    g = gen(98)
    q, k, v = qkv(99, B, Lq, Lk, H, Hk, D, BF16)
    dout, lengths = normal(g, B, Lq, H, D, to=BF16), torch.full((B,), Lk, dtype=torch.int32, device=DEV)
    mask = torch.ones(B, Lk, dtype=torch.bool, device=DEV)
    out, dq, dk, dv = (torch.empty_like(t) for t in (q, q, k, v))
    lse = torch.empty(B, H, Lq, device=DEV)
    s1 = torch.empty(max(1, ops.xattn_fwd_scratch_floats(B, Lq, Lk, H, Hk, D)), device=DEV)
    s2 = torch.empty(ops.xattn_bwd_scratch_floats(B, Lq, Lk, H, Hk, D), device=DEV)

    def step():
        ops.xattn_fwd(q, k, v, out, lse, 0.125, lengths, mask, s1)
        ops.xattn_bwd(dout, q, k, v, out, lse, dq, dk, dv, 0.125, s2, lengths, mask)
    step()
    torch.cuda.synchronize()
    graph = new_graph()
    with torch.cuda.graph(graph):
        step()
    for lens in ([Lk, 1, Lk // 2, 65], [0, 0, 0, 0], [0, Lk, 0, 33], [-5, Lk + 9, 64, 2]):
        lengths.copy_(torch.tensor(lens, dtype=torch.int32))
        mask.copy_(torch.rand(B, Lk, generator=g, device=DEV) < 0.7)
        for t in (out, dq, dk, dv, s1, s2):
            t.fill_(7.0)
        graph.replay()
        leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
        want = attention.cross_attention(*leaves, lengths, mask, 0.125)
        grads = torch.autograd.grad(want, leaves, dout)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip((out, dq, dk, dv), (want, *grads))), lens


def test_gradients_under_capture_are_refused():
    q, k, v = qkv(31, 1, 4, 8, 2, 2, 64, BF16)
    graph, kept = new_graph(), []
    leaf = q.clone().requires_grad_()
    x, w = normal(gen(1), 4, 64), torch.ones(64, device=DEV, requires_grad=True)
    with torch.cuda.graph(graph):
        kept.append(attention.cross_attention(q, k, v))
        with pytest.raises(RuntimeError, match="graph capture"):
            attention.cross_attention(leaf, k, v)
        with pytest.raises(RuntimeError, match="graph capture"):
            attention.layer_norm(x, w)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept[0], attention.cross_attention(q, k, v))


def test_what_is_written_in_place_counts_as_written():
    """A graph that saved a tensor refuses to use it once rotary(out=...) or an optimizer step has written it."""
    g = gen(92)
    sections = (8, 12, 12)
    x, pos, freqs = normal(g, 1, 3, 2, 64), torch.ones(1, 3, 3, device=DEV, dtype=torch.int32), attention.rotary_frequencies(sections)
    w = torch.nn.Parameter(normal(g, 64))
    y = (x * w).sum()
    with torch.no_grad():
        attention.rotary(x, pos, freqs, sections, out=x)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()
    for contiguous in (True, False):
        p = torch.nn.Parameter(normal(g, 8, 8))
        loss = p.square().sum()
        p.grad = torch.ones(8, 8, device=DEV) if contiguous else torch.ones(8, 8, device=DEV).t()
        optim.AdamW([p]).step()
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


def test_adamw_refuses_parameters_that_share_memory():
    buf = torch.zeros(100, device=DEV)
    a, b = torch.nn.Parameter(buf[:60]), torch.nn.Parameter(buf[40:])
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    with pytest.raises(ValueError, match="share memory"):
        optim.AdamW([a, b]).step()
    c, d = torch.nn.Parameter(buf[:40]), torch.nn.Parameter(buf[40:])         # (side by side is fine)
    c.grad, d.grad = torch.ones_like(c), torch.ones_like(d)
    optim.AdamW([c, d], lr=1.0, weight_decay=0.0).step()
    assert (buf < -0.9).all()


def test_lazily_negated_views_are_not_taken_for_their_storage():
    c = torch.randn(4, 64, dtype=torch.complex64, generator=gen(93), device=DEV).conj().imag
    assert c.is_neg()
    with pytest.raises(ValueError, match="resolve_neg"):
        attention.layer_norm(c)
    p = torch.nn.Parameter(torch.zeros(4, 64, device=DEV))
    q = torch.nn.Parameter(torch.zeros(4, 64, device=DEV))
    p.grad, q.grad = c, c.resolve_neg().contiguous()
    optim.AdamW([p], lr=1.0).step(), optim.AdamW([q], lr=1.0).step()
    assert torch.equal(p, q)


def test_layer_norm_rows_far_from_zero_with_odd_channels():
    """Where no channel is, mean * rstd would be infinite: it must not reach the sums of the backward pass."""
    for C in (13, 1001, 5003):
        x = torch.full((3, C), 2e38 / C * 0.5, device=DEV).requires_grad_()
        d = normal(gen(94), 3, C)
        dx, = torch.autograd.grad(attention.layer_norm(x), x, d)
        assert torch.isfinite(dx).all(), C


# --------------------------------------------------------------------------- AdamW
def plain_codes(t, root):
    """Codes and scales of flat values in blocks of 256, every operation rounded to 32 bits by itself."""
    rows = torch.nn.functional.pad(t.reshape(-1), (0, -t.numel() % 256)).view(-1, 256)
    top = rows.abs().amax(1, keepdim=True)
    none = top < 2.0 ** -100
    scale = torch.where(none, torch.zeros_like(top), top * (1.0 / 448.0))
    inv = torch.where(none, torch.zeros_like(top), top.reciprocal() * 448.0)
    c = (rows * inv).to(torch.float8_e4m3fn).float()
    if root:
        c = torch.where(~none & (rows > 0), c.clamp(min=2.0 ** -9), c)
    return c.view(-1)[:t.numel()].view(t.shape), scale.view(-1)


def plain_values(c, scale):
    return (torch.nn.functional.pad(c.reshape(-1), (0, -c.numel() % 256)).view(-1, 256) * scale[:, None]).view(-1)[:c.numel()].view(c.shape)


def adamw_reference(p, g, state, lr, betas, eps, wd, bits):
    """One step in torch's elementwise operations on fp32 values; returns p (64 bits) and the new state."""
    b1, b2 = betas
    t = state["t"] + 1
    if bits == 8:
        m, r = plain_values(*state["m"]), plain_values(*state["r"])
        v = r * r
    else:
        m, v = state["m"], state["v"]
    g = g.float()
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    r = torch.sqrt(v)
    mh, rh = m.double() / (1 - b1 ** t), r.double() / (1 - b2 ** t) ** 0.5
    update = lr * mh / (rh + eps)
    new = p.double() * (1 - lr * wd) - update
    state = {"t": t, "m": plain_codes(m, False), "r": plain_codes(r, True)} if bits == 8 else {"t": t, "m": m, "v": v}
    return new, update.abs(), state


SIZES = [(1,), (255,), (256,), (257,), (3, 5, 7), (64, 1, 3, 3), (4096,), (4097,), (0,), (10000,), (2, 128, 129)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw(kind, bits):
    """Moments have the bits of the plain evaluation (each operation rounded by itself); p is off by the roundings of its own
    chain: 3 e of p, 12 e of the update, and its type's u."""
    g = gen(40)
    lr, betas, eps, wd = 3e-3, (0.9, 0.99), 1e-8, 0.1
    params = [torch.nn.Parameter(normal(g, *s, to=kind)) for s in SIZES]
    buf = normal(g, 700, to=kind)
    params += [torch.nn.Parameter(buf[3:600]), torch.nn.Parameter(buf[601:602])]            # tensors at odd addresses
    before = buf.clone()
    opt = optim.AdamW(params, lr=lr, betas=betas, eps=eps, weight_decay=wd, state_bits=bits)
    zero = lambda p: ((torch.zeros(p.shape, device=DEV), torch.zeros(-(-p.numel() // 256), device=DEV)) if bits == 8 else torch.zeros(p.shape, device=DEV))
    states = [{"t": 0, "m": zero(p), "r": zero(p), "v": zero(p)} for p in params]
    for step in range(4):
        for i, p in enumerate(params):
            p.grad = None if (step + i) % 5 == 4 else normal(g, *p.shape, to=kind, scale=10.0 ** (i % 7 - 4))
            if p.grad is not None and i == 4:
                p.grad = torch.zeros_like(p)
            if p.grad is not None and p.dim() == 3 and step == 1:
                p.grad = p.grad.transpose(0, 2).contiguous().transpose(0, 2)                # not contiguous
        old = [p.detach().clone() for p in params]
        opt.step()
        for i, p in enumerate(params):
            if p.grad is None or p.numel() == 0:
                assert torch.equal(p, old[i])
                continue
            want, update, states[i] = adamw_reference(old[i], p.grad, states[i], lr, betas, eps, wd, bits)
            within(p.detach(), want, U[kind] * want.abs() + 3 * E * old[i].double().abs() + 12 * E * update + 1e-38, f"p {i} step {step}")
            s = opt.state[p]
            assert int(s["step"]) == states[i]["t"]
            if bits == 32:
                assert torch.equal(s["exp_avg"], states[i]["m"]) and torch.equal(s["exp_avg_sq"], states[i]["v"]), (i, step)
            else:
                for name, (codes, scale) in (("exp_avg", states[i]["m"]), ("exp_avg_sq_root", states[i]["r"])):
                    assert torch.equal(s[name].float(), codes) and torch.equal(s[name + "_scale"], scale), (i, step, name)
    assert torch.equal(buf[:3], before[:3]) and torch.equal(buf[600:601], before[600:601]) and torch.equal(buf[602:], before[602:])
    for flat in opt.flat_state():
        for name, t in flat.items():
            if name.endswith("_scale"):
                continue
            t, at = t.float().clone(), 0
            for p in params:
                t[at:at + p.numel()] = 0
                at += -(-p.numel() // 256) * 256
            assert bool((t == 0).all()), name                                                # what lies between the tensors


def test_adamw_code_borders():
    """Every midpoint between two e4m3 values and its neighbours rounds as torch's conversion does (ties to even)."""
    codes = torch.arange(0, 127, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn).float()
    mids = (codes[1:] + codes[:-1]) / 2
    vals = torch.cat([codes, mids, torch.nextafter(mids, mids * 0), torch.nextafter(mids, mids + 500)])
    vals = torch.cat([vals, -vals])
    vals = torch.nn.functional.pad(vals, (0, -vals.numel() % 255))
    rows = torch.cat([torch.full((vals.numel() // 255, 1), 448.0, device=DEV), vals.view(-1, 255)], 1)      # scale of one
    p = torch.nn.Parameter(torch.zeros(rows.numel(), device=DEV))
    opt = optim.AdamW([p], lr=0.0, betas=(0.0, 0.0), state_bits=8)
    p.grad = rows.reshape(-1).clone()
    opt.step()
    s = opt.state[p]
    assert bool((s["exp_avg_scale"] == 1).all())
    assert torch.equal(s["exp_avg"].float(), rows.reshape(-1).to(torch.float8_e4m3fn).float())
    want, scale = plain_codes(rows.reshape(-1).square().sqrt(), True)
    assert torch.equal(s["exp_avg_sq_root"].float(), want) and torch.equal(s["exp_avg_sq_root_scale"], scale)
    assert bool((s["exp_avg_sq_root"].float()[p.grad != 0] > 0).all())                       # a root is never lost


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_not_numbers_and_tiny_gradients(bits):
    p = torch.nn.Parameter(torch.ones(1024, device=DEV))
    opt = optim.AdamW([p], lr=1e-2, weight_decay=0.0, state_bits=bits)
    p.grad = torch.ones_like(p)
    p.grad[700] = float("nan")
    p.grad[256:512] = 1e-32                                                                   # under the smallest block scale
    opt.step()
    assert bool(p[700].isnan()) and int(p.isnan().sum()) == 1
    p.grad = torch.ones_like(p)
    opt.step()
    bad = p.isnan()
    assert bool(bad[700]) and not bool(bad[:512].any()) and int(bad.sum()) == (1 if bits == 32 else 256)


def test_adamw_follows_torch():
    """32-bit moments against torch.optim.AdamW in 64 bits over 20 steps with a schedule: each step adds at most 3 e of p and
    12 e of its update."""
    g = gen(42)
    base = [normal(g, 300, 7), normal(g, 41)]
    mine, theirs = [torch.nn.Parameter(t.clone()) for t in base], [torch.nn.Parameter(t.double()) for t in base]
    groups = lambda ps: [{"params": [ps[0]]}, {"params": [ps[1]], "weight_decay": 0.0, "lr": 5e-3}]
    a = optim.AdamW(groups(mine), lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    b = torch.optim.AdamW(groups(theirs), lr=1e-2, betas=(0.9, 0.95), weight_decay=0.1)
    sa, sb = torch.optim.lr_scheduler.ExponentialLR(a, 0.9), torch.optim.lr_scheduler.ExponentialLR(b, 0.9)
    for _ in range(20):
        for p, q in zip(mine, theirs):
            p.grad = normal(g, *p.shape)
            q.grad = p.grad.double()
        a.step(), b.step(), sa.step(), sb.step()
    for p, q in zip(mine, theirs):
        within(p.detach(), q.detach(), 20 * (4 * E * q.detach().abs() + 40 * E * 1e-2 * torch.ones_like(q)), "p")


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_state_travels(bits):
    g = gen(43)
    make = lambda: [torch.nn.Parameter(normal(gen(44), 500, 3)), torch.nn.Parameter(normal(gen(45), 17, to=BF16))]
    grads = [[normal(g, 500, 3), normal(g, 17, to=BF16)] for _ in range(4)]

    def run(opt, ps, steps):
        for s in steps:
            for p, d in zip(ps, grads[s]):
                p.grad = d
            opt.step()
    one = make()
    a = optim.AdamW(one, state_bits=bits)
    run(a, one, range(4))
    two = make()
    b = optim.AdamW(two, state_bits=bits)
    run(b, two, range(2))
    saved, at = copy.deepcopy(b.state_dict()), [p.detach().clone() for p in two]
    three = make()
    c = optim.AdamW(three, state_bits=bits, lr=7.0)
    run(c, three, [3])                                                      # (a used optimizer takes the state over)
    for p, t in zip(three, at):
        p.data.copy_(t)
    pointers = [t.data_ptr() for f in c.flat_state() for t in f.values()]
    c.load_state_dict(saved)
    assert pointers == [t.data_ptr() for f in c.flat_state() for t in f.values()]
    run(c, three, [2, 3])
    four = copy.deepcopy(two)
    assert all(torch.equal(p, q) for p, q in zip(one, three)) and all(torch.equal(p, q) for p, q in zip(two, four))
    with pytest.raises(ValueError, match="bits"):
        optim.AdamW(make(), state_bits=40 - bits).load_state_dict(saved)
    bad = copy.deepcopy(saved)
    bad["state"][0]["exp_avg"] = bad["state"][0]["exp_avg"][:3]
    with pytest.raises(ValueError, match="shape"):
        c.load_state_dict(bad)


def test_adamw_takes_over_a_torch_state():
    p, q = torch.nn.Parameter(normal(gen(46), 100)), torch.nn.Parameter(normal(gen(46), 100))
    a, b = optim.AdamW([p], lr=1e-2), torch.optim.AdamW([q], lr=1e-2)
    for i in range(3):
        q.grad = normal(gen(50 + i), 100)
        b.step()
    p.data.copy_(q.data)
    a.load_state_dict(b.state_dict())
    p.grad = q.grad = normal(gen(60), 100)
    a.step(), b.step()
    within(p.detach(), q.detach(), 8 * E * q.detach().double().abs() + 40 * E * 1e-2, "p")


def test_adamw_captured():
    """A captured step replays with the gradients at their addresses and goes on counting; parameters that moved are
    followed by the next eager step, and a capture that would need a new table is refused."""
    ps = [torch.nn.Parameter(normal(gen(47), n)) for n in (5000, 3)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = optim.AdamW(ps, lr=1e-2, state_bits=8), optim.AdamW(qs, lr=1e-2, state_bits=8)
    grads = [torch.zeros_like(p) for p in ps]
    for p, d in zip(ps, grads):
        p.grad = d
    graph = new_graph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(new_graph()):
            a.step()
    a.step()
    for q in qs:
        q.grad = torch.zeros_like(q)
    b.step()
    with torch.cuda.graph(graph):
        a.step()
    for i in range(3):
        for d, q in zip(grads, qs):
            d.copy_(normal(gen(70 + i), *d.shape))
            q.grad = d.clone()
        graph.replay()
        b.step()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), i
    for p, q in zip(ps, qs):
        p.data = p.data.clone()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(new_graph()):
            a.step()
    a.step(), b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


def test_adamw_refuses_on_the_device():
    p = torch.nn.Parameter(torch.zeros(8, device=DEV))
    opt = optim.AdamW([p])
    p.grad = torch.zeros(8, device=DEV)
    opt.step()
    p.data = torch.zeros(9, device=DEV)
    with pytest.raises(RuntimeError, match="changed its size"):
        opt.step()
    for bad, error in ((torch.zeros(8, 8, device=DEV).t(), "contiguous"), (torch.zeros(8, device=DEV, dtype=F16), "float16")):
        q = torch.nn.Parameter(bad)
        q.grad = torch.zeros_like(q)
        with pytest.raises((ValueError, TypeError), match=error):
            optim.AdamW([q]).step()
    q = torch.nn.Parameter(torch.zeros(8, device=DEV))
    opt = optim.AdamW([{"params": [q]}])
    opt.param_groups[0]["params"].append(torch.nn.Parameter(torch.zeros(8, device=DEV)))
    q.grad = torch.zeros(8, device=DEV)
    opt.step()                                                             # (before the first step a group may still grow)
    opt.param_groups[0]["params"].append(torch.nn.Parameter(torch.zeros(8, device=DEV)))
    with pytest.raises(RuntimeError, match="add_param_group"):
        opt.step()


def test_adamw_more_tensors_than_one_launch_takes():
    ps = [torch.nn.Parameter(normal(gen(i), 5)) for i in range(900)]
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    a, b = optim.AdamW(ps, lr=1e-2), optim.AdamW([{"params": [q]} for q in qs], lr=1e-2)
    for p, q in zip(ps, qs):
        p.grad = q.grad = torch.ones_like(p)
    for p, q in list(zip(ps, qs))[440:880]:                                # a whole launch without gradients
        p.grad = q.grad = None
    a.step(), b.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))


# --------------------------------------------------------------------------- the operators together
def test_training_step_of_a_cross_attention_block():
    """Decoder tokens attend to an encoder's feature map: norm, projections, rotary positions on both grids, cross
    attention, output projection; gradients against the same chain in 64 bits, then one AdamW step.

    About a dozen tensors between the inputs and a gradient are rounded to bf16, each by at most u = 2^-8 of itself; the
    errors of the elements are independent, so the 2-norm of the result is off by less than 12 u of itself."""
    B, C, H, Hk, D = 2, 256, 4, 2, 64
    g = gen(80)
    sections, freqs = (8, 12, 12), attention.rotary_frequencies((8, 12, 12))
    grid = lambda s, n, step: torch.stack(torch.meshgrid(torch.arange(s) * 1.0, torch.arange(n) * step, torch.arange(n) * step, indexing="ij"), -1).reshape(-1, 3).to(DEV)
    pq, pk = grid(1, 16, 1.0), grid(1, 8, 2.0)                             # the encoder's map has half the resolution
    x, enc = normal(g, B, 256, C, to=BF16), normal(g, B, 64, C, to=BF16)
    lengths = torch.tensor([64, 40], dtype=torch.int32, device=DEV)
    wq, wk, wv, wo = (torch.nn.Parameter(normal(g, n, C, to=BF16, scale=C ** -0.5)) for n in (H * D, Hk * D, Hk * D, C))
    norm = attention.LayerNorm(C).to(DEV)
    norm.weight.data.add_(normal(g, C, scale=0.1))
    target = normal(g, B, 256, C)
    params = [wq, wk, wv, wo, norm.weight, norm.bias]

    def block(x, enc, wq, wk, wv, wo, w, b, exact):
        if exact:
            x, enc, wq, wk, wv, wo, w, b = (t.detach().double().requires_grad_() for t in (x, enc, wq, wk, wv, wo, w, b))
            n = ln_exact(x, w, b)[0]
        else:
            n = attention.layer_norm(x, w, b)
        q, k, v = (n @ wq.t()).view(B, 256, H, D), (enc @ wk.t()).view(B, 64, Hk, D), (enc @ wv.t()).view(B, 64, Hk, D)
        if exact:
            def turn(t, pos):
                axis = torch.tensor([a for a, m in enumerate(sections) for _ in range(m)], device=DEV)
                ang = (pos.double()[:, axis] * freqs)[None, :, None]
                one, two = t.chunk(2, -1)
                return torch.cat([one * ang.cos() - two * ang.sin(), two * ang.cos() + one * ang.sin()], -1)
            q, k = turn(q, pq), turn(k, pk)
            s = q.transpose(1, 2) @ k.transpose(1, 2).repeat_interleave(2, 1).transpose(-1, -2) * D ** -0.5
            s = s.masked_fill(~hidden(B, 64, lengths, None)[:, None, None], -torch.inf)
            o = (s.softmax(-1) @ v.transpose(1, 2).repeat_interleave(2, 1)).transpose(1, 2)
        else:
            q, k = attention.rotary(q, pq, freqs, sections), attention.rotary(k, pk, freqs, sections)
            o = attention.cross_attention(q, k, v, lengths)
        y = x + o.reshape(B, 256, H * D) @ wo.t()
        loss = ((y.double() if exact else y.float()) - target).square().mean()
        return y, torch.autograd.grad(loss, (x, enc, wq, wk, wv, wo, w, b) if exact else (x, enc, *params))
    x.requires_grad_(), enc.requires_grad_()
    y, grads = block(x, enc, *params, exact=False)
    ye, exact = block(x, enc, *params, exact=True)
    for name, a, b in zip(("y", "x", "enc", "wq", "wk", "wv", "wo", "w", "b"), (y, *grads), (ye, *exact)):
        off = ((a.double() - b).norm() / b.norm()).item()
        assert off <= 12 * U[BF16], (name, off)
    for p, d in zip(params, grads[2:]):
        p.grad = d
    old = [p.detach().clone() for p in params]
    opt = optim.AdamW(params, lr=1e-3, state_bits=8)
    opt.step()
    for p, t in zip(params, old):                                           # a first step moves by lr where there is a gradient
        want = t.double() * (1 - 1e-5) - 1e-3 * p.grad.double() / (p.grad.double().abs() + 1e-8)
        within(p.detach(), want, U[p.dtype] * want.abs() + 20 * E * 1e-3 + 3 * E * t.double().abs(), "p")
