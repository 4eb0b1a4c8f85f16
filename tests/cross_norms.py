"""Bounds for the 2-norms of cross attention's gradients.

An element-wise bound has to take the worst of every rounding at once, and over hundreds of rows or keys that is more than
the gradient itself: it finds outliers and nothing else.  The norm of the error is bounded here by how roundings add up
when they are independent, so that a term left out (Dl, a tile of keys or rows, some percent of a factor) shows.

u is half a step of the type relative to a value, so a rounding has a standard deviation of at most r = u / sqrt(3) of it.
Rounded to the type are: P and dS before the second products, o (which Dl is formed from, and which was formed from
rounded P), and the results.  In 32 bits (e = 2^-24) a sum of n terms in some order is off by a few sqrt(n) e: a score by
4 sqrt(D) e of the sum of |q||k| scale, and the row's sum of weights by (8 sqrt(n) + 64) e, exponentials and log-sum included
(together rel of P); dP by 8 sqrt(D) e, and the sums over n keys or rows by 4 sqrt(n) e, of the root of the sum of their
terms' squares.

Per row i: sigma_D^2 = r^2 sum_c (dO o)^2 + r^2 sum_j (P dP)^2 + (rel Dl)^2 (a weight's rounding moves all channels of o).
Per score: sigma_S^2 = (r^2 + rel^2 + 16 n e^2) dS^2 + P^2 sigma_dP^2; all scores of a row also share P sigma_D and rel dS.
   var dq = scale^2 (sum_j sigma_S^2 k^2 + (sigma_D sum_j P k)^2) + (rel^2 + r^2) dq^2
   var dk = scale^2  sum_i (sigma_S^2 + P^2 sigma_D^2 + rel^2 dS^2) q^2 + r^2 dk^2
   var dv =          sum_i (r^2 + rel^2 + 16 n e^2) P^2 dO^2 + r^2 dv^2
(r^2 of the results: plus the square of half a step of the type's smallest values.)  The squared norm of the error has the sum
of these as its expectation; with N independent rows or keys it is a mean of N numbers about one, so 1 + 4 / sqrt(N) times
the root is a bound that four standard deviations keep (five, for a single row)."""
import torch

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALL = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
BF16, F16 = torch.bfloat16, torch.float16

# (batch, queries, keys, heads, key heads, channels)
SHAPES = [(1, 1, 1, 1, 1, 8), (2, 1, 77, 8, 8, 64), (1, 33, 1, 2, 1, 32), (2, 3, 5, 4, 2, 40), (1, 64, 64, 2, 2, 64), (2, 65, 63, 3, 3, 96),
          (1, 100, 129, 6, 2, 128), (3, 127, 200, 2, 1, 80), (1, 300, 257, 4, 4, 24), (2, 129, 640, 8, 1, 128), (1, 5, 1000, 16, 4, 56),
          (1, 700, 40, 2, 2, 72), (1, 1, 3001, 8, 2, 128), (4, 2, 2500, 4, 4, 64), (1, 1025, 513, 1, 1, 120), (1, 31, 700, 1, 1, 104)]
SHARED = [(3, 700, 300, 4, 2), (5, 260, 1500, 2, 1), (1, 3000, 70, 4, 4), (2, 1100, 130, 12, 3), (300, 40, 65, 2, 2)]
CASES = [(shape, kind) for shape in SHAPES for kind in (BF16, F16)] + [((*sizes, dim), BF16) for sizes in SHARED for dim in (64, 128)]


def inputs(seed, shape, kind, device="cpu"):
    """q, k, v, dO; v and dO share a direction, so that dP is far from zero and Dl matters in every score."""
    B, Lq, Lk, H, G, D = shape
    gen = torch.Generator().manual_seed(seed)
    make = lambda n, heads, shift: (torch.randn(B, n, heads, D, generator=gen) + shift).to(kind).to(device)
    return make(Lq, H, 0.0), make(Lk, G, 0.0), make(Lk, G, 1.0), make(Lq, H, 1.0)


def some_keys(seed, shape, device="cpu"):
    """lengths and a mask that leave an entry empty, one with a single key, and one whole"""
    B, Lk = shape[0], shape[2]
    gen = torch.Generator().manual_seed(seed)
    lengths = torch.randint(0, Lk + 1, (B,), generator=gen, dtype=torch.int32)
    lengths[0] = Lk
    if B > 2:
        lengths[1], lengths[2] = 0, 1
    return lengths.to(device), (torch.rand(B, Lk, generator=gen) < 0.7).to(device)


def visible(k, lengths=None, mask=None):
    ok = torch.ones(k.shape[:2], dtype=torch.bool, device=k.device)
    if lengths is not None:
        ok &= torch.arange(k.shape[1], device=k.device)[None] < lengths[:, None]
    return ok if mask is None else ok & mask.bool()


def parts(q, k, v, dout, lengths=None, mask=None):
    """q, k, v, dO [batch][heads][...][channels] in 64 bits (hidden keys zero), P, o, dP and Dl."""
    group = q.shape[2] // k.shape[2]
    ok = visible(k, lengths, mask)
    q, k, v, do = (t.detach().double().transpose(1, 2) for t in (q, k, v, dout))
    k, v = (torch.where(ok[:, None, :, None], t, 0.0).repeat_interleave(group, 1) for t in (k, v))
    s = (q @ k.transpose(-1, -2).contiguous() * q.shape[-1] ** -0.5).masked_fill(~ok[:, None, None], -torch.inf)
    lse = s.logsumexp(-1, keepdim=True)
    p = torch.where(torch.isinf(lse), 0.0, (s - lse).exp())
    o = p @ v
    return q, k, v, do, p, o, do @ v.transpose(-1, -2).contiguous(), (do * o).sum(-1, keepdim=True), group


def gradients(q, k, do, p, ds, group, p_dv=None):
    scale = q.shape[-1] ** -0.5
    fold = lambda t: t.unflatten(1, (-1, group)).sum(2)
    back = lambda t: t.transpose(-1, -2).contiguous()
    return {"dq": ds @ k * scale, "dk": fold(back(ds) @ q) * scale, "dv": fold(back(p if p_dv is None else p_dv) @ do)}


def exact_and_variance(q, k, v, dout, lengths=None, mask=None):
    """{name: (gradient, variance of its error)}, [batch][heads][tokens][channels] in 64 bits."""
    kind, D, n = q.dtype, q.shape[3], k.shape[1]
    r2, small2 = U[kind] ** 2 / 3, SMALL[kind] ** 2
    scale2 = 1.0 / D
    q, k, v, do, p, o, dp, dl, group = parts(q, k, v, dout, lengths, mask)
    rows = group * q.shape[2]
    ds = p * (dp - dl)
    back = lambda t: t.transpose(-1, -2).contiguous()
    fold = lambda t: t.unflatten(1, (-1, group)).sum(2)
    terms = (q.abs() @ back(k.abs())).amax(-1, keepdim=True) * D ** -0.5 if n else torch.zeros_like(dl)
    rel2 = ((4 * D ** 0.5 * terms + 8 * n ** 0.5 + 64) * E) ** 2
    var_d = r2 * ((do * o) ** 2).sum(-1, keepdim=True) + r2 * ((p * dp) ** 2).sum(-1, keepdim=True) + rel2 * dl ** 2
    var_dp = 64 * D * E ** 2 * (do ** 2 @ back(v ** 2))
    per_key = (r2 + rel2 + 16 * n * E ** 2) * ds ** 2 + p ** 2 * var_dp
    per_row = (r2 + rel2 + 16 * rows * E ** 2) * ds ** 2 + p ** 2 * (var_dp + var_d) + rel2 * ds ** 2
    want = gradients(q, k, do, p, ds, group)
    var = {"dq": scale2 * (per_key @ k ** 2 + var_d * (p @ k) ** 2) + (rel2 + r2) * want["dq"] ** 2 + small2,
           "dk": scale2 * fold(back(per_row) @ q ** 2) + r2 * want["dk"] ** 2 + small2,
           "dv": fold(back((r2 + rel2 + 16 * rows * E ** 2) * p ** 2) @ do ** 2) + r2 * want["dv"] ** 2 + small2}
    return {name: (want[name], var[name]) for name in want}


def ratio(got, want, var, rows):
    """Largest of |error| / bound over the heads of the entries and over the whole tensor; rows: of a head, for N."""
    worst = 0.0
    for over, many in (((2, 3), 1), ((0, 1, 2, 3), want.shape[0] * want.shape[1])):
        bound = var.sum(over).sqrt() * (1 + 4 / max(1, min(rows, want.shape[2]) * many) ** 0.5)
        off = ((got - want) ** 2).sum(over).sqrt()
        part = torch.where(off <= bound, off / bound.clamp(min=1e-300), off / bound)        # (0 / 0: nothing is off)
        worst = max(worst, float("inf") if bool(part.isnan().any()) else part.max().item() if part.numel() else 0.0)
    return worst


def ratios(got, bounds, rows):
    return {name: ratio(got[name].double(), *bounds[name], rows) for name in got}


def rounded(q, k, v, dout, lengths=None, mask=None):
    """The gradients with every rounding to the type where the bounds count one, the rest in 64 bits."""
    kind = q.dtype
    q, k, v, do, p, _, dp, _, group = parts(q, k, v, dout, lengths, mask)
    cut = lambda t: t.float().to(kind).double()
    o = cut(cut(p * (128.0 if kind == F16 else 1.0)) @ v / (128.0 if kind == F16 else 1.0))
    ds = p * (dp - (do * o).sum(-1, keepdim=True))
    up = 2.0 ** (14 - ds.abs().max().clamp(min=1e-30).log2().ceil()) if kind == F16 else 1.0     # (dS travels times a power of two,
    ds, p_up = cut(ds * up) / up, 2.0 ** 15 if kind == F16 else 1.0                              # and P too)
    return {name: cut(t) for name, t in gradients(q, k, do, p, ds, group, cut(p * p_up) / p_up).items()}


def mutants(q, k, v, dout, lengths=None, mask=None):
    """name: gradients with a mistake in them"""
    q, k, v, do, p, _, dp, dl, group = parts(q, k, v, dout, lengths, mask)
    right = gradients(q, k, do, p, p * (dp - dl), group)
    keys, rows = torch.ones(p.shape[-1], dtype=p.dtype, device=p.device), torch.ones(p.shape[-2], 1, dtype=p.dtype, device=p.device)
    keys[:64], rows[:32] = 0, 0
    first = torch.zeros(p.shape[1], 1, 1, dtype=p.dtype, device=p.device)
    first[::group] = 1                                                      # (rows are missing from one head of a group)
    gone = 1 - first * (1 - rows)
    some = {"no Dl": gradients(q, k, do, p, p * dp, group), "Dl * 0.9": gradients(q, k, do, p, p * (dp - 0.9 * dl), group),
            "factor 1.02": {name: 1.02 * t for name, t in right.items()},
            "64 keys left out": {"dq": gradients(q, k, do, p, p * (dp - dl) * keys, group)["dq"]},
            "32 rows left out": {name: t for name, t in gradients(q, k, do, p * gone, p * (dp - dl) * gone, group).items() if name != "dq"}}
    for name in ("no Dl", "Dl * 0.9"):
        del some[name]["dv"]
    return right, some
