"""Token operators of a cross-attention block, beside the convolutional path: layer norm, rotary positions of several
axes, and cross attention to an encoder's states, forward and backward on hand-written kernels.

A call whose arguments need nothing but the launch goes straight to it (csrc/bind.cpp); the Python code here does the rest:
the checks with their messages, and the copies of what is not laid out for the kernels.

They have no counterpart in the reference, whose only attention is the Self_Attn layer (src/rinet.py:150-181).
Tensors live on a ROCm device (there is no CPU path) in fp32, bf16 or fp16 (cross attention: bf16 or fp16); sums,
statistics and softmax are fp32 whatever the type.  Every call runs on the current stream of its tensors' device and
allocates what it needs from torch's allocator, so calls on different streams share nothing.

The functions here are differentiable backwards, once; tensors with a forward-mode tangent are refused, and so is a call
under torch.jit.trace or make_fx.  Gradients are not made for graph capture: torch's AccumulateGrad nodes remember the
stream of an earlier eager pass, and a captured backward that meets one ends the process.  A captured step calls the
forward and backward functions of reid_gan_amd.ops on buffers of its own (as TrainStep does); without gradients the
functions here may be captured as they are.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch
from torch.autograd.function import once_differentiable

from . import ops
from ._lib import direct

__all__ = ["layer_norm", "LayerNorm", "rotary", "rotary_frequencies", "cross_attention"]

F32 = torch.float32
_CONTIGUOUS = torch.contiguous_format
_CROSS_TYPES = (torch.bfloat16, torch.float16)


def _check_tensor(what: str, name: str, t, types, device=None):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what}: {name} is a tensor, not {type(t).__name__}")
    if t.dtype not in types:
        raise TypeError(f"{what}: {name} is {t.dtype}, not one of {', '.join(str(d).replace('torch.', '') for d in types)}")
    if device is not None and t.device != device:
        raise ValueError(f"{what}: {name} is on {t.device}, not on {device}")
    if t.layout is not torch.strided or t.is_neg():
        raise ValueError(f"{what}: {name} is sparse or a lazily negated view; pass a dense tensor (resolve_neg())")


def _on_gpu(what: str, t: torch.Tensor):
    if not t.is_cuda:
        raise RuntimeError(f"{what}: tensors must be on a ROCm device; there is no CPU path")


def _check_recording(what: str, *tensors):
    if direct().traced():
        raise RuntimeError(f"{what}: cannot be traced (the trace would hold the allocation of the result without the kernel that "
                           "writes it)")
    if direct().dual(*tensors):
        raise RuntimeError(f"{what}: there is no forward-mode derivative, and a tensor has a tangent (take it off with unpack_dual)")


def _not_captured(what: str):
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: gradients are not taken under graph capture; capture the forward and backward "
                           "functions of reid_gan_amd.ops instead")


def _once(backward):
    """A backward function without a second derivative: asking for one raises.  (once_differentiable says so too, at the
    price of a small kernel's launch in every first derivative.)"""
    guarded = once_differentiable(backward)

    def run(ctx, grad):
        _check_recording("backward", grad)
        return guarded(ctx, grad) if torch.is_grad_enabled() else backward(ctx, grad)
    return run


# --------------------------------------------------------------------------- layer norm
def _rows(t: torch.Tensor) -> torch.Tensor:
    """t, or a view (a copy where there is none) as [rows][C], with adjacent channels and rows that do not overlap."""
    if t.is_contiguous():
        return t
    C = t.shape[-1]
    t = t.reshape(-1, C)
    if (C > 1 and t.stride(1) != 1) or t.stride(0) < C:
        t = t.contiguous()
    return t


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        _not_captured("layer_norm")
        rows = _rows(x)
        y = torch.empty_like(x, memory_format=_CONTIGUOUS)
        stats = x.new_empty((2, x.numel() // x.shape[-1]), dtype=F32)
        ops.layer_norm_fwd(rows, weight, bias, y, stats, eps)
        ctx.save_for_backward(rows, weight, stats)
        ctx.meta = x.shape, None if bias is None else bias.dtype
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        _not_captured("layer_norm")
        rows, weight, stats = ctx.saved_tensors
        shape, bias_type = ctx.meta
        need_x, need_w, need_b, _ = ctx.needs_input_grad
        C = shape[-1]
        dx = torch.empty_like(rows, memory_format=_CONTIGUOUS)
        dw = torch.empty_like(weight) if need_w else None
        db = rows.new_empty((C,), dtype=bias_type) if need_b else None
        scratch = None
        if need_w or need_b:
            scratch = stats.new_empty((ops.layer_norm_bwd_scratch_floats(stats.shape[1], C, rows.dtype),))
        ops.layer_norm_bwd(_rows(dy), rows, weight, stats, dx, dw, db, scratch)
        return dx.view(shape) if need_x else None, dw, db, None


def _check_layer_norm(x, weight, bias, eps):
    _check_tensor("layer_norm", "x", x, ops.TOKEN_TYPES)
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError("layer_norm: x has no last axis to normalise")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        _check_tensor("layer_norm", name, t, (F32,) if x.dtype is F32 else (F32, x.dtype), x.device)
        if t.shape != x.shape[-1:] or not t.is_contiguous():
            raise ValueError(f"layer_norm: {name} must be a contiguous [{x.shape[-1]}] tensor, not {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype is not bias.dtype:
        raise TypeError("layer_norm: weight and bias have different types")
    if not eps >= 0:
        raise ValueError("layer_norm: eps is negative")
    _on_gpu("layer_norm", x)


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last axis: (x - mean) / sqrt(var + eps) * weight + bias.

    x: any shape; rows are read where they lie when their channels are adjacent.  weight, bias: [C], contiguous, both fp32
    or both of x's type, each optional.  The result is contiguous and of x's type; weight and bias gradients are summed
    in fp32 in a fixed order."""
    y = direct().layer_norm(x, weight, bias, eps)
    if y is not None:
        return y
    _check_recording("layer_norm", x, weight, bias)
    _check_layer_norm(x, weight, bias, eps)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNormFn.apply(x, weight, bias, eps)
    y = torch.empty_like(x, memory_format=_CONTIGUOUS)
    ops.layer_norm_fwd(_rows(x), weight, bias, y, None, eps)
    return y


class LayerNorm(torch.nn.Module):
    """layer_norm with its parameters (names and initialisation of torch.nn.LayerNorm over one axis)."""

    def __init__(self, channels: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True):
        super().__init__()
        self.channels, self.eps = int(channels), eps
        self.weight = torch.nn.Parameter(torch.ones(self.channels)) if elementwise_affine else None
        self.bias = torch.nn.Parameter(torch.zeros(self.channels)) if elementwise_affine and bias else None

    def forward(self, x):
        if x.shape[-1] != self.channels:
            raise ValueError(f"LayerNorm: {x.shape[-1]} channels, built for {self.channels}")
        return layer_norm(x, self.weight, self.bias, self.eps)


# --------------------------------------------------------------------------- rotary positions
def rotary_frequencies(sections: Sequence[int], base: float = 10000.0, shared: bool = False, device="cuda") -> torch.Tensor:
    """fp64 table of radians per unit of position, one entry per pair of channels.  Every axis has a ladder of its own,
    base ** (-j / pairs of the axis); shared: one ladder runs through the sections, base ** (-j / all pairs)."""
    sections = [int(n) for n in sections]
    if not 1 <= len(sections) <= 4 or min(sections) < 0 or sum(sections) == 0:
        raise ValueError("rotary_frequencies: sections are the numbers of pairs of one to four axes")
    ladders = [sum(sections)] if shared else sections
    return torch.cat([float(base) ** (-torch.arange(n, dtype=torch.float64) / max(n, 1)) for n in ladders]).to(device)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    def span(t):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


class _RotaryFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, positions, freqs, sections, interleaved, inverse):
        _not_captured("rotary")
        ctx.save_for_backward(positions, freqs)
        ctx.meta = (sections, interleaved, inverse)
        y = torch.empty_like(x, memory_format=_CONTIGUOUS)
        ops.rotary(x, y, positions, freqs, sections, interleaved, inverse)
        return y

    @staticmethod
    @_once
    def backward(ctx, dy):
        _not_captured("rotary")
        positions, freqs = ctx.saved_tensors
        sections, interleaved, inverse = ctx.meta
        if dy.stride(-1) != 1:
            dy = dy.contiguous()
        dx = torch.empty_like(dy, memory_format=_CONTIGUOUS)
        ops.rotary(dy, dx, positions, freqs, sections, interleaved, not inverse)
        return dx, None, None, None, None, None


def rotary(x: torch.Tensor, positions: torch.Tensor, freqs: torch.Tensor, sections: Sequence[int], interleaved: bool = False,
           inverse: bool = False, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Turns the channel pairs of x [batch][tokens][heads][channels] by the tokens' positions.

    positions: [batch][tokens][axes] or [tokens][axes], int32, int64 or fp32 (an encoder's coarser grid has positions
    between the decoder's).  sections: pairs of each axis (slice, row, column ...), one to four; freqs: fp64 table of
    rotary_frequencies, sum(sections) entries.  Pair j is channels (j, j + pairs), or (2j, 2j + 1) when interleaved;
    channels behind the pairs pass through.  Angles are formed in 64 bits, so far positions keep their precision.
    inverse turns back (and is the gradient, which x alone has: positions and freqs that require one are refused).  out: where
    to write, also x itself (no gradients then)."""
    if out is None:
        y = direct().rotary(x, positions, freqs, sections, interleaved, inverse)
        if y is not None:
            return y
    _check_recording("rotary", x, positions, freqs, out)
    _check_tensor("rotary", "x", x, ops.TOKEN_TYPES)
    if x.dim() != 4:
        raise ValueError("rotary: x is [batch][tokens][heads][channels]")
    B, L, _, D = x.shape
    axes, pairs = len(sections), sum(sections)
    if not 1 <= axes <= 4 or min(sections) < 0 or not 0 < 2 * pairs <= D:
        raise ValueError(f"rotary: sections {tuple(sections)} do not fit {D} channels (one to four axes, two channels a pair)")
    _check_tensor("rotary", "positions", positions, ops.POSITION_TYPES, x.device)
    if positions.dim() == 2:
        positions = positions.unsqueeze(0).expand(B, -1, -1)
    if positions.shape != (B, L, axes):
        raise ValueError(f"rotary: positions are [batch][tokens][{axes}] for x {tuple(x.shape)}, not {tuple(positions.shape)}")
    _check_tensor("rotary", "freqs", freqs, (torch.float64,), x.device)
    if freqs.shape != (pairs,) or not freqs.is_contiguous():
        raise ValueError(f"rotary: freqs is a contiguous table of {pairs} entries")
    if torch.is_grad_enabled() and (positions.requires_grad or freqs.requires_grad):
        raise RuntimeError("rotary: positions and freqs have no gradient; pass them detached")
    adjacent = D == 1 or x.stride(3) == 1
    if out is None:
        _on_gpu("rotary", x)
        if not adjacent:
            x = x.contiguous()
        if x.requires_grad and torch.is_grad_enabled():
            return _RotaryFn.apply(x, positions, freqs, tuple(sections), interleaved, inverse)
        out = torch.empty_like(x, memory_format=_CONTIGUOUS)
    else:
        if torch.is_grad_enabled() and (x.requires_grad or out.requires_grad):
            raise RuntimeError("rotary: out= has no gradient; leave it out, or use torch.no_grad()")
        if out is x and not adjacent:
            raise ValueError("rotary: in place needs adjacent channels")
        _check_tensor("rotary", "out", out, (x.dtype,), x.device)
        if out.shape != x.shape or (out.stride(3) != 1 and D > 1):
            raise ValueError("rotary: out has x's shape and adjacent channels")
        if any(s == 0 and n > 1 for n, s in zip(out.shape, out.stride())):
            raise ValueError("rotary: out is an expanded tensor")
        same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
        if x.numel() and ((not same and _overlap(out, x)) or _overlap(out, positions) or _overlap(out, freqs)):
            raise ValueError("rotary: out overlaps x, positions or freqs without being x")
        _on_gpu("rotary", x)
        if not adjacent:
            x = x.contiguous()
        torch.autograd.graph.increment_version(out)              # (a graph that saved what is written here must not use it)
    ops.rotary(x, out, positions, freqs, sections, interleaved, inverse)
    return out


# --------------------------------------------------------------------------- cross attention
def _laid_out(t: torch.Tensor) -> torch.Tensor:
    """t [batch][tokens][heads][channels] as the kernels read it: adjacent channels, strides in multiples of 8 elements,
    16-byte alignment (a copy only where it is not)."""
    a, b, c, d = t.stride()
    if d == 1 and not ((a | b | c) & 7 or t.data_ptr() & 15) and a >= 0 and 0 <= b <= 1 << 23 and c >= 0:
        return t
    return t.clone(memory_format=_CONTIGUOUS)


def _near(t: torch.Tensor, share: int) -> torch.Tensor:
    """t laid out, and the heads that share a key head (`share` of them) within 2^31 bytes, as the gradients' kernels read q and
    dout."""
    t = _laid_out(t)
    far = (t.shape[1] * t.stride(1) + share * t.stride(2)) * 2 >= 1 << 31
    return t.clone(memory_format=_CONTIGUOUS) if far else t


def _attend(q, k, v, lengths, key_mask, scale, lse):
    (B, Lq, H, D), (_, Lk, G, _) = q.shape, k.shape
    out = torch.empty_like(q, memory_format=_CONTIGUOUS)
    n = ops.xattn_fwd_scratch_floats(B, Lq, Lk, H, G, D)
    ops.xattn_fwd(q, k, v, out, lse, scale, lengths, key_mask, q.new_empty((n,), dtype=F32) if n else None)
    return out


class _CrossFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, key_mask, scale):
        _not_captured("cross_attention")
        q, k, v = _near(q, q.shape[2] // k.shape[2]), _laid_out(k), _laid_out(v)
        B, Lq, H, _ = q.shape
        lse = q.new_empty((B, H, Lq), dtype=F32)
        out = _attend(q, k, v, lengths, key_mask, scale, lse)
        ctx.save_for_backward(q, k, v, out, lse, lengths, key_mask)
        ctx.scale = scale
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        _not_captured("cross_attention")
        q, k, v, out, lse, lengths, key_mask = ctx.saved_tensors
        dq, dk, dv = (torch.empty_like(t, memory_format=_CONTIGUOUS) for t in (q, k, v))
        (B, Lq, H, D), (_, Lk, G, _) = q.shape, k.shape
        if Lq == 0:
            return dq, dk.zero_(), dv.zero_(), None, None, None
        scratch = lse.new_empty((ops.xattn_bwd_scratch_floats(B, Lq, Lk, H, G, D),))
        ops.xattn_bwd(_near(dout, H // G), q, k, v, out, lse, dq, dk, dv, ctx.scale, scratch, lengths, key_mask)
        return dq, dk, dv, None, None, None


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, lengths: Optional[torch.Tensor] = None,
                    key_mask: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """softmax(scale q k^T) v of queries [batch][queries][heads][channels] over an encoder's states k, v
    [batch][keys][key heads][channels], of any other length.

    Head h reads key head h // (heads // key heads).  lengths: int32 [batch], the first so many keys of each entry
    count; key_mask: bool or uint8 [batch][keys], nonzero keys count; with both, keys that both allow.  An entry without
    keys gives zeros and no gradient; hidden keys have no effect whatever they hold, and get zero gradients.  scale:
    channels ** -0.5 unless given (between 1e-37 and 1e30).  channels: a multiple of 8 up to 128, bf16 or fp16.  Views are
    read where they lie when their channels are adjacent and their strides are multiples of 8 elements; others are copied.
    With gradients, the queries of an entry are under 2^31 bytes."""
    o = direct().cross_attention(q, k, v, lengths, key_mask, scale)
    if o is not None:
        return o
    _check_recording("cross_attention", q, k, v)
    _check_tensor("cross_attention", "q", q, _CROSS_TYPES)
    device, kind = q.device, (q.dtype,)
    _check_tensor("cross_attention", "k", k, kind, device)
    _check_tensor("cross_attention", "v", v, kind, device)
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4 or ks != v.shape or qs[0] != ks[0] or qs[3] != ks[3]:
        raise ValueError(f"cross_attention: q [batch][queries][heads][channels] and k, v [batch][keys][key heads][channels] do "
                         f"not fit: {tuple(qs)}, {tuple(ks)}, {tuple(v.shape)}")
    B, _, H, D = qs
    if H == 0 or ks[2] == 0 or H % ks[2]:
        raise ValueError(f"cross_attention: {H} heads do not divide over {ks[2]} key heads")
    if D % 8 or not 8 <= D <= 128:
        raise ValueError(f"cross_attention: {D} channels are not a multiple of 8 up to 128")
    if lengths is not None:
        _check_tensor("cross_attention", "lengths", lengths, (torch.int32,), device)
        if lengths.shape != (B,) or not lengths.is_contiguous():
            raise ValueError(f"cross_attention: lengths is a contiguous [{B}] tensor")
    if key_mask is not None:
        _check_tensor("cross_attention", "key_mask", key_mask, (torch.bool, torch.uint8), device)
        if key_mask.shape != (B, k.shape[1]):
            raise ValueError(f"cross_attention: key_mask is [{B}][{k.shape[1]}], not {tuple(key_mask.shape)}")
        if key_mask.stride(0) < 0 or (key_mask.stride(1) != 1 and key_mask.shape[1] > 1):
            key_mask = key_mask.contiguous()
    scale = D ** -0.5 if scale is None else float(scale)
    if not 1e-37 < scale < 1e30:
        raise ValueError("cross_attention: scale is a positive number between 1e-37 and 1e30")
    wanted = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if wanted and (qs[1] * H * D + H // ks[2] * D) * 2 >= 1 << 31:
        raise ValueError(f"cross_attention: gradients of {qs[1]} queries of {H} x {D} channels (2^31 bytes or more an entry) are not "
                         "taken; pass fewer queries")
    _on_gpu("cross_attention", q)
    if wanted:
        return _CrossFn.apply(q, k, v, lengths, key_mask, scale)
    return _attend(_laid_out(q), _laid_out(k), _laid_out(v), lengths, key_mask, scale, None)
