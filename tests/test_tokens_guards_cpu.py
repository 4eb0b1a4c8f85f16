"""What the token operators refuse before any launch, because a result would lack something in silence; no GPU needed."""
import struct

import pytest
import torch
from torch.autograd import forward_ad

from reid_gan_amd import _lib, attention, ops, optim

BF16 = torch.bfloat16


def calls():
    """name: function of its tensors, the tensors"""
    x, w, b = torch.ones(5, 64), torch.ones(64), torch.zeros(64)
    r, pos, freqs = torch.ones(1, 3, 2, 64), torch.ones(1, 3, 3), attention.rotary_frequencies((8, 12, 12), device="cpu")
    q, k, v = (torch.ones(1, n, 2, 64, dtype=BF16) for n in (3, 9, 9))
    return {"layer_norm": (attention.layer_norm, (x, w, b)),
            "rotary": (lambda t, p, f: attention.rotary(t, p, f, (8, 12, 12)), (r, pos, freqs)),
            "cross_attention": (attention.cross_attention, (q, k, v))}


@pytest.mark.parametrize("name", ["layer_norm", "rotary", "cross_attention"])
def test_forward_mode_derivatives_are_refused(name):
    call, args = calls()[name]
    with forward_ad.dual_level():
        for i in range(3):
            dual = [forward_ad.make_dual(t, torch.ones_like(t)) if j == i else t for j, t in enumerate(args)]
            with pytest.raises(RuntimeError, match="forward-mode"):
                call(*dual)
        with pytest.raises(RuntimeError, match="no CPU path"):              # (no tangent: nothing to refuse but the device)
            call(*args)


@pytest.mark.parametrize("name", ["layer_norm", "rotary", "cross_attention"])
def test_traces_are_refused(name):
    from torch.fx.experimental.proxy_tensor import make_fx
    call, args = calls()[name]
    with pytest.raises(RuntimeError, match="traced"):
        torch.jit.trace(call, args, check_trace=False)
    with pytest.raises(RuntimeError, match="traced"):
        make_fx(lambda *ts: call(*ts))(*args)
    with pytest.raises(RuntimeError, match="no CPU path"):                  # (outside a trace: nothing to refuse but the device)
        call(*args)


def test_rotary_refuses_gradients_of_its_tables():
    call, (x, pos, freqs) = calls()["rotary"]
    for leaf in (pos, freqs):
        leaf.requires_grad_()
        with pytest.raises(RuntimeError, match="positions and freqs have no gradient"):
            call(x, pos, freqs)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):
            call(x, pos, freqs)
        leaf.requires_grad_(False)


@pytest.mark.parametrize("scale", [1e-46, 1e-38, 1e30])
def test_cross_attention_refuses_scales_that_32_bits_lose(scale):
    """A factor of zero would turn the -infinity of hidden keys into NaN, and with it whole rows."""
    call, args = calls()["cross_attention"]
    with pytest.raises(ValueError, match="scale"):
        call(*args, scale=scale)
    at, strides = 1 << 20, (64, 64, 64)                                     # (an address that nothing dereferences)
    desc = struct.pack("=12q24q8qd", *(at,) * 5, 0, 0, *(at,) * 5, *strides * 8, 0, 1, 1, 1, 1, 1, 64, 1, scale)
    for entry in (_lib.lib.ried_xattn_fwd, _lib.lib.ried_xattn_bwd):
        with pytest.raises(RuntimeError, match="scale"):
            entry(desc, None)


def test_cross_attention_takes_small_scales():
    call, args = calls()["cross_attention"]
    with pytest.raises(RuntimeError, match="no CPU path"):
        call(*args, scale=1e-36)


@pytest.mark.parametrize("entry", ["maximize", "amsgrad"])
def test_adamw_refuses_states_of_another_update(entry):
    """A torch state whose groups ask for an update that is not this one's."""
    p = torch.nn.Parameter(torch.zeros(4))
    saved = torch.optim.AdamW([p], **{entry: True}).state_dict()
    with pytest.raises(ValueError, match="no maximize and no amsgrad"):
        optim.AdamW([p]).load_state_dict(saved)


def buffer_calls(device):
    """name: (function of its tensors, the tensors by name) of the functions on buffers"""
    z = lambda *shape, to=BF16: torch.zeros(*shape, dtype=to, device=device)
    F32 = torch.float32
    rows = dict(x=z(4, 64), w=z(64, to=F32), b=z(64, to=F32), y=z(4, 64), stats=z(2, 4, to=F32))
    back = dict(dy=z(4, 64), x=z(4, 64), w=z(64, to=F32), stats=z(2, 4, to=F32), dx=z(4, 64), dw=z(64, to=F32), db=z(64, to=F32),
                scratch=z(4096, to=F32))
    turn = dict(x=z(1, 3, 2, 8), y=z(1, 3, 2, 8), pos=z(1, 3, 1, to=F32), freqs=z(4, to=torch.float64))
    some = dict(q=z(1, 2, 2, 64), k=z(1, 4, 2, 64), v=z(1, 4, 2, 64), out=z(1, 2, 2, 64), lse=z(1, 2, 2, to=F32),
                lengths=z(1, to=torch.int32), mask=z(1, 4, to=torch.bool), scratch=z(4096, to=F32))
    grads = dict(some, dout=z(1, 2, 2, 64), dq=z(1, 2, 2, 64), dk=z(1, 4, 2, 64), dv=z(1, 4, 2, 64))
    return {"layer_norm_fwd": (lambda x, w, b, y, stats: ops.layer_norm_fwd(x, w, b, y, stats, 1e-5), rows),
            "layer_norm_bwd": (lambda **t: ops.layer_norm_bwd(**t), back),
            "rotary": (lambda x, y, pos, freqs: ops.rotary(x, y, pos, freqs, (4,), False, False), turn),
            "xattn_fwd": (lambda q, k, v, out, lse, lengths, mask, scratch: ops.xattn_fwd(q, k, v, out, lse, 0.125, lengths, mask, scratch), some),
            "xattn_bwd": (lambda q, k, v, out, lse, lengths, mask, scratch, dout, dq, dk, dv:
                          ops.xattn_bwd(dout, q, k, v, out, lse, dq, dk, dv, 0.125, scratch, lengths, mask), grads)}


@pytest.mark.parametrize("name", list(buffer_calls("cpu")))
def test_functions_on_buffers_refuse_host_memory(name):
    call, tensors = buffer_calls("cpu")[name]
    with pytest.raises(AssertionError, match="ROCm device"):
        call(**tensors)


def test_layer_norm_on_buffers_refuses_parameters_of_two_types():
    call, tensors = buffer_calls("cpu")["layer_norm_fwd"]
    for name in ("w", "b"):
        with pytest.raises(AssertionError) as error:
            call(**{**tensors, name: tensors[name].to(BF16)})
        assert "ROCm" not in str(error.value)


def test_cross_attention_refuses_gradients_of_too_many_queries_before_it_works_on_them():
    meta = lambda n: torch.zeros(1, n, 16, 128, dtype=BF16, device="meta")
    for q, error in ((meta(1 << 19), "fewer queries"), (meta((1 << 19) - 1), "no CPU path")):
        with pytest.raises((ValueError, RuntimeError), match=error):
            attention.cross_attention(q.requires_grad_(), meta(77), meta(77))
