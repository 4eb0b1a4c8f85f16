"""What the token operators refuse before any launch, because a result would lack something in silence; no GPU needed."""
import struct

import pytest
import torch
from torch.autograd import forward_ad

from reid_gan_amd import _lib, attention, optim

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
