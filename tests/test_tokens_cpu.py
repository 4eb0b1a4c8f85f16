"""What the token operators (layer norm, rotary positions, cross attention, AdamW) refuse, and what their host sides
compute; no GPU needed: the refusals come before any launch."""
import ctypes
import math
import struct

import pytest
import torch

from reid_gan_amd import _lib, attention, ops, optim

lib = _lib.lib
P = 1 << 20            # an aligned address that nothing here dereferences


def _z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("call, error", [
    (lambda: attention.layer_norm(_z(4, 8)), "no CPU path"),
    (lambda: attention.layer_norm(_z(4, 8, dtype=torch.float64)), "float64"),
    (lambda: attention.layer_norm(torch.tensor(1.0)), "no last axis"),
    (lambda: attention.layer_norm(_z(4, 0)), "no last axis"),
    (lambda: attention.layer_norm(_z(4, 8), _z(4)), "contiguous"),
    (lambda: attention.layer_norm(_z(4, 8), _z(16)[::2]), "contiguous"),
    (lambda: attention.layer_norm(_z(4, 8), _z(8, dtype=torch.float16)), "float16"),
    (lambda: attention.layer_norm(_z(4, 8), _z(8), _z(8, dtype=torch.float32)), "different types"),
    (lambda: attention.layer_norm(_z(4, 8), eps=-1.0), "negative"),
    (lambda: attention.layer_norm([1.0]), "tensor"),
    (lambda: attention.LayerNorm(8)(_z(4, 16)), "16 channels"),
])
def test_layer_norm_refuses(call, error):
    with pytest.raises((ValueError, TypeError, RuntimeError), match=error):
        call()


def _rot(x=None, pos=None, freqs=None, sections=(1, 2, 1), **kw):
    x = _z(2, 3, 4, 8) if x is None else x
    pos = torch.zeros(2, 3, 3, dtype=torch.int32) if pos is None else pos
    freqs = attention.rotary_frequencies(sections, device="cpu") if freqs is None else freqs
    return attention.rotary(x, pos, freqs, sections, **kw)


@pytest.mark.parametrize("call, error", [
    (lambda: _rot(), "no CPU path"),
    (lambda: _rot(x=_z(3, 4, 8)), "batch"),
    (lambda: _rot(sections=(2, 2, 2)), "do not fit"),
    (lambda: _rot(sections=(1, 1, 1, 1, 0), freqs=torch.zeros(4, dtype=torch.float64)), "do not fit"),
    (lambda: _rot(pos=torch.zeros(2, 3, 2, dtype=torch.int32)), "positions"),
    (lambda: _rot(pos=torch.zeros(2, 3, 3, dtype=torch.int16)), "int16"),
    (lambda: _rot(freqs=torch.zeros(4)), "float32"),
    (lambda: _rot(freqs=torch.zeros(5, dtype=torch.float64)), "table of 4"),
    (lambda: _rot(out=_z(2, 3, 4, 16)), "shape"),
    (lambda: _rot(out=_z(2, 3, 1, 8).expand(2, 3, 4, 8)), "expanded"),
    (lambda: _rot(x=_z(2, 3, 4, 8).requires_grad_(), out=_z(2, 3, 4, 8)), "no gradient"),
    (lambda: attention.rotary_frequencies((0, 0)), "sections"),
])
def test_rotary_refuses(call, error):
    with pytest.raises((ValueError, TypeError, RuntimeError), match=error):
        call()


def test_rotary_refuses_an_overlapping_result():
    buf = _z(2 * 3 * 4 * 8 + 8)
    x, y = buf[:192].view(2, 3, 4, 8), buf[8:].view(2, 3, 4, 8)
    with pytest.raises(ValueError, match="overlaps"):
        _rot(x=x, out=y)
    t = _z(2, 3, 8, 4).transpose(2, 3)
    with pytest.raises(ValueError, match="adjacent"):
        _rot(x=t, out=t)


def test_rotary_frequencies():
    f = attention.rotary_frequencies((2, 3), base=100.0, device="cpu")
    assert f.dtype is torch.float64
    assert torch.allclose(f, torch.tensor([1, 100 ** -0.5, 1, 100 ** (-1 / 3), 100 ** (-2 / 3)], dtype=torch.float64), rtol=1e-15)
    g = attention.rotary_frequencies((2, 3), base=100.0, shared=True, device="cpu")
    assert torch.allclose(g, 100.0 ** (-torch.arange(5, dtype=torch.float64) / 5), rtol=1e-15)


def _cross(q=(2, 5, 4, 64), k=(2, 7, 2, 64), v=None, kind=torch.bfloat16, **kw):
    return attention.cross_attention(_z(*q, dtype=kind), _z(*k, dtype=kind), _z(*(v or k), dtype=kind), **kw)


@pytest.mark.parametrize("call, error", [
    (lambda: _cross(), "no CPU path"),
    (lambda: _cross(kind=torch.float32), "float32"),
    (lambda: _cross(k=(1, 7, 2, 64)), "do not fit"),
    (lambda: _cross(k=(2, 7, 2, 32)), "do not fit"),
    (lambda: _cross(v=(2, 8, 2, 64)), "do not fit"),
    (lambda: _cross(k=(2, 7, 3, 64)), "divide"),
    (lambda: _cross(q=(2, 5, 4, 12), k=(2, 7, 2, 12)), "multiple of 8"),
    (lambda: _cross(q=(2, 5, 4, 136), k=(2, 7, 2, 136)), "multiple of 8"),
    (lambda: _cross(lengths=torch.zeros(2, dtype=torch.int64)), "int64"),
    (lambda: _cross(lengths=torch.zeros(3, dtype=torch.int32)), "lengths"),
    (lambda: _cross(key_mask=torch.zeros(2, 8, dtype=torch.bool)), "key_mask"),
    (lambda: _cross(key_mask=torch.zeros(2, 7)), "float32"),
    (lambda: _cross(scale=0.0), "positive"),
    (lambda: _cross(scale=math.nan), "positive"),
    (lambda: _cross(scale=math.inf), "positive"),
])
def test_cross_attention_refuses(call, error):
    with pytest.raises((ValueError, TypeError, RuntimeError), match=error):
        call()


def _desc(**over):
    d = dict(q=P, k=P, v=P, o=P, lse=P, lengths=0, key_mask=0, scratch=P, dout=P, dq=P, dk=P, dv=P)
    s = {n: (5 * 256, 256, 64) for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv")}
    z = dict(mask_stride=0, batch=2, queries=5, keys=5, heads=4, groups=4, dim=64, type=1)
    scale = over.pop("scale", 0.125)
    for key, value in over.items():
        (d if key in d else z if key in z else s)[key.replace("_stride", "") if key not in d and key not in z else key] = value
    return struct.pack("=12q24q8qd", *d.values(), *(x for t in s.values() for x in t), *z.values(), scale)


@pytest.mark.parametrize("over, error", [
    (dict(q=0), "q is null"),
    (dict(k=P + 8), "k is null or not 16-byte"),
    (dict(v_stride=(1280, 256, 68)), "strides of v"),
    (dict(k_stride=(1280, 1 << 24, 64)), "token stride"),
    (dict(type=0), "types"),
    (dict(dim=60), "head dimension"),
    (dict(dim=256), "head dimension"),
    (dict(heads=6), "bad sizes"),
    (dict(keys=1 << 31), "out of range"),
    (dict(scale=-1.0), "scale"),
    (dict(scale=math.nan), "scale"),
])
def test_cross_attention_entry_points_refuse(over, error):
    for name in ("ried_xattn_fwd", "ried_xattn_bwd"):
        with pytest.raises(RuntimeError, match=error):
            getattr(lib, name)(_desc(**dict(over)), None)


def test_cross_attention_backward_entry_point_refuses():
    for over, error in ((dict(dout=0), "dout"), (dict(lse=0), "lse"), (dict(scratch=0), "scratch"), (dict(queries=0), "no queries"),
                        (dict(queries=1 << 24, q_stride=(0, 256, 64)), "2.31 bytes")):
        with pytest.raises(RuntimeError, match=error):
            lib.ried_xattn_bwd(_desc(**over), None)
    with pytest.raises(RuntimeError, match="null descriptor"):
        lib.ried_xattn_fwd(None, None)


def test_descriptor_has_the_layout_of_the_header():
    """ried_xattn_t: 12 pointers, 24 strides, 8 integers and the scale, without padding."""
    assert ops._XATTN.size == 12 * 8 + 24 * 8 + 8 * 8 + 8 == ctypes.sizeof(ctypes.c_longlong) * 44 + ctypes.sizeof(ctypes.c_double)


def test_layer_norm_entry_points_refuse():
    ok = [P, 8, None, None, P, 8, None, None, 4, 8, 1e-5, 1, 0, None]
    for at, value, error in ((0, None, "null"), (1, 4, "overlap"), (9, 0, "bad sizes"), (11, 3, "types"), (12, 2, "types"), (8, 1 << 32, "rows")):
        bad = list(ok)
        bad[at] = value
        with pytest.raises(RuntimeError, match=error):
            lib.ried_layer_norm_fwd(*bad)
    ok = [P, 8, P, 8, None, P, P, P, 8, P, None, P, 4, 8, 1, 0, None]
    for at, value, error in ((0, None, "null"), (5, None, "null"), (11, None, "scratch"), (8, 7, "overlap")):
        bad = list(ok)
        bad[at] = value
        with pytest.raises(RuntimeError, match=error):
            lib.ried_layer_norm_bwd(*bad)


def test_rotary_entry_point_refuses():
    ok = [P, 96, 32, 8, P, 96, 32, 8, P, 0, 9, 3, 1, P, 1, 2, 1, 0, 2, 3, 4, 8, 0, 0, 1, None]
    for at, value, error in ((0, None, "null"), (9, 3, "type"), (24, 5, "type"), (14, 3, "do not fit"), (14, -1, "sections"),
                             (20, 0, "sizes"), (5, 100, "in place")):
        bad = list(ok)
        bad[at] = value
        with pytest.raises(RuntimeError, match=error):
            lib.ried_rotary(*bad)


def test_adamw_entry_point_refuses():
    ok = [P, P, P, P, 1, P, P, 1e-3, 0.9, 0.99, 1e-8, 0.01, 0, 32, None]
    for at, value, error in ((0, None, "null"), (7, -1.0, "negative"), (8, 1.0, "betas"), (9, math.nan, "betas"), (12, 2, "fp32"), (13, 16, "bits")):
        bad = list(ok)
        bad[at] = value
        with pytest.raises(RuntimeError, match=error):
            lib.ried_adamw_jobs(*bad)


def test_scratch_sizes():
    assert ops.xattn_fwd_scratch_floats(2, 4096, 4096, 16, 16, 128) == 0          # enough rows: no split
    n = ops.xattn_fwd_scratch_floats(1, 1, 65536, 8, 8, 128)                      # one row per head: the keys are split
    assert n > 0 and n % (8 * 129) == 0
    assert ops.xattn_bwd_scratch_floats(1, 1, 1, 1, 1, 8) == 8
    assert ops.xattn_bwd_scratch_floats(0, 1, 1, 1, 1, 8) == 0
    assert ops.layer_norm_bwd_scratch_floats(0, 8, torch.float32) == 0
    assert ops.layer_norm_bwd_scratch_floats(10, 8, torch.float32) % 16 == 0


def test_adamw_refuses():
    p = torch.nn.Parameter(torch.zeros(4))
    with pytest.raises(ValueError, match="bits"):
        optim.AdamW([p], state_bits=16)
    with pytest.raises(ValueError, match="negative"):
        optim.AdamW([p], lr=-1.0)
    with pytest.raises(ValueError, match="betas"):
        optim.AdamW([p], betas=(0.9, 1.0))
    with pytest.raises(ValueError, match="negative"):
        optim.AdamW([{"params": [p], "eps": -1.0}])
    with pytest.raises(TypeError, match="number"):
        optim.AdamW([p], lr=torch.tensor(1e-3))
    opt = optim.AdamW([p])                                   # (parameters may still move to the device)
    p.grad = torch.zeros(4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        opt.step()
    with pytest.raises(ValueError, match="other parameter groups"):
        opt.load_state_dict({"state": {}, "param_groups": []})
    other = optim.AdamW([p], state_bits=8).state_dict()
    with pytest.raises(ValueError, match="8 bits"):
        opt.load_state_dict(other)
