"""The bounds of tests/cross_norms.py: they hold for gradients that are rounded where the kernels round, and not for gradients
with a mistake.  The mistakes are made here, in the formulas, on the CPU."""
import pytest
import torch

import cross_norms as N


def check(shape, kind, lengths=None, mask=None, seed=0):
    q, k, v, dout = N.inputs(sum(shape) + seed, shape, kind)
    bounds = N.exact_and_variance(q, k, v, dout, lengths, mask)
    rows = shape[1]
    got = N.ratios(N.rounded(q, k, v, dout, lengths, mask), bounds, rows)
    assert max(got.values()) <= 1, got
    right, wrong = N.mutants(q, k, v, dout, lengths, mask)
    for what, grads in wrong.items():
        for name, t in grads.items():
            size = right[name].norm().item()
            if what in ("no Dl", "Dl * 0.9") or size > 1e-9:                # (a factor on a gradient of zero is no mistake)
                assert N.ratio(t, *bounds[name], rows) > 1, (what, name, N.ratio(t, *bounds[name], rows))


@pytest.mark.parametrize("shape, kind", N.CASES)
def test_bounds_tell_roundings_from_mistakes(shape, kind):
    check(shape, kind)


@pytest.mark.parametrize("shape", [(4, 40, 130, 4, 2, 64), (4, 200, 64, 2, 2, 32), (4, 3, 1100, 6, 2, 96), (4, 257, 900, 2, 1, 128)])
@pytest.mark.parametrize("kind", [N.BF16, N.F16])
def test_bounds_with_hidden_keys(shape, kind):
    lengths, mask = N.some_keys(sum(shape), shape)
    check(shape, kind, lengths, mask)
    check(shape, kind, lengths, None, seed=1)


def test_a_head_without_keys_allows_nothing():
    shape = (4, 5, 70, 2, 2, 64)
    q, k, v, dout = N.inputs(3, shape, N.BF16)
    lengths = torch.tensor([70, 0, 33, 2], dtype=torch.int32)
    bounds = N.exact_and_variance(q, k, v, dout, lengths)
    got = {name: t.clone() for name, (t, _) in bounds.items()}
    assert max(N.ratios(got, bounds, 5).values()) == 0
    got["dq"][1, 0, 0, 0] = 1e-30
    assert N.ratios(got, bounds, 5)["dq"] > 1
