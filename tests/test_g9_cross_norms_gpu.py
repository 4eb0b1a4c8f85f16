"""Cross attention's gradients within bounds of their errors' norms (cross_norms.py, where the bounds are derived; that they
tell a rounding from a mistake is checked on the CPU)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

import cross_norms as N
from reid_gan_amd import attention


def check(shape, kind, lengths=None, mask=None, seed=0):
    q, k, v, dout = N.inputs(sum(shape) + seed, shape, kind, "cuda")
    leaves = [t.detach().clone().requires_grad_() for t in (q, k, v)]
    grads = torch.autograd.grad(attention.cross_attention(*leaves, lengths, mask), leaves, dout)
    got = {name: t.transpose(1, 2) for name, t in zip(("dq", "dk", "dv"), grads)}
    off = N.ratios(got, N.exact_and_variance(q, k, v, dout, lengths, mask), shape[1])
    print(shape, kind, {name: round(x, 2) for name, x in off.items()})
    assert max(off.values()) <= 1, off


@pytest.mark.parametrize("shape, kind", N.CASES)
def test_cross_attention_gradient_norms(shape, kind):
    check(shape, kind)


@pytest.mark.parametrize("shape", [(4, 40, 130, 4, 2, 64), (4, 200, 64, 2, 2, 32), (4, 3, 1100, 6, 2, 96), (4, 257, 900, 2, 1, 128)])
@pytest.mark.parametrize("kind", [N.BF16, N.F16])
def test_cross_attention_gradient_norms_with_hidden_keys(shape, kind):
    lengths, mask = N.some_keys(sum(shape), shape, "cuda")
    check(shape, kind, lengths, mask)
    check(shape, kind, lengths, None, seed=1)


@pytest.mark.parametrize("shape", [(4, 1024, 1500, 16, 4, 64), (2, 2048, 2048, 4, 4, 128), (1, 2, 8192, 8, 8, 64), (1, 4096, 8192, 2, 1, 128)])
@pytest.mark.parametrize("kind", [N.BF16, N.F16])
def test_cross_attention_gradient_norms_of_large_batches(shape, kind):
    check(shape, kind)
    check(shape, kind, N.some_keys(sum(shape), shape, "cuda")[0], None, seed=1)
