"""FP32 results of the 8-bit linear layer over long contractions and many tiles.

Operands that the codes hold exactly, so that products are those of the inputs.

Long sums of one sign: an instruction of 32 terms may lose 2^-22 of the sum so far (FP32 has 24 bits; two are left for alignment
inside the tensor core).  The accumulator is emptied after 2048 elements, 64 instructions, which loses at most 64 * 2^-22 of the
chunk's sum; n chunks are added in FP32, at most n * 2^-24.  Together 2^-16 + n * 2^-24 of the result, whatever the length.

Integers: |a|, |b| <= 15 and at most 6016 terms give sums below 2^21, which FP32 holds exactly in any order.
"""
import pytest
import torch

import nvfp4_training as nv

pytestmark = pytest.mark.gpu


def positive(g, *shape):
    """Four significant bits over seven powers of two: products have steps of 2^-18 and long sums of them more than 24 bits."""
    return torch.ldexp(torch.randint(8, 16, shape, device="cuda", generator=g) / 8, -torch.randint(0, 7, shape, device="cuda", generator=g))


def integers(g, *shape):
    return torch.randint(-15, 16, shape, device="cuda", generator=g).float()


@pytest.mark.parametrize("m,k,n", [(2048, 66000, 2304), (128, 528000, 128), (1, 528000, 7)])       # paired tiles; split clusters
def test_long_sums_of_one_sign(m, k, n):
    g = torch.Generator(device="cuda").manual_seed(k + n)
    x, w = positive(g, m, k), positive(g, n, k)
    with torch.no_grad():
        y = nv.fp8_linear(x, w)
    want = x[:64].double() @ w[:256].double().t()
    chunks = k // 2048 + 9                                                 # up to eight shares, each with a last short chunk
    assert bool(((y[:64, :256].double() - want).abs() <= (2.0 ** -16 + chunks * 2.0 ** -24) * want).all())


def test_long_weight_gradient():
    g = torch.Generator(device="cuda").manual_seed(3)
    tokens = 528000
    x, dy = positive(g, tokens, 128), positive(g, tokens, 128)
    w = torch.ones(128, 128, device="cuda", requires_grad=True)
    dw, = torch.autograd.grad(nv.fp8_linear(x, w), w, dy)
    want = dy.double().t() @ x.double()
    assert bool(((dw.double() - want).abs() <= (2.0 ** -16 + (tokens // 2048 + 9) * 2.0 ** -24) * want).all())


# one to three chunks, so that the accumulators alternate out of step with the tiles; ragged edges; rows that TMA cannot store
@pytest.mark.parametrize("k", [128, 2048, 2050, 4097, 6016])
@pytest.mark.parametrize("m,n", [(4096, 4864), (4100, 4865), (2057, 2308), (300, 200), (16, 4096), (5, 9)])
def test_chunks_and_tiles(m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    x, w, b = integers(g, m, k), integers(g, n, k), integers(g, n)
    with torch.no_grad():
        y, plain = nv.fp8_linear(x, w, b), nv.fp8_linear(x, w)
    want = x.double() @ w.double().t()
    assert torch.equal(plain.double(), want) and torch.equal(y.double(), want + b.double())
    from nvfp4_training import _native
    _native.check_status()
