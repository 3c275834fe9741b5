"""16-bit results of the 8-bit linear layer over long contractions.

Operands that the codes hold exactly, so that products are those of the inputs.

Sums of one sign: an instruction of 32 terms may lose 2^-22 of the sum so far (FP32 has 24 bits; two are left for alignment
inside the tensor core).  The accumulator is emptied after at most 4096 elements, 128 instructions, which loses at most
128 * 2^-22 = 2^-15 of the chunk's sum; n chunks are added in FP32, at most n * 2^-24.  The stored type adds half a step, eps / 2
relative to the value.

Integers: |a|, |b| <= 15 and at most 4096 terms a chunk give sums below 2^20, which the accumulator holds exactly in any order, and
totals below 2^24, so that the result is the sum rounded once.
"""
import pytest
import torch

import nvfp4_training as nv

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def positive(g, *shape, dtype):
    """Four significant bits over seven powers of two."""
    return torch.ldexp(torch.randint(8, 16, shape, device="cuda", generator=g) / 8, -torch.randint(0, 7, shape, device="cuda", generator=g)).to(dtype)


def bound(want, dtype, k):
    chunks = k // 4096 + 9                                                 # up to eight shares, each with a last short chunk
    return (torch.finfo(dtype).eps / 2 * 1.001 + 2.0 ** -15 + chunks * 2.0 ** -24) * want


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,k,n", [(2048, 264000, 2304), (128, 528000, 128), (1, 528000, 7)])      # paired tiles; split clusters
def test_long_sums_of_one_sign(m, k, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(k + n)
    x, w = positive(g, m, k, dtype=dtype), positive(g, n, k, dtype=dtype) / 8          # inside FP16
    with torch.no_grad():
        y = nv.fp8_linear(x, w)
    want = x[:64].double() @ w[:256].double().t()
    assert bool(((y[:64, :256].double() - want).abs() <= bound(want, dtype, k)).all())


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_long_weight_and_input_gradients(dtype):
    g = torch.Generator(device="cuda").manual_seed(3)
    long = 528000
    x, dy = positive(g, long, 128, dtype=dtype), positive(g, long, 128, dtype=dtype) / 8
    w = torch.ones(128, 128, device="cuda", dtype=dtype, requires_grad=True)
    dw, = torch.autograd.grad(nv.fp8_linear(x, w), w, dy)
    want = dy.double().t() @ x.double()
    assert bool(((dw.double() - want).abs() <= bound(want, dtype, long)).all())
    x = positive(g, 40, 128, dtype=dtype).requires_grad_(True)
    w, dy = positive(g, long, 128, dtype=dtype), positive(g, 40, long, dtype=dtype) / 8
    dx, = torch.autograd.grad(nv.fp8_linear(x, w), x, dy)
    want = dy.double() @ w.double()
    assert bool(((dx.double() - want).abs() <= bound(want, dtype, long)).all())


# one to four chunks, so that the accumulators alternate out of step with the tiles; ragged edges; rows that TMA cannot store
@pytest.mark.parametrize("k", [4096, 4097, 8192, 12300, 16384])
@pytest.mark.parametrize("m,n", [(2304, 2560), (2057, 2308), (300, 200), (16, 2048), (5, 9)])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_chunks_and_tiles(m, n, k, dtype):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    integers = lambda *shape: torch.randint(-15, 16, shape, device="cuda", generator=g).to(dtype)
    x, w, b = integers(m, k) / 8, integers(n, k), integers(n)              # an eighth: inside FP16
    with torch.no_grad():
        y, plain = nv.fp8_linear(x, w, b), nv.fp8_linear(x, w)
    want = x.double() @ w.double().t()
    assert torch.equal(plain, want.to(dtype)) and torch.equal(y, (want + b.double()).to(dtype))
    from nvfp4_training import _native
    _native.check_status()
