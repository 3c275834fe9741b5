"""The 8-bit linear layer: codes and scales bit for bit against the formula in 64 bits, products against those of the
dequantised operands in 64 bits.

Tolerance of a product: FP32 accumulation of K exact products.  Whatever the order, each of at most K / 32 additions of a
32-term dot product and each addition inside one is off by less than 2^-22 of the magnitudes summed so far (FP32 has 24 bits;
two are left for alignment inside the tensor core), hence 2^-22 * (K / 32 + 32) * sum |a b|, and half a step of the stored type.
"""
import pytest
import torch

import nvfp4_training as nv

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def quantised(x, block_rows, block_cols):
    """(values, exponents per block) by the formula, in 64 bits: e smallest with amax <= 448 * 2^e."""
    rows, cols = x.shape
    t = torch.nn.functional.pad(x.double(), (0, -cols % block_cols, 0, -rows % block_rows))
    t = t.view(t.shape[0] // block_rows, block_rows, t.shape[1] // block_cols, block_cols)
    amax = t.abs().amax(3, keepdim=True).amax(1, keepdim=True)
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, (e - 9 + (m > 0.875).int()).clamp(min=-127), 0)
    two = lambda n: ((n.long() + 1023) << 52).view(torch.float64)
    v = t / two(e)
    _, ve = torch.frexp(v)
    step = two((ve - 1).clamp(min=-6) - 3)
    q = torch.round(v / step) * step * two(e)
    return q.reshape(t.shape[0] * block_rows, -1)[:rows, :cols], e[:, 0, :, 0]


def codes_to_values(packing, rows, cols):
    """What codes [rows, cols_p] and the swizzled scale blocks behind them stand for, and the exponent of every (row, block)."""
    rb, cb = -(-rows // 128), -(-cols // 128)
    codes, scales = packing[:rows * cb * 128].view(rows, cb * 128), packing[rows * cb * 128:]
    words = scales.view(rb, cb, 32, 4, 4)                                  # row % 32, row / 32, four copies
    assert bool((words == words[..., :1]).all())
    e = words[..., 0].permute(0, 3, 2, 1).reshape(rb * 128, cb).int() - 127
    two = ((e.long() + 1023) << 52).view(torch.float64)[:rows].repeat_interleave(128, 1)
    return codes.view(torch.float8_e4m3fn).double() * two, e


def rand(g, *shape, dtype=F32):
    x = torch.randn(*shape, device="cuda", generator=g) * torch.exp(2 * torch.randn(shape[0], 1, device="cuda", generator=g))
    return x.to(dtype)


@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (128, 128), (130, 257), (37, 1000), (300, 264), (513, 40)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("square", [False, True])
def test_codes_and_scales(rows, cols, dtype, square):
    from nvfp4_training.fp8 import _quantize
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + cols)
    x = rand(g, rows, cols, dtype=dtype)
    x[:, cols // 2] = 0
    if rows > 128:
        x[128:, :128] = 0                                                  # a block of zeros
        x[0, :] = 448 * 2.0 ** torch.randint(-3, 3, (cols,), device="cuda", generator=g)      # exactly the largest code
    q, t, sums = _quantize(x, row=True, col=True, square=square, column_sums=True)
    shape = (128, 128) if square else (1, 128)
    want, e = quantised(x, *shape)
    got, ge = codes_to_values(q, rows, cols)
    assert torch.equal(got[:, :cols], want) and not got[:, cols:].any()
    assert torch.equal(ge[:rows], e.repeat_interleave(128, 0)[:rows] if square else e)
    want, e = quantised(x.t(), *shape)
    got, ge = codes_to_values(t, cols, rows)
    assert torch.equal(got[:, :rows], want) and not got[:, rows:].any()
    assert torch.equal(ge[:cols], e.repeat_interleave(128, 0)[:cols] if square else e)
    block_sums = torch.nn.functional.pad(x.double(), (0, 0, 0, -rows % 128)).view(-1, 128, cols).sum(1)
    assert bool(((sums.double() - block_sums).abs() <= 2.0 ** -20 * x.double().abs().sum(0)).all())
    only, none, _ = _quantize(x, row=True, col=False, square=square)
    assert none is None and torch.equal(only, q)


def test_range_of_the_scale():
    """Blocks at the ends of the number range, and blocks with values that are not finite."""
    from nvfp4_training.fp8 import _quantize
    x = torch.zeros(8, 256, device="cuda", dtype=BF16)
    x[0, :4] = torch.tensor([3.3e38, -1e38, 1e36, 1.0])
    x[1, :4] = torch.tensor([2.0 ** -126, -(2.0 ** -127), 2.0 ** -133, 0])
    x[2, 0], x[2, 1] = 2.0 ** -133, -(2.0 ** -133)
    x[3, 5], x[4, 6], x[5, 7] = float("inf"), float("-inf"), float("nan")
    x[3:6, 128:] = 1.5
    packing, _, _ = _quantize(x, row=True, col=False)
    got, e = codes_to_values(packing, 8, 256)
    want, we = quantised(x[:3], 1, 128)
    assert torch.equal(got[:3], want) and torch.equal(e[:3], we)
    assert got[3:6, :128].isnan().all() and torch.equal(got[3:6, 128:], x[3:6, 128:].double()) and not got[6:].any()


def product_bound(a, b, dtype, want, k):
    spread = a.abs() @ b.abs().t()
    return torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + 2.0 ** -22 * (k / 32 + 32) * spread + (2.0 ** -25 if dtype == F16 else 0)


def check(got, want, bound):
    over = (got.double() - want).abs() - bound
    assert got.shape == want.shape and bool((over <= 0).all()), over.max().item()


# paired 256 x 256 tiles, split clusters of every size, one token, ragged and tiny extents, more than one wave
SHAPES = [(1, 128, 128), (1, 4096, 512), (1, 1024, 4096), (7, 1, 1), (3, 130, 1), (128, 256, 1024), (129, 384, 136), (256, 256, 256), (300, 200, 640),
          (1000, 1152, 1072), (513, 640, 1000), (2048, 256, 4096), (4096, 1024, 2304), (77, 3000, 4000)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype,wdtype", [(BF16, BF16), (F32, F32), (F16, F32), (BF16, F32)])
def test_forward_and_backward(m, k, n, dtype, wdtype):
    g = torch.Generator(device="cuda").manual_seed(m + k + n)
    x = rand(g, m, k, dtype=dtype)
    x = (x.float() / x.float().abs().max() * 20).to(dtype).requires_grad_(True)       # inside FP16
    w = (torch.randn(n, k, device="cuda", generator=g) / k ** 0.5).to(wdtype).requires_grad_(True)
    b = torch.randn(n, device="cuda", generator=g).to(wdtype).requires_grad_(True)
    dy = (0.01 * torch.randn(m, n, device="cuda", generator=g)).to(dtype)
    y = nv.fp8_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert (y.dtype, dx.dtype, dw.dtype, db.dtype) == (dtype, dtype, wdtype, wdtype)
    xq, wq, gq = quantised(x.detach(), 1, 128)[0], quantised(w.detach(), 128, 128)[0], quantised(dy, 1, 128)[0]
    want = xq @ wq.t() + b.detach().double()
    check(y, want, product_bound(xq, wq, dtype, want, k) + 2.0 ** -23 * b.detach().double().abs())
    want = gq @ wq
    check(dx, want, product_bound(gq, wq.t(), dtype, want, n))
    gt, xt = quantised(dy.t(), 1, 128)[0], quantised(x.detach().t(), 1, 128)[0]
    want = gt @ xt.t()
    check(dw, want, product_bound(gt, xt, wdtype, want, m))
    want = dy.double().sum(0)
    check(db, want, torch.finfo(wdtype).eps / 2 * 1.01 * want.abs() + 2.0 ** -20 * dy.double().abs().sum(0))
    packed = nv.fp8_pack(w)
    with torch.no_grad():
        assert torch.equal(nv.fp8_linear(x, packed, b), y) and torch.equal(packed.dequantize().double(), wq.float().double())
    again = nv.fp8_linear(x, packed, b)
    assert torch.equal(torch.autograd.grad(again, x, dy)[0], dx)
    from nvfp4_training import _native
    _native.check_status()


@pytest.mark.parametrize("m,k,n", [(200, 384, 260), (1, 1024, 512), (2000, 512, 4096)])
def test_only_what_is_asked_for(m, k, n):
    g = torch.Generator(device="cuda").manual_seed(1)
    x, w, b = rand(g, m, k, dtype=BF16), rand(g, n, k, dtype=BF16), rand(g, 1, n, dtype=F32)[0]
    dy = rand(g, m, n, dtype=BF16)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(nv.fp8_linear(*full), full, dy)
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        assert torch.equal(torch.autograd.grad(nv.fp8_linear(*some), some[i], dy)[0], want[i])
    assert torch.equal(nv.fp8_linear(x, w), nv.fp8_linear(x, w, torch.zeros_like(b)))


def test_shapes_strides_and_empty_batches():
    g = torch.Generator(device="cuda").manual_seed(2)
    w = rand(g, 200, 256, dtype=BF16)
    base = rand(g, 60, 600, dtype=BF16)
    for x in (base[:, 17:273], base[:, ::2][:, :256], base[:, :256].t().contiguous().t(), base[:1, :256].expand(60, 256), base[:, 8:264].view(3, 4, 5, 256)):
        assert torch.equal(nv.fp8_linear(x, w), nv.fp8_linear(x.contiguous(), w))
    assert torch.equal(nv.fp8_linear(base[:, :256], w.t().contiguous().t()), nv.fp8_linear(base[:, :256], w))
    assert torch.equal(nv.fp8_linear(base[0, :256], w), nv.fp8_linear(base[:1, :256], w)[0])
    leaf = base[:, :256].clone().requires_grad_(True)
    dy = rand(g, 200, 60, dtype=BF16).t()                                 # a transposed gradient
    assert torch.equal(torch.autograd.grad(nv.fp8_linear(leaf, w), leaf, dy)[0], torch.autograd.grad(nv.fp8_linear(leaf, w), leaf, dy.contiguous())[0])
    leaves = [torch.empty(0, 256, device="cuda", dtype=BF16, requires_grad=True), w.clone().requires_grad_(True),
              torch.ones(200, device="cuda", requires_grad=True)]
    y = nv.fp8_linear(*leaves)
    dx, dw, db = torch.autograd.grad(y, leaves, torch.empty_like(y))
    assert y.shape == (0, 200) and dx.shape == (0, 256) and not dw.any() and not db.any()


@pytest.mark.parametrize("m", [1, 64, 700])
def test_rows_do_not_touch_each_other(m):
    """A row's result depends on that row alone, also beside rows that are not finite."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w = rand(g, m, 640, dtype=BF16), rand(g, 520, 640, dtype=BF16)
    y = nv.fp8_linear(x, w)
    bad = x.clone()
    bad[0, 3] = float("nan")
    z = nv.fp8_linear(bad, w)
    assert z[0].isnan().all() and torch.equal(z[1:], y[1:])


def test_gradient_against_differences():
    """The layer's own function is a step function, so the products' gradients are held against differences where rounding
    does nothing: small whole numbers, a power of two as the step."""
    g = torch.Generator(device="cuda").manual_seed(4)
    whole = lambda *shape: torch.randint(-3, 4, shape, device="cuda", generator=g).float()
    x, w, b, dy = whole(40, 256), whole(72, 256), whole(72), whole(40, 72)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(nv.fp8_linear(*leaves), leaves, dy)
    for i, grad in enumerate(grads):
        direction = whole(*grad.shape)
        at = [t.detach() for t in leaves]
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + direction, at[i] - direction           # at most 6: exact in e4m3
        slope = ((nv.fp8_linear(*plus).double() - nv.fp8_linear(*minus).double()) * dy.double()).sum() / 2
        assert slope.item() == (grad.double() * direction.double()).sum().item()


def test_streams_graphs_and_repeats():
    g = torch.Generator(device="cuda").manual_seed(5)
    for m, k, n in ((16, 1024, 512), (900, 512, 1024)):
        x, w = rand(g, m, k, dtype=BF16).requires_grad_(True), rand(g, n, k, dtype=BF16).requires_grad_(True)
        b = rand(g, 1, n)[0].requires_grad_(True)
        dy = rand(g, m, n, dtype=BF16)
        keep = nv.fp8_linear(x, w, b)
        want = torch.autograd.grad(keep, (x, w, b), dy, retain_graph=True)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = torch.autograd.grad(nv.fp8_linear(x, w, b), (x, w, b), dy)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        leaves = [t.detach().clone().requires_grad_(True) for t in (x, w, b)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = nv.fp8_linear(*leaves)
            grads = torch.autograd.grad(y, leaves, dy)
        with torch.no_grad():
            leaves[0].mul_(-1.5)
            leaves[1].add_(0.25)
        for _ in range(2):
            graph.replay()
        again = nv.fp8_linear(*leaves)
        assert torch.equal(y, again) and all(torch.equal(p, q) for p, q in zip(grads, torch.autograd.grad(again, leaves, dy)))
