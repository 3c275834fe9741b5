"""Layer norm (with the residual sum) against the formulas in 64 bits.

Tolerances: a stored result is off by half a step of its type relative to its value, u = finfo(t).eps / 2, plus what FP32
arithmetic leaves: z comes from a difference and a product with rstd (relative error under 2^-20 of max |z| for the widths
here, whose sums of up to 2^16 terms are trees), so every bound below is u * |want| + 2^-18 * scale, where scale is the
largest magnitude that enters the sum the value comes from.
"""
import pytest
import torch

import nvfp4_training as nv

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
LOOSE = 2.0 ** -18


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def check(got, want, scale, what, terms=1):
    bound = unit(got.dtype) * want.abs() * 1.01 + LOOSE * scale * terms
    if got.dtype == F16:
        bound = bound + 2.0 ** -25             # half a step of the subnormal range
    over = (got.double() - want).abs() - bound
    assert got.shape == want.shape and bool((over <= 0).all()), (what, over.max().item())


def reference(total, w, b, eps):
    s = total.double()
    mu = s.mean(-1, keepdim=True)
    var = ((s - mu) ** 2).mean(-1, keepdim=True)
    rstd = (var + eps) ** -0.5
    z = (s - mu) * rstd
    h = z if w is None else z * w.double()
    return (h if b is None else h + b.double()), z, rstd


def gradients(z, rstd, w, dh, dsum):
    dh = dh.double()
    u = dh if w is None else dh * w.double()
    dx = rstd * (u - u.mean(-1, keepdim=True) - z * (u * z).mean(-1, keepdim=True))
    return dx if dsum is None else dx + dsum.double(), (dh * z).sum(0), dh.sum(0), u


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


# one warp, several vectors of it, a CTA per row, odd widths, one feature, past the register kernels (element by element
# above 4096, in vectors above 32768 elements)
WIDTHS = [1, 7, 8, 40, 255, 256, 520, 768, 1027, 2048, 4096, 4104, 5120, 9001, 16400]


@pytest.mark.parametrize("cols", WIDTHS)
@pytest.mark.parametrize("dtype,delta_dtype,out_dtype,wdtype", [(BF16, BF16, BF16, F32), (F16, None, F16, F16), (F32, BF16, BF16, F32), (F32, F32, F32, BF16)])
def test_forward_and_backward(cols, dtype, delta_dtype, out_dtype, wdtype):
    g = torch.Generator(device="cuda").manual_seed(cols)
    rows = 37 if cols < 4000 else 11
    x = (rand(g, rows, cols) + 3 * rand(g, rows, 1)).to(dtype).requires_grad_(True)
    delta = None if delta_dtype is None else rand(g, rows, cols, dtype=delta_dtype).requires_grad_(True)
    w = (1 + 0.2 * rand(g, cols)).to(wdtype).requires_grad_(True)
    b = (0.2 * rand(g, cols)).to(wdtype).requires_grad_(True)
    dh = rand(g, rows, cols, dtype=out_dtype)
    dsum = rand(g, rows, cols, dtype=dtype) if delta is not None else None
    if delta is None:
        total, h = x.detach(), nv.layer_norm(x, w, b, out_dtype=out_dtype)
        grads = torch.autograd.grad(h, (x, w, b), dh)
        dx, dd, dw, db = grads[0], None, *grads[1:]
    else:
        total, h = nv.add_layer_norm(x, delta, w, b, out_dtype=out_dtype)
        assert torch.equal(total, (x.detach().float() + delta.detach().float()).to(dtype))
        dx, dd, dw, db = torch.autograd.grad((h, total), (x, delta, w, b), (dh, dsum))
        assert dd.dtype == delta_dtype
    assert h.dtype == out_dtype and dx.dtype == dtype and dw.dtype == wdtype and db.dtype == wdtype
    want, z, rstd = reference(total.detach(), w.detach(), b.detach(), 1e-5)
    # the difference s - mu loses what FP32 loses of |s|: 2^-24 |s| rstd, inside LOOSE as long as |s| rstd < 2^6
    spread = (total.detach().double().abs() * rstd).max()
    check(h, want, max(1.0, spread.item()), "h")
    wdx, wdw, wdb, u = gradients(z, rstd, w.detach(), dh, dsum)
    size = (rstd * u.abs().max(-1, keepdim=True).values).max().item() * max(1.0, z.abs().max().item()) ** 2 + 1
    check(dx, wdx, size * max(1.0, spread.item()), "dx")
    if dd is not None:
        check(dd, wdx, size * max(1.0, spread.item()), "ddelta")
    check(dw, wdw, dh.abs().max().item() * max(1.0, spread.item()) * rows, "dw")
    check(db, wdb, dh.abs().max().item() * rows, "db")


def test_gradient_against_differences():
    """d loss along a direction, in 64-bit differences of the formula, against the kernel's gradients (FP32 in and out)."""
    g = torch.Generator(device="cuda").manual_seed(5)
    x, d, w, b = (rand(g, 9, 72), rand(g, 9, 72), 1 + 0.1 * rand(g, 72), rand(g, 72))
    dh, dt = rand(g, 9, 72), rand(g, 9, 72)
    leaves = [t.requires_grad_(True) for t in (x, d, w, b)]
    total, h = nv.add_layer_norm(*leaves)
    grads = torch.autograd.grad((h, total), leaves, (dh, dt))

    def loss(ts):
        s = ts[0] + ts[1]
        return (reference(s, ts[2], ts[3], 1e-5)[0] * dh.double()).sum() + (s * dt.double()).sum()
    for i, grad in enumerate(grads):
        direction = rand(g, *grad.shape).double()
        at = [t.detach().double() for t in leaves]
        step = 1e-5
        plus, minus = list(at), list(at)
        plus[i], minus[i] = at[i] + step * direction, at[i] - step * direction
        slope = (loss(plus) - loss(minus)).item() / (2 * step)
        along = (grad.double() * direction).sum().item()
        # central differences: step^2 in 64 bits; FP32 gradients: LOOSE of the summed magnitudes
        assert abs(slope - along) <= 1e-6 * abs(slope) + LOOSE * (grad.double() * direction).abs().sum().item() + 1e-6


@pytest.mark.parametrize("offset", [0.0, 1000.0])
def test_large_mean_and_constant_rows(offset):
    """A mean far above the spread keeps its variance; a constant row has variance 0 and gives the bias."""
    g = torch.Generator(device="cuda").manual_seed(3)
    x = rand(g, 16, 1024) + offset
    x[3] = 7.0
    b = rand(g, 1024)
    h = nv.layer_norm(x, None, b)
    want = reference(x, None, b, 1e-5)[0]
    spread = 1.0 + offset          # |s| rstd with a spread of one
    check(h[:3], want[:3], spread, "h")
    assert torch.equal(h[3], b)


@pytest.mark.parametrize("layout", ["pitched", "transposed", "expanded", "4d", "offset"])
def test_strides(layout):
    g = torch.Generator(device="cuda").manual_seed(8)
    if layout == "pitched":
        x = rand(g, 33, 400, dtype=BF16)[:, 48:304]
    elif layout == "transposed":
        x = rand(g, 256, 33, dtype=BF16).t()
    elif layout == "expanded":
        x = rand(g, 1, 256, dtype=BF16).expand(33, 256)
    elif layout == "4d":
        x = rand(g, 2, 5, 3, 256, dtype=BF16).transpose(1, 2)
    else:
        x = rand(g, 33 * 256 + 1, dtype=BF16)[1:].view(33, 256)       # rows that start off the 16-byte grid
    h = nv.layer_norm(x)
    check(h, reference(x, None, None, 1e-5)[0], 8.0, "h")
    leaf = x.detach().requires_grad_(True)
    dh = rand(g, *x.shape[:-1], 512, dtype=BF16)[..., ::2]            # a gradient with strides of its own
    dx, = torch.autograd.grad(nv.layer_norm(leaf), leaf, dh)
    _, z, rstd = reference(x, None, None, 1e-5)
    check(dx, gradients(z, rstd, None, dh, None)[0], 64.0, "dx")


def test_only_some_inputs_need_gradients():
    g = torch.Generator(device="cuda").manual_seed(4)
    x, w, b = rand(g, 40, 128, dtype=BF16), 1 + rand(g, 128), rand(g, 128)
    dh = rand(g, 40, 128, dtype=BF16)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(nv.layer_norm(*full), full, dh)
    for i in range(3):
        some = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(nv.layer_norm(*some), some[i], dh)
        assert torch.equal(got, want[i])
    # only the residual path carries a gradient: it passes through, the parameters get zeros
    leaves = [t.clone().requires_grad_(True) for t in (x, x, w, b)]
    total, h = nv.add_layer_norm(*leaves)
    dx, dd, dw, db = torch.autograd.grad(total, leaves, dh)
    assert torch.equal(dx, dh) and torch.equal(dd, dh) and not dw.any() and not db.any()
    # only the norm's own path
    total, h = nv.add_layer_norm(*leaves)
    dx, dd = torch.autograd.grad(h, leaves[:2], dh)
    assert torch.equal(dx, dd)


def test_empty_and_single_rows():
    w = torch.ones(64, device="cuda", requires_grad=True)
    b = torch.zeros(64, device="cuda", requires_grad=True)
    x = torch.empty(0, 64, device="cuda", dtype=BF16, requires_grad=True)
    h = nv.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(h, (x, w, b), torch.empty(0, 64, device="cuda", dtype=BF16))
    assert h.shape == dx.shape == (0, 64) and not dw.any() and not db.any()
    v = torch.randn(64, device="cuda")
    check(nv.layer_norm(v), reference(v, None, None, 1e-5)[0], 8.0, "vector")


def test_not_finite_rows_stay_apart():
    x = torch.randn(40, 256, device="cuda")
    clean = nv.layer_norm(x)
    x[5, 3], x[9, 200] = float("nan"), float("inf")
    h = nv.layer_norm(x)
    assert h[5].isnan().all() and h[9].isnan().any()
    keep = [i for i in range(40) if i not in (5, 9)]
    assert torch.equal(h[keep], clean[keep])


def test_repeats_bit_for_bit():
    g = torch.Generator(device="cuda").manual_seed(6)
    for cols in (768, 5120, 1027):
        leaves = [rand(g, 3000, cols, dtype=BF16).requires_grad_(True), torch.ones(cols, device="cuda", requires_grad=True),
                  torch.zeros(cols, device="cuda", requires_grad=True)]
        dh = rand(g, 3000, cols, dtype=BF16)
        runs = [torch.autograd.grad(nv.layer_norm(*leaves), leaves, dh) for _ in range(3)]
        assert all(torch.equal(a, c) for r in runs[1:] for a, c in zip(runs[0], r))


def test_other_stream_and_graph():
    g = torch.Generator(device="cuda").manual_seed(7)
    x = rand(g, 300, 512, dtype=BF16).requires_grad_(True)
    w = (1 + 0.1 * rand(g, 512)).requires_grad_(True)
    dh = rand(g, 300, 512, dtype=BF16)
    eager = nv.layer_norm(x, w)          # this eager graph stays alive while the same leaves are captured
    want = torch.autograd.grad(eager, (x, w), dh, retain_graph=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(nv.layer_norm(x, w), (x, w), dh)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    captured = [t.detach().clone().requires_grad_(True) for t in (x, w)]
    graphs = []
    for _ in range(2):                   # two graphs with the same operators
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            h = nv.layer_norm(*captured)
            grads = torch.autograd.grad(h, captured, dh)
        graphs.append((graph, h, grads))
    with torch.no_grad():
        captured[0].mul_(2)
        captured[1].add_(1)
    fresh = [t.detach().clone().requires_grad_(True) for t in captured]
    h2 = nv.layer_norm(*fresh)
    want = torch.autograd.grad(h2, fresh, dh)
    for graph, h, grads in graphs + graphs[:1]:
        graph.replay()
        assert torch.equal(h, h2) and all(torch.equal(a, b) for a, b in zip(grads, want))


def test_module_under_autocast_hands_its_amax_on():
    from nvfp4_training._backend.quant import known_amax
    torch.manual_seed(0)
    norm = nv.LayerNorm(320).cuda()
    norm.load_state_dict(torch.nn.LayerNorm(320).state_dict())
    x = torch.randn(64, 320, device="cuda", requires_grad=True)
    assert norm(x).dtype == F32
    with torch.autocast("cuda", dtype=BF16):
        h = norm(x)
    assert h.dtype == BF16 and known_amax(h)[0].item() == h.detach().abs().max().item()
    h.float().square().sum().backward()
    assert x.grad is not None and norm.weight.grad.dtype == F32
    plain = torch.nn.LayerNorm(320, elementwise_affine=False)
    assert nv.LayerNorm(320, elementwise_affine=False)(x).shape == plain(x).shape


@pytest.mark.parametrize("cols", [16, 64, 1024, 2040, 2048, 4096, 6144, 8184, 8192, 8200])
@pytest.mark.parametrize("rows", [1, 3, 700])
@pytest.mark.parametrize("dtype,delta_dtype", [(BF16, BF16), (F32, BF16), (F32, F32)])
def test_widths_around_the_kernels_borders(cols, rows, dtype, delta_dtype):
    """Few and many rows on both sides of each width at which the work is divided differently (tolerances as above)."""
    g = torch.Generator(device="cuda").manual_seed(cols + rows)
    x, d = rand(g, rows, cols, dtype=dtype).requires_grad_(True), rand(g, rows, cols, dtype=delta_dtype).requires_grad_(True)
    w, b = (1 + 0.2 * rand(g, cols)).requires_grad_(True), rand(g, cols).requires_grad_(True)
    dh, ds = rand(g, rows, cols, dtype=dtype), rand(g, rows, cols, dtype=dtype)
    total, h = nv.add_layer_norm(x, d, w, b)
    grads = torch.autograd.grad((h, total), (x, d, w, b), (dh, ds))
    want, z, rstd = reference(total.detach(), w.detach(), b.detach(), 1e-5)
    check(h, want, 8.0, "h")
    wdx, wdw, wdb, u = gradients(z, rstd, w.detach(), dh, ds)
    size = (rstd * u.abs().max(-1, keepdim=True).values).max().item() * max(1.0, z.abs().max().item()) ** 2 + 1
    for got, want, scale in zip(grads, (wdx, wdx, wdw, wdb), (8 * size, 8 * size, 8 * dh.abs().max().item() * rows, dh.abs().max().item() * rows)):
        check(got, want, scale, "gradients")
    from nvfp4_training import _native
    _native.check_status()


def test_second_derivatives_are_refused_where_they_would_pass_through():
    x = torch.randn(4, 64, device="cuda", requires_grad=True)
    pos = torch.arange(4, device="cuda").view(1, 4, 1)
    w = torch.randn(64, 64, device="cuda", requires_grad=True)
    for y in (nv.layer_norm(x), nv.rotary_axes(x.view(1, 4, 1, 64), None, pos, (32,))[0], nv.fp8_linear(x, w)):
        dx, = torch.autograd.grad((y * y).sum(), x, create_graph=True)       # first derivatives with a graph are fine
        with pytest.raises(RuntimeError):
            torch.autograd.grad(dx.sum(), x)
