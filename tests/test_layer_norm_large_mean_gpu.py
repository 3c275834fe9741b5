"""The layer norm where rows lie far from zero against their spread.

A constant row of few significant bits has a sum that FP32 holds, so its mean is exact, its differences are zero, and so is z: the
result is the bias, nothing reaches the weight's gradient, and dx is rstd (u - mean(u)) with rstd = 1 / sqrt(eps).
"""
import pytest
import torch

import nvfp4_training as nv

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
VALUES = [1000.0, -1000.0, 248.0, 7.0, 0.0]

# every way the rows are fetched and shared out: odd widths, groups of rows, warps with a part of their columns, eight and
# sixteen columns a thread, past 8192
widths = pytest.mark.parametrize("cols", [7, 49, 64, 520, 768, 1000, 1024, 1027, 2048, 2360, 2560, 4096, 5120, 6144, 8192, 9001])
types = pytest.mark.parametrize("dtype,out_dtype", [(F32, F32), (F32, BF16), (BF16, BF16), (F16, F16)])


def constant_rows(cols, dtype, out_dtype):
    g = torch.Generator(device="cuda").manual_seed(cols)
    x = torch.tensor(VALUES, device="cuda")[:, None].expand(len(VALUES), cols).to(dtype)
    w, b = 1 + torch.randn(cols, device="cuda", generator=g), torch.randn(cols, device="cuda", generator=g)
    return x, w, b, torch.randn(len(VALUES), cols, device="cuda", generator=g).to(out_dtype)


@widths
@types
def test_constant_rows_give_the_bias(cols, dtype, out_dtype):
    x, w, b, _ = constant_rows(cols, dtype, out_dtype)
    want = b.to(out_dtype).expand(len(VALUES), cols)
    assert torch.equal(nv.layer_norm(x, w, b, out_dtype=out_dtype), want)
    total, h = nv.add_layer_norm(x, torch.zeros_like(x), w, b, out_dtype=out_dtype)
    assert torch.equal(h, want) and torch.equal(total, x)


@widths
@types
def test_constant_rows_leave_the_weight_alone(cols, dtype, out_dtype):
    x, w, b, dh = constant_rows(cols, dtype, out_dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(nv.layer_norm(*leaves, out_dtype=out_dtype), leaves, dh)
    assert not dw.any()
    u = dh.double() * w.double()
    want = (u - u.mean(-1, keepdim=True)) * 1e-5 ** -0.5
    # a product, a mean over a tree of sums, two more operations and rsqrt in FP32, each below 2^-22 of the largest |u| rstd
    bound = torch.finfo(dtype).eps / 2 * 1.01 * want.abs() + 2.0 ** -18 * u.abs().max(-1, keepdim=True).values * 1e-5 ** -0.5
    assert bool(((dx.double() - want).abs() <= bound).all())
    assert bool(((db.double() - dh.double().sum(0)).abs() <= 2.0 ** -21 * dh.double().abs().sum(0)).all())
