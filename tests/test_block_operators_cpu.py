"""Refusals of the transformer-block operators: the public functions' checks of their arguments and the C entry points',
neither of which needs a GPU."""
import ctypes as C

import pytest
import torch

import nvfp4_training as nv

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def x(*shape, dtype=BF16):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: nv.layer_norm([1.0])),
    (TypeError, lambda: nv.layer_norm(x(2, 8, dtype=torch.int32))),
    (TypeError, lambda: nv.layer_norm(x(2, 8, dtype=torch.float64))),
    (ValueError, lambda: nv.layer_norm(x())),
    (ValueError, lambda: nv.layer_norm(x(2, 0))),
    (ValueError, lambda: nv.layer_norm(x(2, 8), eps=-1.0)),
    (ValueError, lambda: nv.layer_norm(x(2, 8), eps=float("nan"))),
    (TypeError, lambda: nv.layer_norm(x(2, 8), out_dtype=F32)),
    (TypeError, lambda: nv.layer_norm(x(2, 8, dtype=F32), out_dtype=F16)),
    (ValueError, lambda: nv.layer_norm(x(2, 8), x(7, dtype=F32))),
    (ValueError, lambda: nv.layer_norm(x(2, 8), x(16, dtype=F32)[::2])),
    (TypeError, lambda: nv.layer_norm(x(2, 8), x(8, dtype=F32), x(8))),
    (ValueError, lambda: nv.layer_norm(x(2, 8))),                                      # a CPU tensor
    (TypeError, lambda: nv.add_layer_norm(x(2, 8), None)),
    (ValueError, lambda: nv.add_layer_norm(x(2, 8), x(3, 8))),
    (ValueError, lambda: nv.add_layer_norm(x(2, 8), x(8))),                           # no broadcasting
    (TypeError, lambda: nv.add_layer_norm(x(2, 8), x(2, 8, dtype=F32))),
    (TypeError, lambda: nv.add_layer_norm(x(2, 8, dtype=F16), x(2, 8))),
])
def test_layer_norm_refusals(error, call):
    with pytest.raises(error):
        call()


Q, POS = x(2, 5, 4, 16), torch.zeros(5, 2, dtype=torch.int64)


@pytest.mark.parametrize("error,call", [
    (ValueError, lambda: nv.rotary_axes(x(5, 4, 16), None, POS, (3, 5))),
    (TypeError, lambda: nv.rotary_axes(Q, x(2, 5, 4, 16, dtype=F32), POS, (3, 5))),
    (ValueError, lambda: nv.rotary_axes(Q, x(2, 5, 4, 8), POS, (3, 5))),
    (ValueError, lambda: nv.rotary_axes(Q, x(2, 6, 4, 16), POS, (3, 5))),
    (ValueError, lambda: nv.rotary_axes(Q, x(2, 5, 0, 16), POS, (3, 5))),
    (ValueError, lambda: nv.rotary_axes(x(2, 5, 0, 16), None, POS, (3, 5))),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, ())),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 0))),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 6))),                         # nine pairs in a head of sixteen features
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 4, 1))),                      # three sections, two axes
    (ValueError, lambda: nv.rotary_axes(x(1, 5, 1, 600), None, POS, (200, 57))),     # above 256 pairs
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 5), layout="pairs")),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 5), frequencies="each")),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 5), theta=0.0)),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 5), theta=float("inf"))),
    (TypeError, lambda: nv.rotary_axes(Q, Q, POS.to(torch.int16), (3, 5))),
    (ValueError, lambda: nv.rotary_axes(Q, Q, torch.zeros(3, 5, 2, dtype=torch.int64), (3, 5))),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS.float().requires_grad_(True), (3, 5))),
    (ValueError, lambda: nv.rotary_axes(Q, Q, POS, (3, 5))),                         # CPU tensors
    (ValueError, lambda: nv.rotary_axes_qkv(x(2, 5, 50), POS, (3, 5), 4)),           # 50 is not 12 heads of anything
    (ValueError, lambda: nv.rotary_axes_qkv(x(2, 5, 4, 48), POS, (3, 5), 4)),
    (ValueError, lambda: nv.rotary_axes_qkv(x(2, 5, 48), POS, (1, 1), 4, 0)),
    (ValueError, lambda: nv.rotary_axes_qkv(x(2, 5, 48), POS, (1, 1), True)),
])
def test_rotary_refusals(error, call):
    with pytest.raises(error):
        call()


def test_entry_points_refuse_before_any_launch():
    from nvfp4_training import _native
    from nvfp4_training.operators import _JOB
    lib = _native.lib()
    buf = C.create_string_buffer(4096)

    def norm(x=buf, xd=1, pitch=8, delta=None, dd=1, eps=1e-5, rows=4, cols=8, total=None, h=buf, hd=1, mean=None, rstd=None):
        return lib.nvfp4_layer_norm(x, xd, pitch, delta, dd, 8, None, None, 0, eps, rows, cols, total, h, hd, mean, rstd, None, None, None)
    assert norm(x=None) == 1 and norm(h=None) == 1 and norm(delta=buf) == 1 and norm(mean=buf) == 1
    assert norm(rows=0) == 1 and norm(cols=0) == 1 and norm(pitch=7) == 1
    assert norm(xd=3) == 3 and norm(hd=0) == 3 and norm(xd=0, hd=2) == 3 and norm(delta=buf, total=buf, dd=2) == 3
    bwd = lambda dd=None, dw=None, part=None, xd=1, hd=1: lib.nvfp4_layer_norm_bwd(buf, hd, 8, buf, xd, 8, buf, buf, None, 0, None, 0, 4, 8, buf, dd,
                                                                                 part, dw, None, None, None, None)
    assert bwd(dw=buf) == 1 and bwd(dd=buf) == 3 and bwd(xd=2, hd=1) == 3
    assert lib.nvfp4_layer_norm_bwd_partials(1, 8) == 1 and lib.nvfp4_layer_norm_bwd_partials(10 ** 9, 8) <= 1024

    turns, axis, strides = (C.c_double * 300)(), (C.c_uint8 * 300)(), (C.c_int64 * 3)()

    def rotary(count=1, dtype=1, dim=16, kind=0, axes=1, pairs=8, heads=2, address=None):
        at = C.addressof(buf) if address is None else address
        tensors = _JOB.pack(at, at, 0, 0, 0, 0, 0, 0, heads, 1) * 4
        return lib.nvfp4_rotary_axes(tensors, count, dtype, 1, 4, dim, buf, kind, strides, axes, turns, axis, pairs, 0, 0, None, None)
    assert rotary(count=0) == 1 and rotary(count=4) == 1 and rotary(dtype=3) == 3 and rotary(kind=4) == 3 and rotary(pairs=9) == 1
    assert rotary(dim=600, pairs=257) == 1 and rotary(heads=0) == 1 and rotary(address=0) == 1
    assert rotary(address=C.addressof(buf) + 1) == 2
    axis[3] = 1
    assert rotary() == 1 and b"axis" in lib.nvfp4_last_error()


W = x(6, 16)


@pytest.mark.parametrize("error,call", [
    (TypeError, lambda: nv.fp8_linear(x(2, 16, dtype=torch.float64), W)),
    (TypeError, lambda: nv.fp8_linear(x(2, 16), W.to(torch.float8_e4m3fn))),
    (TypeError, lambda: nv.fp8_linear(x(2, 16), None)),
    (ValueError, lambda: nv.fp8_linear(x(2, 15), W)),
    (ValueError, lambda: nv.fp8_linear(x(), W)),
    (ValueError, lambda: nv.fp8_linear(x(2, 16), x(16))),
    (ValueError, lambda: nv.fp8_linear(x(2, 0), x(6, 0))),
    (ValueError, lambda: nv.fp8_linear(x(2, 16), x(0, 16))),
    (ValueError, lambda: nv.fp8_linear(x(2, 16), W, x(5))),
    (ValueError, lambda: nv.fp8_linear(x(2, 16), W, x(12)[::2])),
    (TypeError, lambda: nv.fp8_linear(x(2, 16), W, x(6, dtype=torch.int8))),
    (ValueError, lambda: nv.fp8_linear(x(2, 16), W)),                                 # CPU tensors
    (TypeError, lambda: nv.fp8_pack(x(6, 16, dtype=torch.uint8))),
    (ValueError, lambda: nv.fp8_pack(x(6))),
    (ValueError, lambda: nv.fp8_pack(x(6, 0))),
    (ValueError, lambda: nv.fp8_pack(W)),
])
def test_fp8_refusals(error, call):
    with pytest.raises(error):
        call()


def test_packed_weight_without_its_transpose_refuses_input_gradients():
    packed = nv.PackedFP8(torch.cat([torch.zeros(6 * 128, dtype=torch.uint8), torch.full((512,), 127, dtype=torch.uint8)]), None, (6, 16), BF16)
    assert packed.dequantize().shape == (6, 16)
    with pytest.raises(ValueError, match="transpose"):
        nv.fp8_linear(x(2, 16).requires_grad_(True), packed)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        nv.fp8_linear(x(2, 16).requires_grad_(True), packed)


def test_fp8_entry_points_refuse_before_any_launch():
    from nvfp4_training import _native
    lib = _native.lib()
    buf = C.create_string_buffer(4096 + 16)
    at = (C.addressof(buf) + 15) // 16 * 16

    def quantize(x=at, dt=1, rows=4, cols=8, pitch=8, codes=at, scales=at, codes_t=None, scales_t=None, sums=None):
        return lib.nvfp4_fp8_quantize(x, dt, rows, cols, pitch, 0, codes, scales, codes_t, scales_t, sums, None)
    assert quantize(x=None) == 1 and quantize(codes=None, scales=None) == 1 and quantize(scales=None) == 1 and quantize(codes_t=at) == 1
    assert quantize(rows=0) == 1 and quantize(cols=0) == 1 and quantize(pitch=7) == 1 and quantize(sums=at) == 1
    assert quantize(dt=3) == 3 and quantize(codes=at + 1) == 2

    def gemm(a=at, m=4, n=8, k=128, bias=None, bd=0, out=at, od=1, ldo=8):
        return lib.nvfp4_fp8_gemm(a, at, at, at, m, n, k, bias, bd, out, od, ldo, None, None)
    assert gemm(a=None) == 1 and gemm(out=None) == 1 and gemm(m=0) == 1 and gemm(n=0) == 1 and gemm(k=64) == 1 and gemm(ldo=7) == 1
    assert gemm(k=0) == 1 and gemm(m=1 << 30) == 1 and gemm(m=1 << 29, n=1 << 29, ldo=1 << 29) == 1
    assert gemm(od=3) == 3 and gemm(bias=at, bd=4) == 3 and gemm(a=at + 8) == 2 and gemm(out=at + 1) == 2
    from nvfp4_training.fp8 import _packing_bytes
    assert all(lib.nvfp4_fp8_packing_bytes(r, k) == _packing_bytes(r, k) for r in (1, 127, 128, 129) for k in (1, 128, 300))
    linear = lambda x=at, work=at, m=4, wd=1, w_t=None: lib.nvfp4_fp8_linear(x, 1, m, 128, 128, at, wd, 8, 128, None, 0, at, work, None, w_t, None, None)
    assert linear(x=None) == 1 and linear(work=None) == 1 and linear(m=0) == 1 and linear(wd=3, w_t=at) == 1
    back = lambda dx=None, dw=None, x_t=None, w_t=None, m=4: lib.nvfp4_fp8_linear_bwd(at, 1, m, 8, 128, 8, x_t, w_t, dx, dw, 1, None, 0, at, None, None)
    assert back() == 1 and back(dx=at) == 1 and back(dw=at) == 1 and back(dx=at, w_t=at, m=0) == 1
    assert lib.nvfp4_column_sums(at, 0, 8, at, 0, None) == 1 and lib.nvfp4_column_sums(at, 1, 8, at, 3, None) == 3


def test_data_parallel_slots_hold_the_8_bit_weights(tmp_path):
    import torch.distributed as dist
    from nvfp4_training.distributed import GradientReducer
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        nvfp4, fp8, small, dense = (torch.nn.Parameter(torch.zeros(n)) for n in (5000, 4096, 64, 9000))
        nvfp4._v4_request_scale = fp8._v6_defer_dense = small._v6_defer_dense = True
        reducer = GradientReducer([nvfp4, fp8, small, dense])
        assert [reducer.has_slot(p) for p in (nvfp4, fp8, small, dense)] == [True, True, False, False]
        assert reducer.layout()[0] == (5000, 4096)
    finally:
        dist.destroy_process_group()
