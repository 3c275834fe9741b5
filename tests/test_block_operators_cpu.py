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
    from nvfp4_training.operators import _Tensor
    lib = _native.lib()
    buf = C.create_string_buffer(4096)

    def norm(x=buf, xd=1, pitch=8, delta=None, dd=1, eps=1e-5, rows=4, cols=8, total=None, h=buf, hd=1, mean=None, rstd=None):
        return lib.nvfp4_layer_norm(x, xd, pitch, delta, dd, 8, None, None, 0, eps, rows, cols, total, h, hd, mean, rstd, None, None)
    assert norm(x=None) == 1 and norm(h=None) == 1 and norm(delta=buf) == 1 and norm(mean=buf) == 1
    assert norm(rows=0) == 1 and norm(cols=0) == 1 and norm(pitch=7) == 1
    assert norm(xd=3) == 3 and norm(hd=0) == 3 and norm(xd=0, hd=2) == 3 and norm(delta=buf, total=buf, dd=2) == 3
    bwd = lambda dd=None, dw=None, part=None, xd=1, hd=1: lib.nvfp4_layer_norm_bwd(buf, hd, 8, buf, xd, 8, buf, buf, None, 0, None, 0, 4, 8, buf, dd,
                                                                                 part, dw, None, None, None)
    assert bwd(dw=buf) == 1 and bwd(dd=buf) == 3 and bwd(xd=2, hd=1) == 3
    assert lib.nvfp4_layer_norm_bwd_partials(1, 8) == 1 and lib.nvfp4_layer_norm_bwd_partials(10 ** 9, 8) <= 1024

    tensors = (_Tensor * 1)()
    turns, axis, strides = (C.c_double * 300)(), (C.c_uint8 * 300)(), (C.c_int64 * 3)()

    def rotary(count=1, dtype=1, dim=16, kind=0, axes=1, pairs=8, heads=2, address=None):
        tensors[0].x = tensors[0].out = C.addressof(buf) if address is None else address
        tensors[0].heads, tensors[0].turn = heads, 1
        return lib.nvfp4_rotary_axes(tensors, count, dtype, 1, 4, dim, buf, kind, strides, axes, turns, axis, pairs, 0, 0, None, None)
    assert rotary(count=0) == 1 and rotary(count=4) == 1 and rotary(dtype=3) == 3 and rotary(kind=4) == 3 and rotary(pairs=9) == 1
    assert rotary(dim=600, pairs=257) == 1 and rotary(heads=0) == 1 and rotary(address=0) == 1
    assert rotary(address=C.addressof(buf) + 1) == 2
    axis[3] = 1
    assert rotary() == 1 and b"axis" in lib.nvfp4_last_error()
