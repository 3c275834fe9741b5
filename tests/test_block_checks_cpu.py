"""Calls of the transformer-block operators that need no GPU to be seen: the kernels are replaced by formulas here, so that what
the public functions hand to autograd, to the optimizer and to other ranks can be held against what they should."""
import pytest
import torch
from torch.autograd import forward_ad

import nvfp4_training as nv
from nvfp4_training import fp8, operators

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture
def without_kernels(monkeypatch):
    """The operators' host side on CPU tensors, with results that depend on nothing but shapes."""
    for module in (operators, fp8):
        monkeypatch.setattr(module, "_check_device", lambda t: None)

    def norm(x, delta, weight, bias, eps, out_dtype, amax, keep_stats):
        rows = x.reshape(-1, x.shape[-1])
        return rows if delta is None else rows * 1, x.to(out_dtype) * 1, torch.zeros(2 * len(rows)) if keep_stats else None
    monkeypatch.setattr(operators, "_norm_forward", norm)
    monkeypatch.setattr(operators, "_turn", lambda tensors, positions, how, inverse: [None if t is None else t * 1 for t in tensors])
    monkeypatch.setattr(fp8, "_forward", lambda x, weight, bias, packed, need_x, need_w: (x.new_zeros(*x.shape[:-1], weight.shape[0]), None, None))


T, W, POS = torch.ones(2, 3, 12), torch.ones(12), torch.zeros(3, 1, dtype=torch.float64)
Q = torch.ones(2, 3, 4, 4)
CALLS = {
    "layer_norm x": (lambda t: nv.layer_norm(t, W), T),
    "layer_norm weight": (lambda t: nv.layer_norm(T, t), W),
    "layer_norm bias": (lambda t: nv.layer_norm(T, None, t), W),
    "add_layer_norm x": (lambda t: nv.add_layer_norm(t, T), T),
    "add_layer_norm delta": (lambda t: nv.add_layer_norm(T, t), T),
    "LayerNorm": (lambda t: nv.LayerNorm(12)(t), T),
    "rotary_axes q": (lambda t: nv.rotary_axes(t, Q, POS, (2,)), Q),
    "rotary_axes k": (lambda t: nv.rotary_axes(Q, t, POS, (2,)), Q),
    "rotary_axes positions": (lambda t: nv.rotary_axes(Q, None, t, (2,)), POS),
    "rotary_axes_qkv": (lambda t: nv.rotary_axes_qkv(t, POS, (2,), 1), T),
    "fp8_linear x": (lambda t: nv.fp8_linear(t, torch.ones(5, 12)), T),
    "fp8_linear weight": (lambda t: nv.fp8_linear(T, t), torch.ones(5, 12)),
    "fp8_linear bias": (lambda t: nv.fp8_linear(T, torch.ones(5, 12), t), torch.ones(5)),
}


@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name", CALLS)
def test_forward_mode_tangents_are_refused(without_kernels, name, grad):
    """A tangent that an operator cannot carry on is an error, never a result that passes for constant."""
    call, at = CALLS[name]
    with torch.set_grad_enabled(grad):
        call(at)                                                   # no level is open
        with forward_ad.dual_level():
            call(at)                                               # no tangent
            with pytest.raises(NotImplementedError):
                call(forward_ad.make_dual(at, torch.ones_like(at)))


@pytest.mark.parametrize("affine", [True, False])
def test_layer_norm_module_holds_its_shape(without_kernels, affine):
    make = lambda shape: nv.LayerNorm(shape, elementwise_affine=affine)
    assert make(8)(torch.ones(2, 8)).shape == (2, 8) and make((8,))(torch.ones(8)).shape == (8,)
    for x in (torch.ones(2, 16), torch.ones(8, 2), torch.ones(()), torch.ones(2, 0)):
        with pytest.raises(ValueError):
            make(8)(x)
    for shape in ((3, 16), ()):
        with pytest.raises(ValueError):
            make(shape)
    swapped = torch.nn.LayerNorm((3, 16), elementwise_affine=affine)          # a module made by nn.LayerNorm, then given this class
    swapped.__class__ = nv.LayerNorm
    with pytest.raises(ValueError):
        swapped(torch.ones(3, 16))


def test_sections_are_integers_also_after_a_call_that_they_equal(without_kernels):
    q, pos = torch.ones(1, 3, 2, 16), torch.zeros(3, 1)
    nv.rotary_axes(q, None, pos, (8,))
    nv.rotary_axes(q, None, pos, (1,))
    for sections in ((8.0,), (True,), (torch.tensor(8),)):
        with pytest.raises(ValueError):
            nv.rotary_axes(q, None, pos, sections)


def test_rotary_refuses_tokens_beyond_its_counters(without_kernels):
    """The kernel counts the features of a token's heads in 32 bits."""
    one, pos = torch.ones(1), torch.zeros(1, 1)
    heads = lambda h, d: one.expand(1, 1, h, d)
    for q, k in ((heads(1 << 20, 1 << 10), None), (heads(1 << 19, 1 << 10), heads(1 << 19, 1 << 10)), (heads(1, 1 << 30), None), (heads(1 << 31, 2), None)):
        with pytest.raises(ValueError, match="features"):
            nv.rotary_axes(q, k, pos, (1,))
    with pytest.raises(ValueError, match="features"):
        nv.rotary_axes_qkv(one.expand(1, 1, 3 << 29), pos, (1,), 1)


def test_rotary_entry_point_refuses_tokens_beyond_its_counters():
    import ctypes as C
    from nvfp4_training import _native
    lib = _native.lib()
    buf = C.create_string_buffer(64)
    at = (C.addressof(buf) + 15) // 16 * 16
    turns, axis, strides = (C.c_double * 1)(), (C.c_uint8 * 1)(), (C.c_int64 * 3)()
    for count, heads, dim in ((1, 1 << 19, 1 << 11), (3, 1 << 19, 1 << 10), (3, (1 << 20) - 1, (1 << 31) - 2)):
        tensors = operators._JOB.pack(at, at, 0, 0, 0, 0, 0, 0, heads, 1) * count
        assert lib.nvfp4_rotary_axes(tensors, count, 1, 1, 1, dim, buf, 0, strides, 1, turns, axis, 1, 0, 0, None, None) == 1
        assert b"features" in lib.nvfp4_last_error()


@pytest.mark.parametrize("cols", [1, 64, 768, 1027, 2048, 4096, 5120, 8192, 8200, 16400, 131072, 1 << 20, (1 << 30) - 1])
@pytest.mark.parametrize("rows", [1, 40, 1024, 16384, 10 ** 7])
def test_layer_norm_scratch_is_what_the_width_uses(cols, rows):
    """Partial sums of the parameters' gradients: one row at least, never more than the rows there are, and 16 MB or one row of them."""
    from nvfp4_training import _native
    parts = _native.lib().nvfp4_layer_norm_bwd_partials(rows, cols)
    assert 1 <= parts <= rows and parts * 2 * cols * 4 <= max(16 << 20, 8 * cols)
