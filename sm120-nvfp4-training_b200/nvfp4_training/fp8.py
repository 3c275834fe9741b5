"""Linear layers in 8-bit floating point: e4m3 operands, one power-of-two scale for each block of 128.

  y  = Q(x) Q(W)^T (+ b)      x in blocks of 1 x 128 along the features, W in blocks of 128 x 128
  dx = Q(dy) Q(W)             dy in blocks of 1 x 128 along the outputs; the weight's blocks are the same in both directions
  dW = Q'(dy)^T Q'(x)         both in blocks of 128 along the tokens;  db = sum of dy

For the layers of an NVFP4 model that do not bear 4 bits (enable_nvfp4(..., fp8_layers=...)), or on their own.  A weight that
does not change is packed once (fp8_pack).  The kernels are nvfp4_fp8_quantize and nvfp4_fp8_gemm of the C-ABI library.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch
from torch import nn

from . import _native as nat
from .operators import _autograd_sees, _check_device, _check_tensor, _once, pitch_of, rows_of

_MAX = 1 << 30


def _ceil128(n):
    return (n + 127) // 128


def _packing_bytes(rows, k):
    """Codes [rows, k padded to 128] and their 512-byte scale blocks, as nvfp4_fp8_packing_bytes counts them."""
    blocks = (k + 127) >> 7
    return rows * blocks * 128 + ((rows + 127) >> 7) * blocks * 512


@dataclass(frozen=True)
class PackedFP8:
    """A weight [rows, cols] laid out for the products: uint8 codes [rows, cols padded to 128] followed by their scale blocks,
    and the same of its transpose (None without it: then no gradient reaches the layer's input)."""
    packing: torch.Tensor
    packing_t: Optional[torch.Tensor]
    shape: tuple
    dtype: torch.dtype

    @property
    def device(self):
        return self.packing.device

    def dequantize(self):
        """FP32 [rows, cols]: the numbers the codes stand for."""
        rows, cols = self.shape
        rb, cb = _ceil128(rows), _ceil128(cols)
        codes = self.packing[:rows * cb * 128].view(rows, cb * 128)
        e = self.packing[rows * cb * 128:].view(rb, cb, 512)[:, :, 0].int() - 127
        scale = ((e.long() + 1023) << 52).view(torch.float64).repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)      # 2^e
        return (codes.view(torch.float8_e4m3fn).double() * scale)[:, :cols].float()


def _bytes(n, beside):
    return beside.new_empty(n, dtype=torch.uint8)


def _quantize(x, *, row, col, square=False, column_sums=False):
    """(packing or None, transposed packing or None, FP32 partial column sums or None) of x [rows, cols]."""
    rows, cols = x.shape
    dev = x.device
    a = _bytes(_packing_bytes(rows, cols), x) if row else None
    t = _bytes(_packing_bytes(cols, rows), x) if col else None
    sums = torch.empty((_ceil128(rows), cols), dtype=torch.float32, device=dev) if column_sums else None
    at, tt = nat.ptr(a), nat.ptr(t)
    with nat.on(dev):
        nat.check(nat.lib().nvfp4_fp8_quantize(x.data_ptr(), nat._CODES[x.dtype], rows, cols, pitch_of(x), square, at,
                                               at and at + rows * _ceil128(cols) * 128, tt, tt and tt + cols * _ceil128(rows) * 128,
                                               nat.ptr(sums), nat.raw_stream(dev)))
    return a, t, sums


def _forward(x, weight, bias, packed, need_x, need_w):
    """(y, transposed packing of x or None, that of the weight or None)."""
    dev, codes = x.device, nat._CODES
    if weight is None:
        n, k = packed.shape
        w, w_code, w_pitch, w_t, w_bytes = packed.packing, nat.E4M3, 0, None, 0
    else:
        n, k = weight.shape
        w = rows_of(weight, k)
        w_code, w_pitch, w_bytes = codes[w.dtype], pitch_of(w), _packing_bytes(n, k)
        w_t = _bytes(_packing_bytes(k, n), x) if need_x else None
    x2 = rows_of(x, k)
    m = x2.shape[0]
    y = x.new_empty((m, n) if x.ndim == 2 else (*x.shape[:-1], n))
    x_t = _bytes(_packing_bytes(k, m), x) if need_w else None
    if m:
        work = _bytes(_packing_bytes(m, k) + w_bytes, x)
        with nat.on(dev):
            nat.check(nat.lib().nvfp4_fp8_linear(x2.data_ptr(), codes[x.dtype], m, k, pitch_of(x2), w.data_ptr(), w_code, n, w_pitch, nat.ptr(bias),
                                                 0 if bias is None else codes[bias.dtype], y.data_ptr(), work.data_ptr(), nat.ptr(x_t), nat.ptr(w_t),
                                                 nat.status_ptr(dev), nat.raw_stream(dev)))
    return y, x_t, (packed.packing_t if weight is None else w_t)


class _Fp8Linear(torch.autograd.Function):
    """weight: the parameter [N, K], packed on every call, or None beside a packed one."""

    @staticmethod
    def forward(ctx, x, weight, bias, packed):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        y, x_t, w_t = _forward(x, weight, bias, packed, need_x, need_w)
        n, k = packed.shape if weight is None else weight.shape
        ctx.how = (x.numel() // k, n, k, need_x, need_w, None if not need_b else bias.dtype, x.shape, x.dtype)
        ctx.save_for_backward(weight, w_t if need_x else None, x_t)
        return y

    @staticmethod
    @_once
    def backward(ctx, grad):
        m, n, k, need_x, need_w, b_dtype, shape, dtype = ctx.how
        weight, w_t, x_t = ctx.saved_tensors
        dev = grad.device
        dx = grad.new_empty(shape, dtype=dtype) if need_x else None
        db = None if b_dtype is None else grad.new_empty(n, dtype=b_dtype)
        dw, taken = _weight_gradient_into(weight) if need_w else (None, None)
        if m:
            columns = need_w or db is not None
            work = _bytes((_packing_bytes(m, n) if need_x else 0) + (_packing_bytes(n, m) + 4 * n * _ceil128(m) if columns else 0), grad)
            g = rows_of(grad, n)
            codes = nat._CODES
            with nat.on(dev):
                nat.check(nat.lib().nvfp4_fp8_linear_bwd(g.data_ptr(), codes[g.dtype], m, n, k, pitch_of(g), nat.ptr(x_t), nat.ptr(w_t), nat.ptr(dx),
                                                         nat.ptr(dw), 0 if dw is None else codes[dw.dtype], nat.ptr(db), 0 if db is None else codes[b_dtype],
                                                         work.data_ptr(), nat.status_ptr(dev), nat.raw_stream(dev)))
        else:                # no rows: zeros, handed on like any other gradient (the other ranks' collectives count on it)
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        if taken is not None:
            taken(dw)
            dw = None
        return dx, dw, db, None


def _weight_gradient_into(weight):
    """(tensor that receives dW, None), or with a function that hands it on where an optimizer collects gradients itself
    (backward_step, captured steps) instead of autograd."""
    new = lambda dtype: torch.empty_like(weight, dtype=dtype, memory_format=torch.contiguous_format)
    sink = getattr(weight, "_v4_pending", None)
    if sink is None or weight.numel() < 4096:          # smaller weights have FP32 moments and take an ordinary gradient
        return new(weight.dtype), None
    reducer = getattr(weight, "_dp_reducer", None)
    if reducer is not None:
        if weight in sink:             # applied again: the slot is on its way to the other ranks, and this part goes to autograd
            return new(weight.dtype), None
        slot = reducer.slot(weight)

        def reduce(_):
            sink[weight] = (slot, None, None)
            reducer.ready(weight)
        return slot.view(weight.shape), reduce

    # FP32 for FP32 masters.  For 16-bit ones BF16, FP16 masters included: the update reads either, 2^-9 of a gradient is far below
    # the noise of its e4m3 operands, and FP16 would lose what is smaller than 6e-8.
    def keep(dw):                                       # a layer applied twice: the sum stays in FP32
        sink[weight] = (dw.add_(sink[weight][0]) if weight in sink else dw, None, None)
    return new(torch.float32 if weight in sink or weight.dtype == torch.float32 else torch.bfloat16), keep


def fp8_pack(weight, *, transpose=True):
    """Lay out a weight [out_features, in_features] (FP32, BF16 or FP16) once, for calls in which it does not change.
    transpose=False leaves out the copy that the gradient of the layer's input needs."""
    _check_tensor("weight", weight)
    if weight.ndim != 2 or 0 in weight.shape or max(weight.shape) >= _MAX:
        raise ValueError("weight must be [out_features, in_features], not empty")
    _check_device(weight)
    q, t, _ = _quantize(rows_of(weight.detach(), weight.shape[1]), row=True, col=transpose, square=True)
    return PackedFP8(q, t, tuple(weight.shape), weight.dtype)


def fp8_linear(x, weight, bias=None):
    """x W^T (+ bias) with both operands in e4m3 under power-of-two scales of blocks of 128, FP32 accumulation, one rounding
    to x's dtype.  x [..., in_features]: FP32, BF16 or FP16 with any strides; weight [out_features, in_features] of any of the
    three (quantised on every call), or what fp8_pack returned; bias [out_features].  Differentiable once in x, weight and
    bias; a packed weight has no gradient.  A value that is not finite makes every product with its block NaN."""
    _check_tensor("x", x)
    packed = weight if isinstance(weight, PackedFP8) else None
    if packed is None:
        _check_tensor("weight", weight)
        if weight.ndim != 2 or 0 in weight.shape or max(weight.shape) >= _MAX:
            raise ValueError("weight must be [out_features, in_features], not empty")
    if x.ndim == 0 or x.shape[-1] != weight.shape[1] or weight.device != x.device:
        raise ValueError(f"x must be [..., {weight.shape[1]}] on the weight's device")
    if x.numel() // weight.shape[1] >= _MAX:
        raise ValueError("too many rows for one call")
    if bias is not None:
        _check_tensor("bias", bias)
        if bias.shape != (weight.shape[0],) or bias.device != x.device or not bias.is_contiguous():
            raise ValueError(f"bias must be a contiguous vector of {weight.shape[0]} features on the input's device")
    if packed is not None and packed.packing_t is None and x.requires_grad and torch.is_grad_enabled():
        raise ValueError("This weight was packed without its transpose: no gradient can reach x")
    _check_device(x)
    if packed is not None:
        weight = None
    if not _autograd_sees(x, weight, bias):
        return _forward(x, weight, bias, packed, False, False)[0]
    return _Fp8Linear.apply(x, weight, bias, packed)


class FP8Linear(nn.Linear):
    """nn.Linear whose three products run in e4m3 (same parameters and state dict).  Under CUDA BF16 autocast the input is
    taken as BF16, as the NVFP4 layers do."""

    def forward(self, input):
        if input.dtype != torch.bfloat16 and torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
            input = input.to(torch.bfloat16)
        return fp8_linear(input, self.weight, self.bias)
