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
from .operators import _check_device, _check_tensor, pitch_of, rows_of

_MAX = 1 << 30


def _ceil128(n):
    return (n + 127) // 128


@dataclass(frozen=True)
class PackedFP8:
    """A weight [rows, cols] laid out for the products: codes uint8 [rows, cols padded to 128], its scale blocks, and the same
    of its transpose (None without it: then no gradient reaches the layer's input)."""
    codes: torch.Tensor
    scales: torch.Tensor
    codes_t: Optional[torch.Tensor]
    scales_t: Optional[torch.Tensor]
    shape: tuple
    dtype: torch.dtype

    @property
    def device(self):
        return self.codes.device

    def dequantize(self):
        """FP32 [rows, cols]: the numbers the codes stand for."""
        rows, cols = self.shape
        e = self.scales.view(_ceil128(rows), _ceil128(cols), 512)[:, :, 0].int() - 127
        scale = ((e.long() + 1023) << 52).view(torch.float64).repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)      # 2^e
        return (self.codes.view(torch.float8_e4m3fn).double() * scale)[:, :cols].float()


def _quantize(x, *, row, col, square=False, column_sums=False):
    """((codes, scales) or None, (codes_t, scales_t) or None, FP32 partial column sums or None) of x [rows, cols]."""
    rows, cols = x.shape
    rb, cb = _ceil128(rows), _ceil128(cols)
    dev = x.device
    a, t, sums = (None, None), (None, None), None
    if row:
        a = (torch.empty((rows, cb * 128), dtype=torch.uint8, device=dev), torch.empty(rb * cb * 512, dtype=torch.uint8, device=dev))
    if col:
        t = (torch.empty((cols, rb * 128), dtype=torch.uint8, device=dev), torch.empty(cb * rb * 512, dtype=torch.uint8, device=dev))
    if column_sums:
        sums = torch.empty((rb, cols), dtype=torch.float32, device=dev)
    with nat.on(dev):
        nat.check(nat.lib().nvfp4_fp8_quantize(x.data_ptr(), nat._CODES[x.dtype], rows, cols, pitch_of(x), square, nat.ptr(a[0]), nat.ptr(a[1]),
                                               nat.ptr(t[0]), nat.ptr(t[1]), nat.ptr(sums), nat.raw_stream(dev)))
    return (a if row else None), (t if col else None), sums


def _gemm(a, b, k, dtype, bias=None, out=None):
    """a, b: (codes, scales) of [M, k] and [N, k]."""
    m, n = a[0].shape[0], b[0].shape[0]
    dev = a[0].device
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=dev)
    with nat.on(dev):
        nat.check(nat.lib().nvfp4_fp8_gemm(a[0].data_ptr(), a[1].data_ptr(), b[0].data_ptr(), b[1].data_ptr(), m, n, _ceil128(k) * 128, nat.ptr(bias),
                                           0 if bias is None else nat._CODES[bias.dtype], out.data_ptr(), nat._CODES[out.dtype], out.stride(0),
                                           nat.status_word(dev).data_ptr(), nat.raw_stream(dev)))
    return out


def _column_sums(partial, dtype):
    out = torch.empty(partial.shape[1], dtype=dtype, device=partial.device)
    with nat.on(out.device):
        nat.check(nat.lib().nvfp4_column_sums(partial.data_ptr(), partial.shape[0], partial.shape[1], out.data_ptr(), nat._CODES[dtype],
                                              nat.raw_stream(out.device)))
    return out


def _inference(x, weight, bias, packed):
    n, k = packed.shape if weight is None else weight.shape
    x2 = rows_of(x, k)
    if not x2.shape[0]:
        return torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
    wq = (packed.codes, packed.scales) if weight is None else _quantize(rows_of(weight, k), row=True, col=False, square=True)[0]
    y = _gemm(_quantize(x2, row=True, col=False)[0], wq, k, x.dtype, bias)
    return y if x.ndim == 2 else y.view(*x.shape[:-1], n)


class _Fp8Linear(torch.autograd.Function):
    """weight: the parameter [N, K], packed on every call, or None beside a packed one."""

    @staticmethod
    def forward(ctx, x, weight, bias, packed):
        need_x, need_w, need_b = ctx.needs_input_grad[:3]
        n, k = packed.shape if weight is None else weight.shape
        x2 = rows_of(x, k)
        m = x2.shape[0]
        ctx.dims, ctx.need, ctx.shape, ctx.dtype = (m, k, n), (need_x, need_w, need_b), x.shape, x.dtype
        ctx.bias_dtype, ctx.weight_dtype = None if bias is None else bias.dtype, None if weight is None else weight.dtype
        if m == 0:
            ctx.save_for_backward(weight)
            return torch.empty((*x.shape[:-1], n), dtype=x.dtype, device=x.device)
        xq, xt, _ = _quantize(x2, row=True, col=need_w)
        if weight is None:
            wq, wt = (packed.codes, packed.scales), (packed.codes_t, packed.scales_t)
        else:
            wq, wt, _ = _quantize(rows_of(weight.detach(), k), row=True, col=need_x, square=True)
        y = _gemm(xq, wq, k, x.dtype, bias)
        ctx.save_for_backward(weight, *(wt if need_x else (None, None)), *(xt if need_w else (None, None)))
        return y.view(*x.shape[:-1], n)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        m, k, n = ctx.dims
        need_x, need_w, need_b = ctx.need
        weight = ctx.saved_tensors[0]
        if m == 0:
            zero = lambda yes, shape, dtype: torch.zeros(shape, dtype=dtype, device=grad.device) if yes else None
            return zero(need_x, ctx.shape, ctx.dtype), zero(need_w, (n, k), ctx.weight_dtype), zero(need_b, (n,), ctx.bias_dtype), None
        _, wt_codes, wt_scales, xt_codes, xt_scales = ctx.saved_tensors
        dx = dw = db = None
        gq, gt, sums = _quantize(rows_of(grad, n), row=need_x, col=need_w or need_b, column_sums=need_b)
        if need_x:
            dx = _gemm(gq, (wt_codes, wt_scales), n, ctx.dtype).view(ctx.shape)
        if need_w:
            dw = _weight_gradient(weight, gt, (xt_codes, xt_scales), m)
        if need_b:
            db = _column_sums(sums, ctx.bias_dtype)
        return dx, dw, db, None


def _weight_gradient(weight, gt, xt, tokens):
    """dW, or None where an optimizer that collects gradients itself (backward_step, captured steps) has taken it."""
    sink = getattr(weight, "_v4_pending", None)
    if sink is None or weight.numel() < 4096:          # smaller weights have FP32 moments and take an ordinary gradient
        return _gemm(gt, xt, tokens, weight.dtype)
    reducer = getattr(weight, "_dp_reducer", None)
    if reducer is not None:
        if weight in sink:
            raise RuntimeError("An 8-bit layer may be applied only once per step under data parallel")
        slot = reducer.slot(weight)
        _gemm(gt, xt, tokens, slot.dtype, out=slot.view(weight.shape))
        sink[weight] = (slot, None, None)
        reducer.ready(weight)
    elif weight in sink:                                # a layer applied twice: the sum stays in FP32
        sink[weight] = (_gemm(gt, xt, tokens, torch.float32).add_(sink[weight][0]), None, None)
    else:
        sink[weight] = (_gemm(gt, xt, tokens, torch.float32 if weight.dtype == torch.float32 else torch.bfloat16), None, None)
    return None


def fp8_pack(weight, *, transpose=True):
    """Lay out a weight [out_features, in_features] (FP32, BF16 or FP16) once, for calls in which it does not change.
    transpose=False leaves out the copy that the gradient of the layer's input needs."""
    _check_tensor("weight", weight)
    if weight.ndim != 2 or 0 in weight.shape or max(weight.shape) >= _MAX:
        raise ValueError("weight must be [out_features, in_features], not empty")
    _check_device(weight)
    w = rows_of(weight.detach(), weight.shape[1])
    q, t, _ = _quantize(w, row=True, col=transpose, square=True)
    return PackedFP8(*q, *(t if transpose else (None, None)), tuple(weight.shape), weight.dtype)


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
    if packed is not None and packed.codes_t is None and x.requires_grad and torch.is_grad_enabled():
        raise ValueError("This weight was packed without its transpose: no gradient can reach x")
    _check_device(x)
    if packed is not None:
        weight = None
    if not (torch.is_grad_enabled() and (x.requires_grad or any(t is not None and t.requires_grad for t in (weight, bias)))):
        return _inference(x, weight, bias, packed)
    return _Fp8Linear.apply(x, weight, bias, packed)


class FP8Linear(nn.Linear):
    """nn.Linear whose three products run in e4m3 (same parameters and state dict).  Under CUDA BF16 autocast the input is
    taken as BF16, as the NVFP4 layers do."""

    def forward(self, input):
        if input.dtype != torch.bfloat16 and torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") == torch.bfloat16:
            input = input.to(torch.bfloat16)
        return fp8_linear(input, self.weight, self.bias)
