"""Operators of an image / video transformer block: layer norm with the residual sum in front of it, and rotary positions over
several axes.  The kernels are nvfp4_layer_norm / nvfp4_layer_norm_bwd and nvfp4_rotary_axes of the C-ABI library; everything
here is differentiable once (in backward mode; forward-mode tangents are refused) and may be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes as C
import math
import struct
from functools import lru_cache

import torch
from torch import nn
from torch.autograd import forward_ad

from . import _native as nat
from ._backend.quant import attach_amax

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _check_tensor(name, t, dtypes=_FLOATS):
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"Unsupported dtype {t.dtype} of {name}")


def _check_device(t):
    """Last of an operator's checks: the arguments fit together, now they also have to be on a GPU."""
    if not t.is_cuda:
        raise ValueError("This operator needs CUDA tensors")


def _autograd_sees(*tensors):
    """Whether a call has to go through its autograd.Function: a gradient may be asked for, or a forward-mode level is open, whose
    tangents only the Function can refuse (a dual tensor has no requires_grad, and a result made without it would count as
    constant)."""
    return forward_ad._current_level >= 0 or (torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors))


def _zeroed_slot(device):
    """float32[4] in the layout of nat.amax for one result; its own zero fill, so that a graph which records it replays it."""
    return torch.zeros(4, dtype=torch.float32, device=device)


# ---- layer norm -------------------------------------------------------------------------------------------------------
def rows_of(t, cols):
    """[rows, cols] view with contiguous rows (any row pitch); a copy only where the layout has no such view."""
    if t.ndim == 2 and t.is_contiguous():
        return t
    flat = t.reshape(-1, cols)
    if (cols > 1 and flat.stride(1) != 1) or (flat.shape[0] > 1 and flat.stride(0) < cols):
        flat = flat.contiguous()
    return flat


def pitch_of(flat):
    return max(flat.stride(0), flat.shape[1])


def _like(t):
    """A new contiguous tensor of t's shape and dtype (empty_like is the cheapest way to one, but copies strides)."""
    return torch.empty_like(t) if t.is_contiguous() else t.new_empty(t.shape)


def _once(impl):
    """torch.autograd.function.once_differentiable, entered only where a second derivative could be asked for: outside
    create_graph=True backward runs without gradients anyway, and the wrapper is host time of every small call."""
    checked = torch.autograd.function.once_differentiable(impl)

    def backward(ctx, *grads):
        return checked(ctx, *grads) if torch.is_grad_enabled() else impl(ctx, *grads)
    return backward


def _norm_forward(x, delta, weight, bias, eps, out_dtype, amax, keep_stats):
    """(total [rows, cols], h, statistics or None): h and a new total in x's shape, total as rows."""
    shape, dev = x.shape, x.device
    cols = shape[-1]
    x2 = rows_of(x, cols)
    rows = x2.shape[0]
    d2, total = None, x2
    if delta is not None:
        d2 = rows_of(delta, cols)
        total = _like(x2)
    h = _like(x) if out_dtype == x.dtype else x.new_empty(shape, dtype=out_dtype)
    stats = x.new_empty(2 * rows, dtype=torch.float32) if keep_stats else None
    if rows:
        at = stats.data_ptr() if keep_stats else None
        affine = weight if weight is not None else bias
        codes = nat._CODES
        with nat.on(dev):
            nat.check(nat.lib().nvfp4_layer_norm(
                x2.data_ptr(), codes[x.dtype], pitch_of(x2), nat.ptr(d2), 0 if d2 is None else codes[d2.dtype], 0 if d2 is None else pitch_of(d2),
                nat.ptr(weight), nat.ptr(bias), 0 if affine is None else codes[affine.dtype], eps, rows, cols,
                None if d2 is None else total.data_ptr(), h.data_ptr(), codes[out_dtype], at, at and at + 4 * rows, nat.ptr(amax),
                nat.status_ptr(dev), nat.raw_stream(dev)))
    return total, h, stats


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, weight, bias, eps, out_dtype, want_amax):
        amax = _zeroed_slot(x.device) if want_amax else None
        total, h, stats = _norm_forward(x, delta, weight, bias, eps, out_dtype, amax, True)
        ctx.save_for_backward(total, stats, weight)
        affine = weight if weight is not None else bias
        ctx.delta_dtype, ctx.shape, ctx.want_amax = None if delta is None else delta.dtype, x.shape, want_amax
        ctx.affine = (weight is not None and ctx.needs_input_grad[2], bias is not None and ctx.needs_input_grad[3],
                      None if affine is None else affine.dtype)
        ctx.set_materialize_grads(False)
        if amax is not None:
            ctx.mark_non_differentiable(amax)
        return (None if delta is None else total if x.ndim == 2 else total.view(x.shape)), h, amax

    @staticmethod
    @_once
    def backward(ctx, dsum, dh, _):
        total, stats, weight = ctx.saved_tensors
        rows, cols = total.shape
        dev = total.device
        need_w, need_b, wdtype = ctx.affine
        if dh is None:       # only the residual path carries a gradient
            dd = None if (dsum is None or ctx.delta_dtype is None) else dsum.to(ctx.delta_dtype)
            zero = torch.zeros(cols, dtype=wdtype, device=dev) if (need_w or need_b) else None
            return dsum, dd, (zero if need_w else None), (zero if need_b else None), None, None, None
        g = rows_of(dh, cols)
        res = None if dsum is None else rows_of(dsum, cols)
        flat = len(ctx.shape) == 2
        dx = _like(total) if flat else total.new_empty(ctx.shape)
        narrow = ctx.delta_dtype is not None and ctx.delta_dtype != total.dtype
        dd = total.new_empty(ctx.shape, dtype=ctx.delta_dtype) if narrow else None
        dw = torch.empty_like(weight) if need_w else None
        db = None if not need_b else torch.empty_like(dw) if need_w else total.new_empty(cols, dtype=wdtype)
        amax = _zeroed_slot(dev) if ctx.want_amax and (narrow or total.dtype == torch.bfloat16) else None
        if rows:
            lib, partial, codes = nat.lib(), None, nat._CODES
            if need_w or need_b:
                partial = stats.new_empty(lib.nvfp4_layer_norm_bwd_partials(rows, cols) * 2 * cols)
            at = stats.data_ptr()
            with nat.on(dev):
                nat.check(lib.nvfp4_layer_norm_bwd(
                    g.data_ptr(), codes[g.dtype], pitch_of(g), total.data_ptr(), codes[total.dtype], pitch_of(total), at, at + 4 * rows,
                    nat.ptr(weight), 0 if wdtype is None else codes[wdtype], nat.ptr(res), 0 if res is None else pitch_of(res), rows, cols,
                    dx.data_ptr(), nat.ptr(dd), nat.ptr(partial), nat.ptr(dw), nat.ptr(db), nat.ptr(amax),
                    nat.status_ptr(dev), nat.raw_stream(dev)))
        else:
            for t in (dw, db):
                if t is not None:
                    t.zero_()
        if not narrow and ctx.delta_dtype is not None:
            dd = dx
        if amax is not None:
            attach_amax(dd if narrow else dx, amax)
        return dx, dd, dw, db, None, None, None


def _layer_norm(x, delta, weight, bias, eps, out_dtype, want_amax=False):
    _check_tensor("x", x)
    if x.ndim == 0 or x.shape[-1] == 0:
        raise ValueError("layer norm needs a last dimension of at least one feature")
    cols = x.shape[-1]
    eps = float(eps)
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError("eps must be finite and not negative")
    out_dtype = x.dtype if out_dtype is None else out_dtype
    if out_dtype != x.dtype and not (x.dtype == torch.float32 and out_dtype == torch.bfloat16):
        raise TypeError("the result has the input's dtype, or BF16 beside an FP32 input")
    if delta is not None:
        _check_tensor("delta", delta)
        if delta.dtype != x.dtype and not (x.dtype == torch.float32 and delta.dtype == torch.bfloat16):
            raise TypeError("delta has the input's dtype, or BF16 beside an FP32 input")
        if delta.shape != x.shape or delta.device != x.device:
            raise ValueError("x and delta must have one shape and device")
    for name, p in (("weight", weight), ("bias", bias)):
        if p is not None:
            _check_tensor(name, p)
            if p.shape != (cols,) or p.device != x.device or not p.is_contiguous():
                raise ValueError(f"{name} must be a contiguous vector of the last dimension's {cols} features on the input's device")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError("weight and bias must have one dtype")
    _check_device(x)
    if not _autograd_sees(x, delta, weight, bias):
        amax = _zeroed_slot(x.device) if want_amax and out_dtype == torch.bfloat16 else None
        total, h, _ = _norm_forward(x, delta, weight, bias, eps, out_dtype, amax, False)
        return (None if delta is None else total if x.ndim == 2 else total.view(x.shape)), h, amax
    return _LayerNorm.apply(x, delta, weight, bias, eps, out_dtype, want_amax and out_dtype == torch.bfloat16)


def layer_norm(x, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension.  x: FP32, BF16 or FP16 with any strides; weight
    and bias (each optional) of one floating dtype.  out_dtype: x's, or torch.bfloat16 beside an FP32 x, which is what an
    NVFP4 or 8-bit layer reads.  Statistics are FP32."""
    return _layer_norm(x, None, weight, bias, eps, out_dtype)[1]


def add_layer_norm(x, delta, weight=None, bias=None, eps=1e-5, *, out_dtype=None):
    """(total, layer_norm(total)) with total = x + delta rounded to x's dtype: the residual sum of a transformer block and
    the norm behind it in one pass.  delta has x's dtype, or BF16 beside an FP32 x (a layer's output under autocast)."""
    if delta is None:
        raise TypeError("delta must be a tensor; use layer_norm without one")
    return _layer_norm(x, delta, weight, bias, eps, out_dtype)[:2]


class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm over the last dimension on this library's kernels (same parameters and state dict).  Under CUDA BF16
    autocast an FP32 input gives a BF16 result, which is what the next converted layer reads; BF16 results carry their amax."""

    def __init__(self, normalized_shape, *args, **options):
        super().__init__(normalized_shape, *args, **options)
        if len(self.normalized_shape) != 1:
            raise ValueError("LayerNorm works over the last dimension alone; nn.LayerNorm takes several")

    def forward(self, x):
        # without affine parameters nothing else holds x against the shape that the module was made for
        if not isinstance(x, torch.Tensor) or x.shape[-1:] != tuple(self.normalized_shape):
            raise ValueError(f"x must have a last dimension of {tuple(self.normalized_shape)}")
        out = torch.bfloat16 if (x.dtype == torch.float32 and torch.is_autocast_enabled("cuda")
                                 and torch.get_autocast_dtype("cuda") == torch.bfloat16) else x.dtype
        _, h, amax = _layer_norm(x, None, self.weight, self.bias, self.eps, out, want_amax=True)
        return h if amax is None else attach_amax(h, amax)


# ---- rotary positions over several axes -----------------------------------------------------------------------------------
_POSITION_KINDS = {torch.int64: 0, torch.int32: 1, torch.float32: 2, torch.float64: 3}
MAX_PAIRS = 256
MAX_TOKEN = 1 << 30        # features of a token's heads, which the kernel counts in 32 bits


_JOB = struct.Struct("=QQqqqqqqii")       # nvfp4_rotary_tensor
_STRIDES = struct.Struct("=qqq")


@lru_cache(maxsize=256)
def _plan(sections, dim, theta, layout, frequencies):
    """Checked once per set of arguments: (host arrays of frequency / (2 pi) and axis of every pair, pairs), axes, interleaved."""
    pairs = sum(sections)
    if 2 * pairs > dim or pairs > MAX_PAIRS:
        raise ValueError(f"sections hold {pairs} pairs; a head of {dim} features has room for {min(dim // 2, MAX_PAIRS)}")
    if layout not in ("half", "interleaved"):
        raise ValueError("layout must be 'half' or 'interleaved'")
    if frequencies not in ("shared", "axis"):
        raise ValueError("frequencies must be 'shared' or 'axis'")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError("theta must be positive and finite")
    turns, axis = (C.c_double * pairs)(), (C.c_uint8 * pairs)()
    j = 0
    for a, n in enumerate(sections):
        for i in range(n):
            turns[j] = theta ** -(i / n if frequencies == "axis" else j / pairs) / (2 * math.pi)
            axis[j] = a
            j += 1
    return (turns, axis, pairs), len(sections), layout == "interleaved"


def _launch_rotary(jobs, positions, plan, axes, interleaved, inverse, amax):
    """jobs: (x, out, turn), each [batch, seq, heads, dim] with contiguous features."""
    x0 = jobs[0][0]
    batch, seq, _, dim = x0.shape
    turns, axis, pairs = plan
    tensors = b"".join([_JOB.pack(x.data_ptr(), out.data_ptr(), *x.stride()[:3], *out.stride()[:3], x.shape[2], turn) for x, out, turn in jobs])
    ps = positions.stride() if positions.ndim == 3 else (0, *positions.stride())
    dev = x0.device
    with nat.on(dev):
        nat.check(nat.lib().nvfp4_rotary_axes(tensors, len(jobs), nat._CODES[x0.dtype], batch, seq, dim, positions.data_ptr(),
                                              _POSITION_KINDS[positions.dtype], _STRIDES.pack(*ps), axes, turns, axis, pairs, interleaved, inverse,
                                              nat.ptr(amax), nat.raw_stream(dev)))


def _features_contiguous(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _turn(tensors, positions, how, inverse):
    """Rotated copies of the tensors that are not None, in one launch."""
    outs = [None if t is None else _like(t) for t in tensors]
    jobs = [(_features_contiguous(t), o, 1) for t, o in zip(tensors, outs) if t is not None and t.numel()]
    if jobs:
        _launch_rotary(jobs, positions, *how, inverse, None)
    return outs


class _RotaryAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, how):
        ctx.save_for_backward(positions)
        ctx.how = how
        ctx.set_materialize_grads(False)
        return tuple(_turn((q, k), positions, how, False))

    @staticmethod
    @_once
    def backward(ctx, dq, dk):
        positions, = ctx.saved_tensors
        return (*_turn((dq, dk), positions, ctx.how, True), None, None)


def _split_heads(t, heads, kv_heads):
    b, s, width = t.shape
    return t.view(b, s, heads + 2 * kv_heads, width // (heads + 2 * kv_heads)).split((heads, kv_heads, kv_heads), dim=2)


class _RotaryFused(torch.autograd.Function):
    """q and k of a fused projection rotated into tensors of their own, v a view of the projection; backward puts the three
    gradients together in one launch."""

    @staticmethod
    def forward(ctx, qkv, positions, how, heads, kv_heads):
        ctx.save_for_backward(positions)
        ctx.how, ctx.dims = how, (qkv.shape, heads, kv_heads)
        ctx.set_materialize_grads(False)
        q, k, v = _split_heads(qkv.detach(), heads, kv_heads)
        return (*_turn((q, k), positions, how, False), v)

    @staticmethod
    @_once
    def backward(ctx, dq, dk, dv):
        positions, = ctx.saved_tensors
        shape, heads, kv_heads = ctx.dims
        some = next(g for g in (dq, dk, dv) if g is not None)
        dqkv = some.new_empty(shape)
        amax = _zeroed_slot(some.device) if some.dtype == torch.bfloat16 else None
        jobs = []
        for g, o, turn in zip((dq, dk, dv), _split_heads(dqkv, heads, kv_heads), (1, 1, 0)):
            if g is None:
                o.zero_()
            else:
                jobs.append((_features_contiguous(g), o, turn))
        if dqkv.numel():
            _launch_rotary(jobs, positions, *ctx.how, True, amax)
        return (dqkv if amax is None else attach_amax(dqkv, amax)), None, None, None, None


def _check_rotary(x, batch, seq, heads, dim, positions, sections, theta, layout, frequencies):
    if heads * dim >= MAX_TOKEN:
        raise ValueError(f"the heads of a token must have fewer than {MAX_TOKEN} features in all")
    sections = tuple(sections)
    if not sections or any(type(n) is not int or n < 1 for n in sections):         # not in _plan: 8.0 and True find the entries of 8 and 1
        raise ValueError("sections must be positive integers: the pairs of a head that each position axis turns")
    how = _plan(sections, dim, float(theta), layout, frequencies)
    _check_tensor("positions", positions, _POSITION_KINDS)
    shape = positions.shape
    if positions.requires_grad:
        raise ValueError("positions have no gradient here; pass them detached")
    if positions.device != x.device or shape[-2:] != (seq, how[1]) or not (len(shape) == 2 or (len(shape) == 3 and shape[0] == batch)):
        raise ValueError(f"positions must be [{seq}, {how[1]}] or [{batch}, {seq}, {how[1]}] on the input's device")
    _check_device(x)
    return how


def rotary_axes(q, k, positions, sections, *, theta=10000.0, layout="half", frequencies="shared"):
    """(q, k) turned by rotary positions over several axes; k may be None.  q [batch, seq, heads, dim], k [batch, seq,
    kv_heads, dim] of one dtype (FP32, BF16, FP16) with any strides; positions [seq, axes] or [batch, seq, axes], int32,
    int64, FP32 or FP64; sections: pairs turned by each axis, in order, at most dim / 2 in all (features behind the turned
    ones pass unchanged).  frequencies 'shared': pair j of all P turns by theta^(-j / P), whatever its axis; 'axis': pair i
    of an axis of n pairs by theta^(-i / n).  layout 'half': pair j is features (j, j + P); 'interleaved': (2j, 2j + 1).
    Angles are FP64: off by about |position * frequency| * 2^-52 radians before sines and cosines are formed in FP32."""
    _check_tensor("q", q)
    if q.ndim != 4:
        raise ValueError("q must be [batch, seq, heads, dim]")
    if k is not None:
        _check_tensor("k", k)
        if k.dtype != q.dtype:
            raise TypeError("q and k must have one dtype")
        if k.ndim != 4 or k.device != q.device or k.shape[:2] != q.shape[:2] or k.shape[3] != q.shape[3]:
            raise ValueError("k must be [batch, seq, kv_heads, dim] beside q")
        if k.shape[2] == 0:
            raise ValueError("k needs at least one head")
    if q.shape[2] == 0:
        raise ValueError("q needs at least one head")
    how = _check_rotary(q, q.shape[0], q.shape[1], q.shape[2] + (0 if k is None else k.shape[2]), q.shape[3], positions, sections, theta, layout, frequencies)
    if not _autograd_sees(q, k):
        return tuple(_turn((q, k), positions, how, False))
    return _RotaryAxes.apply(q, k, positions, how)


def rotary_axes_qkv(qkv, positions, sections, heads, kv_heads=None, *, theta=10000.0, layout="half", frequencies="shared"):
    """(q, k, v) of a fused projection qkv [batch, seq, (heads + 2 * kv_heads) * dim], q and k turned as by rotary_axes, v a
    view of qkv.  The gradient of qkv is written in one pass over those of q, k and v."""
    _check_tensor("qkv", qkv)
    kv_heads = heads if kv_heads is None else kv_heads
    if type(heads) is not int or type(kv_heads) is not int or heads < 1 or kv_heads < 1:
        raise ValueError("heads and kv_heads must be positive integers")
    if qkv.ndim != 3 or qkv.shape[2] == 0 or qkv.shape[2] % (heads + 2 * kv_heads):
        raise ValueError("qkv must be [batch, seq, (heads + 2 * kv_heads) * dim]")
    dim = qkv.shape[2] // (heads + 2 * kv_heads)
    how = _check_rotary(qkv, qkv.shape[0], qkv.shape[1], heads + 2 * kv_heads, dim, positions, sections, theta, layout, frequencies)
    qkv = _features_contiguous(qkv)
    if not _autograd_sees(qkv):
        q, k, v = _split_heads(qkv, heads, kv_heads)
        return (*_turn((q, k), positions, how, False), v)
    return _RotaryFused.apply(qkv, positions, how, heads, kv_heads)
