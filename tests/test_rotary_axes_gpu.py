"""Rotary positions over several axes against the turn of complex numbers in 64 bits.

Tolerance: each result is a cos - b sin.  sincospi is off by under 2 steps of FP32 and its argument by half a step, an angle
error of at most pi * 2^-25; products and the sum add three roundings: below 2^-21 (|a| + |b|) in all, and half a step of
the stored type.
"""
import pytest
import torch

import nvfp4_training as nv

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def reference(x, positions, sections, layout, frequencies, theta=10000.0, inverse=False):
    x = x.double()
    b, s, h, d = x.shape
    pairs = sum(sections)
    pos = positions.double()
    pos = pos[None].expand(b, s, -1) if pos.ndim == 2 else pos
    angle = torch.zeros(b, s, 1, pairs, dtype=torch.float64, device=x.device)
    j = 0
    for a, n in enumerate(sections):
        for i in range(n):
            angle[:, :, 0, j] = pos[:, :, a] * theta ** -(i / n if frequencies == "axis" else j / pairs)
            j += 1
    unit = torch.polar(torch.ones_like(angle), -angle if inverse else angle)
    if layout == "half":
        z = torch.complex(x[..., :pairs], x[..., pairs:2 * pairs]) * unit
        head = torch.cat([z.real, z.imag], -1)
    else:
        z = torch.complex(x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2]) * unit
        head = torch.stack([z.real, z.imag], -1).flatten(-2)
    return torch.cat([head, x[..., 2 * pairs:]], -1)


def check(got, want, size):
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() * 1.01 + 2.0 ** -21 * 2 * size + (2.0 ** -25 if got.dtype == F16 else 0)
    assert got.shape == want.shape and bool(((got.double() - want).abs() <= bound).all()), ((got.double() - want).abs() - bound).max().item()


def rand(g, *shape, dtype=F32):
    return torch.randn(*shape, device="cuda", generator=g).to(dtype)


def positions(g, b, s, axes, kind=torch.int64, high=5000):
    return torch.randint(-high, high, (b, s, axes), device="cuda", generator=g).to(kind)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("frequencies", ["shared", "axis"])
@pytest.mark.parametrize("dim,sections", [(128, (16, 24, 24)), (64, (32,)), (72, (12, 12, 12)), (80, (10, 10)), (48, (5, 7)), (16, (1,)), (30, (3, 3)), (7, (2, 1)),
                                          (512, (100, 100, 56)), (256, (40, 40))])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_apart_forward_and_backward(layout, frequencies, dim, sections, dtype):
    g = torch.Generator(device="cuda").manual_seed(dim)
    b, s, h, hk = 2, 19, 6, 2
    pos = positions(g, b, s, len(sections))
    q, k = rand(g, b, s, h, dim, dtype=dtype).requires_grad_(True), rand(g, b, s, hk, dim, dtype=dtype).requires_grad_(True)
    how = dict(layout=layout, frequencies=frequencies)
    oq, ok = nv.rotary_axes(q, k, pos, sections, **how)
    for got, x in ((oq, q), (ok, k)):
        check(got, reference(x.detach(), pos, sections, layout, frequencies), 6.0)
        assert torch.equal(got[..., 2 * sum(sections):], x[..., 2 * sum(sections):])
    dq, dk = rand(g, b, h, s, dim, dtype=dtype).transpose(1, 2), rand(g, b, s, hk, dim, dtype=dtype)
    gq, gk = torch.autograd.grad((oq, ok), (q, k), (dq, dk))
    check(gq, reference(dq, pos, sections, layout, frequencies, inverse=True), 6.0)
    check(gk, reference(dk, pos, sections, layout, frequencies, inverse=True), 6.0)


@pytest.mark.parametrize("heads,kv_heads,dim,sections,dtype", [(4, 4, 64, (8, 12, 12), BF16), (5, 1, 72, (4, 30), F16), (3, 2, 48, (5, 7), F32)])
def test_fused_forward_and_backward(heads, kv_heads, dim, sections, dtype):
    from nvfp4_training._backend.quant import known_amax
    g = torch.Generator(device="cuda").manual_seed(dim)
    b, s = 3, 21
    qkv = rand(g, b, s, (heads + 2 * kv_heads) * dim, dtype=dtype).requires_grad_(True)
    pos = positions(g, 1, s, len(sections), torch.int32)[0]
    q, k, v = nv.rotary_axes_qkv(qkv, pos, sections, heads, kv_heads)
    parts = qkv.detach().view(b, s, -1, dim).split((heads, kv_heads, kv_heads), dim=2)
    check(q, reference(parts[0], pos, sections, "half", "shared"), 6.0)
    check(k, reference(parts[1], pos, sections, "half", "shared"), 6.0)
    assert torch.equal(v, parts[2]) and v.data_ptr() == parts[2].data_ptr()
    grads = [rand(g, b, n, s, dim, dtype=dtype).transpose(1, 2) for n in (heads, kv_heads, kv_heads)]
    seen = {}
    qkv.register_hook(lambda t: seen.update(amax=known_amax(t)))
    torch.autograd.backward((q, k, v), grads)
    want = torch.cat([reference(grads[0], pos, sections, "half", "shared", inverse=True), reference(grads[1], pos, sections, "half", "shared", inverse=True),
                      grads[2].double()], dim=2).flatten(2)
    check(qkv.grad, want, 6.0)
    if dtype == BF16:
        assert seen["amax"][0].item() == qkv.grad.abs().max().item()
    # a part that nothing used has a gradient of zeros
    q, k, v = nv.rotary_axes_qkv(qkv, pos, sections, heads, kv_heads)
    got, = torch.autograd.grad((q, v), qkv, (grads[0], grads[2]))
    got = got.view(b, s, -1, dim)
    assert not got[:, :, heads:heads + kv_heads].any() and torch.equal(got[:, :, heads + kv_heads:], grads[2])


@pytest.mark.parametrize("kind", [torch.int64, torch.int32, torch.float32, torch.float64])
def test_positions_of_every_kind_and_far_ones(kind):
    g = torch.Generator(device="cuda").manual_seed(2)
    pos = positions(g, 2, 33, 2, kind, high=2 ** 24)
    if kind in (torch.float32, torch.float64):
        pos = pos / 8                                         # fractional positions (frames per second)
    if kind == torch.int64:
        pos = pos * 2 ** 8 + 1                                # above 2^31
    q = rand(g, 2, 33, 3, 32)
    # 2^32 turns-worth of angle leave 2^-21 of a radian in FP64, below the bound's 2^-20 * 6
    check(nv.rotary_axes(q, None, pos, (8, 8))[0], reference(q, pos, (8, 8), "half", "shared"), 8.0)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_alignment(layout):
    g = torch.Generator(device="cuda").manual_seed(4)
    pos = positions(g, 2, 17, 4)[..., ::2]                     # positions with strides
    base = rand(g, 2 * 17 * 5 * 64 + 8, dtype=BF16)
    views = [rand(g, 2, 5, 17, 64, dtype=BF16).transpose(1, 2), rand(g, 2, 17, 5, 100, dtype=BF16)[..., 30:94], rand(g, 2, 17, 5, 128, dtype=BF16)[..., ::2],
             base[1:1 + 2 * 17 * 5 * 64].view(2, 17, 5, 64), base[4:4 + 2 * 17 * 5 * 64].view(2, 17, 5, 64),
             rand(g, 1, 17, 1, 64, dtype=BF16).expand(2, 17, 5, 64)]
    for x in views:
        check(nv.rotary_axes(x, x, pos, (16, 16), layout=layout)[1], reference(x, pos, (16, 16), layout, "shared"), 6.0)


@pytest.mark.parametrize("batch,seq,heads,kv", [(1, 1, 1, 1), (1, 1, 32, 8), (1, 3, 40, 40), (4, 700, 2, 1), (0, 5, 2, 2), (2, 0, 2, 2)])
def test_lengths_from_nothing_to_many(batch, seq, heads, kv):
    g = torch.Generator(device="cuda").manual_seed(seq)
    pos = positions(g, batch, seq, 3)
    q, k = (rand(g, batch, seq, n, 128, dtype=BF16).requires_grad_(True) for n in (heads, kv))
    oq, ok = nv.rotary_axes(q, k, pos, (16, 24, 24))
    dq, dk = torch.autograd.grad((oq, ok), (q, k), (torch.ones_like(oq), torch.ones_like(ok)))
    assert dq.shape == q.shape and dk.shape == k.shape
    if q.numel():
        check(oq, reference(q.detach(), pos, (16, 24, 24), "half", "shared"), 6.0)
        check(ok, reference(k.detach(), pos, (16, 24, 24), "half", "shared"), 6.0)


def test_back_turns_what_forward_turned():
    g = torch.Generator(device="cuda").manual_seed(9)
    q = rand(g, 2, 50, 4, 64).requires_grad_(True)
    pos = positions(g, 2, 50, 2)
    o, none = nv.rotary_axes(q, None, pos, (10, 22))
    assert none is None
    back, = torch.autograd.grad(o, q, o.detach())
    assert (back - q).abs().max() <= 2.0 ** -18 * q.abs().max()


def test_streams_graphs_and_repeats():
    g = torch.Generator(device="cuda").manual_seed(11)
    qkv = rand(g, 2, 64, 12 * 32, dtype=BF16).requires_grad_(True)
    pos = positions(g, 2, 64, 2)
    dq = rand(g, 2, 64, 4, 32, dtype=BF16)
    keep = nv.rotary_axes_qkv(qkv, pos, (8, 8), 4)
    want = torch.autograd.grad(keep, qkv, (dq, dq, dq), retain_graph=True)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(nv.rotary_axes_qkv(qkv, pos, (8, 8), 4), qkv, (dq, dq, dq))[0]
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    leaf = qkv.detach().clone().requires_grad_(True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = nv.rotary_axes_qkv(leaf, pos, (8, 8), 4)
        grad = torch.autograd.grad(outs, leaf, (dq, dq, dq))[0]
    with torch.no_grad():
        leaf.copy_(-qkv)
        pos.add_(3)
    graph.replay()
    again = nv.rotary_axes_qkv(leaf, pos, (8, 8), 4)
    assert all(torch.equal(a, b) for a, b in zip(outs, again))
    assert torch.equal(grad, torch.autograd.grad(again, leaf, (dq, dq, dq))[0])


def test_in_place_edits_do_not_go_unseen():
    """v is a view of the projection: writing to it either is refused or counts in the gradients."""
    g = torch.Generator(device="cuda").manual_seed(12)
    qkv = rand(g, 1, 6, 12 * 16).requires_grad_(True)
    pos = positions(g, 1, 6, 1)
    q, k, v = nv.rotary_axes_qkv(qkv * 1.0, pos, (8,), 4)
    try:
        v.mul_(2)
    except RuntimeError:
        return
    grad, = torch.autograd.grad(v.sum(), qkv)
    assert torch.equal(grad.view(1, 6, 12, 16)[:, :, 8:], torch.full((1, 6, 4, 16), 2.0, device="cuda"))


def test_edited_positions_are_noticed():
    q = torch.randn(1, 4, 1, 16, device="cuda", requires_grad=True)
    pos = torch.arange(4, device="cuda").view(4, 1)
    out, _ = nv.rotary_axes(q, None, pos, (8,))
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        out.sum().backward()
