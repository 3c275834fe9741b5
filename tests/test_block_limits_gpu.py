"""The transformer-block operators at the ends of what they allow: tensors of more than 2^31 elements (only the last rows hold
values, and only they are compared), the first call of a process inside a graph capture, and calls on several streams at once."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import nvfp4_training as nv

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16
LAST = 5


def tail_filled(rows, cols, g):
    x = torch.zeros(rows, cols, dtype=BF16, device="cuda")
    x[-LAST:] = torch.randn(LAST, cols, device="cuda", generator=g).to(BF16)
    return x


def same_tail(big, small):
    return torch.equal(big[-LAST:], small)


def test_layer_norm_beyond_2_31_elements():
    g = torch.Generator(device="cuda").manual_seed(0)
    rows, cols = 2 ** 31 // 4096 + 300, 4096
    x, d, dh = (tail_filled(rows, cols, g) for _ in range(3))
    w = torch.randn(cols, device="cuda", generator=g).requires_grad_(True)
    leaves = [t.requires_grad_(True) for t in (x, d)]
    total, h = nv.add_layer_norm(*leaves, w)
    grads = torch.autograd.grad(h, (*leaves, w), dh)
    small = [t.detach()[-LAST:].clone().requires_grad_(True) for t in leaves]
    t2, h2 = nv.add_layer_norm(*small, w)
    want = torch.autograd.grad(h2, (*small, w), dh[-LAST:])
    assert same_tail(total, t2) and same_tail(h, h2) and same_tail(grads[0], want[0])
    assert not grads[0][:1000].any() and not h[:1000].any()
    # the rows of zeros add nothing; the others are added in another order: 2^-20 of their magnitudes
    assert bool(((grads[2] - want[2]).abs() <= 2.0 ** -18 * LAST * 40).all())


def test_rotary_beyond_2_31_elements():
    seq, heads, dim = 2 ** 31 // (16 * 64) + 50, 16, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    q = tail_filled(seq, heads * dim, g).view(1, seq, heads, dim)
    pos = torch.arange(seq, device="cuda")[:, None].expand(seq, 2)
    out = nv.rotary_axes(q, None, pos, (12, 20))[0]
    want = nv.rotary_axes(q[:, -LAST:], None, pos[-LAST:], (12, 20))[0]
    assert same_tail(out[0], want[0]) and not out[0, :1000].any()
    # the fused gradient: three tensors of 2^31 / 3 elements and more in one of 2^31
    seq = 2 ** 31 // (48 * 64) + 50
    parts = [tail_filled(seq, heads * dim, g).view(1, seq, heads, dim) for _ in range(3)]
    qkv = torch.zeros(1, seq, 48 * dim, dtype=BF16, device="cuda", requires_grad=True)
    grad, = torch.autograd.grad(nv.rotary_axes_qkv(qkv, pos[:seq], (12, 20), heads), qkv, parts)
    leaf = torch.zeros(1, LAST, 48 * dim, dtype=BF16, device="cuda", requires_grad=True)
    want, = torch.autograd.grad(nv.rotary_axes_qkv(leaf, pos[seq - LAST:seq], (12, 20), heads), leaf, [t[:, -LAST:] for t in parts])
    assert same_tail(grad[0], want[0]) and not grad[0, :1000].any()


def test_fp8_linear_beyond_2_31_elements():
    g = torch.Generator(device="cuda").manual_seed(2)
    tokens, k, n = 2 ** 31 // 4096 + 300, 4096, 128
    x = tail_filled(tokens, k, g)
    w = torch.randn(n, k, device="cuda", generator=g).to(BF16)
    y = nv.fp8_linear(x, w)
    assert same_tail(y, nv.fp8_linear(x[-LAST:], w)) and not y[:1000].any()
    # a result of more than 2^31 elements, and its gradient
    w = torch.randn(k, n, device="cuda", generator=g).to(BF16)
    x = tail_filled(tokens, n, g).requires_grad_(True)
    y = nv.fp8_linear(x, w)
    small = x.detach()[-LAST:].clone().requires_grad_(True)
    y2 = nv.fp8_linear(small, w)
    assert same_tail(y, y2) and not y[:1000].any()
    dy = tail_filled(tokens, k, g)
    assert same_tail(torch.autograd.grad(y, x, dy)[0], torch.autograd.grad(y2, small, dy[-LAST:])[0])


FIRST_CALL = """
import sys
sys.path.insert(0, sys.argv[1])
import torch
import nvfp4_training as nv
torch.cuda.init()
x = torch.randn(40, 512, device="cuda").bfloat16().requires_grad_(True)
w = torch.randn(768, 512, device="cuda").bfloat16().requires_grad_(True)
gain = torch.ones(512, device="cuda", requires_grad=True)
pos = torch.arange(40, device="cuda").view(1, 40, 1)
dy = torch.randn(1, 40, 4, 64, device="cuda").bfloat16()
def step(x, w, gain):
    q, k, v = nv.rotary_axes_qkv(nv.fp8_linear(nv.layer_norm(x, gain), w).view(1, 40, 768), pos, (32,), 4)
    return (q, k, v, *torch.autograd.grad((q, k, v), (x, w, gain), (dy, dy, dy)))
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = step(x, w, gain)
graph.replay()
want = step(*(t.detach().clone().requires_grad_(True) for t in (x, w, gain)))
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
from nvfp4_training import _native
_native.check_status()
print("captured first")
"""


def test_first_call_of_a_process_inside_a_capture():
    folder = str(Path(__file__).resolve().parents[1] / "sm120-nvfp4-training_b200")
    done = subprocess.run([sys.executable, "-c", FIRST_CALL, folder], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "captured first" in done.stdout, done.stderr[-2000:]


def test_calls_on_four_streams_at_once():
    """Workspaces and statistics of calls that overlap do not meet: every stream gets what it gets alone."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = torch.randn(1024, 1024, device="cuda", generator=g).to(BF16).requires_grad_(True)
    gain = torch.ones(1024, device="cuda", requires_grad=True)
    inputs = [torch.randn(m, 1024, device="cuda", generator=g).to(BF16).requires_grad_(True) for m in (1, 100, 700, 3000)]

    def step(x):
        h = nv.layer_norm(x, gain)
        y = nv.fp8_linear(h, w)
        return (y, *torch.autograd.grad(y, (x, w, gain), torch.ones_like(y)))
    want = [step(x) for x in inputs]
    streams = [torch.cuda.Stream() for _ in inputs]
    torch.cuda.synchronize()
    got = [[] for _ in inputs]
    for _ in range(5):
        for i, (x, stream) in enumerate(zip(inputs, streams)):
            with torch.cuda.stream(stream):
                got[i].append(step(x))
    torch.cuda.synchronize()
    for runs, one in zip(got, want):
        for run in runs:
            assert all(torch.equal(a, b) for a, b in zip(run, one))
