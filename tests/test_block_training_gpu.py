"""The operators together, as a video transformer uses them: residual sum + layer norm, 8-bit projections, rotary positions over
time, height and width; on their own against the formulas in 64 bits, and inside converted models (eager, captured, resumed)."""
import copy

import pytest
import torch
from torch import nn
from torch.nn import functional as F

import nvfp4_training as nv

pytestmark = pytest.mark.gpu
SECTIONS = (4, 6, 6)


class Block(nn.Module):
    def __init__(self, dim, heads, kv_heads, hidden):
        super().__init__()
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, dim // heads
        self.norm1, self.norm2 = nn.LayerNorm(dim), nn.LayerNorm(dim)
        self.qkv, self.out = nn.Linear(dim, (heads + 2 * kv_heads) * self.head_dim), nn.Linear(dim, dim)
        self.up, self.down = nn.Linear(dim, hidden), nn.Linear(hidden, dim)

    def forward(self, x, delta, positions, ops):
        b, s, d = x.shape
        x, h = ops.add_norm(x, delta, self.norm1)
        q, k, v = ops.rotary(ops.linear(h, self.qkv), positions, self.heads, self.kv_heads)
        k, v = (t.repeat_interleave(self.heads // self.kv_heads, dim=2) for t in (k, v))
        weights = torch.softmax(torch.einsum("bshd,bthd->bhst", q, k) / self.head_dim ** 0.5, dim=-1)
        x, h = ops.add_norm(x, ops.linear(torch.einsum("bhst,bthd->bshd", weights, v).reshape(b, s, d), self.out), self.norm2)
        return x, ops.linear(F.gelu(ops.linear(h, self.up)), self.down)


class Kernels:
    @staticmethod
    def add_norm(x, delta, norm):
        return nv.add_layer_norm(x, delta, norm.weight, norm.bias, norm.eps)

    @staticmethod
    def linear(x, layer):
        return nv.fp8_linear(x, layer.weight, layer.bias)

    @staticmethod
    def rotary(qkv, positions, heads, kv_heads):
        return nv.rotary_axes_qkv(qkv, positions, SECTIONS, heads, kv_heads, frequencies="axis", layout="interleaved")


def e4m3(x, block_rows, block_cols):
    rows, cols = x.shape
    t = F.pad(x, (0, -cols % block_cols, 0, -rows % block_rows))
    t = t.view(t.shape[0] // block_rows, block_rows, t.shape[1] // block_cols, block_cols)
    m, e = torch.frexp(t.abs().amax(3, keepdim=True).amax(1, keepdim=True))
    two = lambda n: ((n.long() + 1023) << 52).view(torch.float64)
    scale = two(torch.where(m > 0, e - 9 + (m > 0.875).int(), 0))
    v = t / scale
    step = two((torch.frexp(v)[1] - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step * scale).reshape(t.shape[0] * block_rows, -1)[:rows, :cols]


class _Linear64(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return e4m3(x, 1, 128) @ e4m3(w, 128, 128).t()

    @staticmethod
    def backward(ctx, g):
        x, w = ctx.saved_tensors
        return e4m3(g, 1, 128) @ e4m3(w, 128, 128), e4m3(g, 128, 1).t() @ e4m3(x, 128, 1)


class Formulas:
    @staticmethod
    def add_norm(x, delta, norm):
        s = x + delta
        return s, F.layer_norm(s, s.shape[-1:], norm.weight, norm.bias, norm.eps)

    @staticmethod
    def linear(x, layer):
        return (_Linear64.apply(x.reshape(-1, x.shape[-1]), layer.weight) + layer.bias).view(*x.shape[:-1], -1)

    @staticmethod
    def rotary(qkv, positions, heads, kv_heads):
        b, s, width = qkv.shape
        q, k, v = qkv.view(b, s, heads + 2 * kv_heads, -1).split((heads, kv_heads, kv_heads), dim=2)
        angle = torch.cat([positions[:, a:a + 1].double() * 10000.0 ** -(torch.arange(n, device=qkv.device, dtype=torch.float64) / n)
                           for a, n in enumerate(SECTIONS)], dim=1)
        unit = torch.polar(torch.ones_like(angle), angle)[:, None]
        turn = lambda t: torch.view_as_real(torch.view_as_complex(t.unflatten(-1, (-1, 2)).contiguous()) * unit).flatten(-2)
        return turn(q), turn(k), v


def grid(t, h, w):
    return torch.stack(torch.meshgrid(*(torch.arange(n, device="cuda") for n in (t, h, w)), indexing="ij"), -1).reshape(-1, 3)


def compare(run, modules, x, bound):
    wide = copy.deepcopy(modules).double()
    sides = []
    for mods, ops, dtype in ((modules, Kernels, torch.float32), (wide, Formulas, torch.float64)):
        leaf = x.to(dtype).requires_grad_(True)
        out = run(mods, leaf, ops)
        slope = torch.linspace(-1, 1, out.shape[-1], device="cuda", dtype=dtype) + 0.1
        sides.append([out, *torch.autograd.grad((out * slope).sum(), [leaf, *(p for p in mods.parameters())], allow_unused=True)])
    for got, want in zip(*sides):
        assert (got is None) == (want is None)
        if got is not None:
            assert got.shape == want.shape
            assert (got.double() - want).norm() <= bound * want.norm() + 1e-9, ((got.double() - want).norm() / want.norm()).item()


def test_norm_projection_rotary_against_the_formulas():
    """One quantised layer.  FP32 operands differ from the 64-bit ones by about 2^-20, so a share of 2 * 2^-20 * 2^4 = 2^-15 of
    the codes falls on the other side of a border and is off by a step, at most 2^-3 of its value: 2^-7.5 * 2^-3 = 2^-10.5 of an
    operand's norm, twice that for a product."""
    torch.manual_seed(0)
    block = Block(128, 4, 2, 300).cuda()
    positions = grid(3, 5, 7)
    x = torch.randn(2, 105, 128, device="cuda")

    def run(block, leaf, ops):
        _, h = ops.add_norm(leaf, 0.5 * leaf, block.norm1)
        return torch.cat([t.flatten(2) for t in ops.rotary(ops.linear(h, block.qkv), positions, block.heads, block.kv_heads)], -1)
    compare(run, block, x, 2.0 ** -9)


def test_blocks_against_the_formulas():
    """Two whole blocks.  Behind the first layer the two sides differ by 2^-10, the second layer's codes therefore on a share of
    2^-5, and so on: the difference settles at the rounding noise itself, a relative 2^-3 / sqrt(12) of each operand on each
    side, 7.2 % of a product; six products on the longest way through add up in squares to 18 %."""
    torch.manual_seed(0)
    blocks = nn.ModuleList([Block(128, 4, 2, 300) for _ in range(2)]).cuda()
    positions = grid(3, 5, 7)
    x = torch.randn(2, 105, 128, device="cuda")

    def run(blocks, leaf, ops):
        y, delta = leaf, torch.zeros_like(leaf)
        for block in blocks:
            y, delta = block(y, delta, positions, ops)
        return y + delta
    compare(run, blocks, x, 0.18)


class Model(nn.Module):
    """Patches in, blocks, patches out; the first and the last layer are the ones that usually stay at 8 bits."""

    def __init__(self, dim=128, hidden=384, patch=48):
        super().__init__()
        self.patch_in = nn.Linear(patch, dim)
        self.norm1, self.norm2 = nn.LayerNorm(dim), nn.LayerNorm(dim)
        self.up, self.down = nn.Linear(dim, hidden), nn.Linear(hidden, dim, bias=False)
        self.patch_out = nn.Linear(dim, patch)

    def forward(self, x):
        y = self.patch_in(x)
        y = y + self.down(F.gelu(self.up(self.norm1(y))))
        return self.patch_out(self.norm2(y))


def loss_fn(model, x, y):
    return F.mse_loss(model(x).float(), y)


def fresh(profile="balanced", **options):
    torch.manual_seed(3)
    return nv.enable_nvfp4(Model(), profile=profile, lr=1e-3, fp8_layers=["patch_*"], fused_norms=True, **options)


def batch():
    g = torch.Generator(device="cuda").manual_seed(9)
    return torch.randn(300, 48, device="cuda", generator=g), torch.randn(300, 48, device="cuda", generator=g)


@pytest.mark.parametrize("profile", ["balanced", "conservative", "same_as_v5", "experimental_m4v4"])
def test_eager_equals_captured(profile):
    from nvfp4_training._backend import quant
    x, y = batch()
    results = []
    for captured in (False, True):
        quant.reset_stats()
        model = fresh(profile)
        assert type(model.patch_in) is nv.FP8Linear and type(model.patch_out) is nv.FP8Linear and type(model.norm1) is nv.LayerNorm
        assert type(model.up).__name__ == "AutocastLinear"
        if captured:
            with nv.capture_step(model, loss_fn, x, y, steps=4) as graph:
                losses = [graph.step(x, y).item() for _ in range(4)]
        else:
            losses = [nv.train_step(model, loss_fn, x, y).item() for _ in range(4)]
        nv.check_finite(model)
        results.append((losses, [p.detach().clone() for p in model.parameters()]))
    assert results[0][0] == results[1][0]
    assert all(torch.equal(a, b) for a, b in zip(results[0][1], results[1][1]))


def test_first_gradients_reach_the_optimizer():
    """One step of the 8-bit layers' masters moves by the sign of their gradients, like those of an unconverted copy."""
    x, y = batch()
    model = fresh("same_as_v5")
    plain = copy.deepcopy({n: p.detach().clone() for n, p in model.named_parameters()})
    torch.manual_seed(3)
    dense = Model().cuda()
    with torch.autocast("cuda", dtype=torch.bfloat16):
        loss_fn(dense, x, y).backward()
    nv.train_step(model, loss_fn, x, y)
    for name in ("patch_in.weight", "patch_out.weight", "norm1.weight", "patch_out.bias"):
        moved = dict(model.named_parameters())[name].detach() - plain[name]
        grad = dict(dense.named_parameters())[name].grad
        strong = grad.abs() > grad.abs().mean()            # weak ones may turn under 4-bit noise of the layers between
        assert ((moved * grad)[strong] < 0).float().mean() > 0.95, name


def test_checkpoint_resumes_exactly(tmp_path):
    x, y = batch()
    model = fresh()
    for _ in range(2):
        nv.train_step(model, loss_fn, x, y)
    nv.save_checkpoint(tmp_path / "m.pt", model)
    want = [nv.train_step(model, loss_fn, x, y).item() for _ in range(2)]
    again = fresh()
    assert nv.load_checkpoint(tmp_path / "m.pt", again) == 2
    assert [nv.train_step(again, loss_fn, x, y).item() for _ in range(2)] == want


def test_layer_applied_twice_in_a_step():
    """Both contributions to an 8-bit weight's gradient arrive, whichever way the optimizer collects them."""
    from nvfp4_training._backend import quant

    class Twice(nn.Module):
        def __init__(self):
            super().__init__()
            self.a = nn.Linear(96, 96, bias=False)
            self.b = nn.Linear(96, 96)

        def forward(self, x):
            return self.b(self.a(F.gelu(self.a(x))))
    x = torch.randn(64, 96, device="cuda")
    y = torch.randn(64, 96, device="cuda")
    runs = []
    for way in range(3):
        quant.reset_stats()          # the NVFP4 layer's stochastic rounding starts from the same seed
        torch.manual_seed(1)
        model = nv.enable_nvfp4(Twice(), profile="same_as_v5", lr=1e-3, fp8_layers=["a"])
        if way == 0:
            nv.train_step(model, loss_fn, x, y)
        elif way == 1:
            with nv.capture_step(model, loss_fn, x, y, steps=1) as graph:
                graph.step(x, y)
        else:
            opt = model.nvfp4_optimizer
            opt.zero_grad(set_to_none=True)
            with torch.autocast("cuda", dtype=torch.bfloat16):
                loss_fn(model, x, y).backward()
            opt.step()
        runs.append(model.a.weight.detach().clone())
    assert torch.equal(runs[0], runs[1])
    # the ordinary path adds the two FP32 gradients in autograd: the same numbers
    assert torch.equal(runs[0], runs[2])


def test_refused_requests():
    with pytest.raises(ValueError, match="names no Linear"):
        fresh_with = Model()
        nv.enable_nvfp4(fresh_with, fp8_layers=["patch_in", "nothing*"])
    with pytest.raises(ValueError, match="sequence"):
        nv.enable_nvfp4(Model(), fp8_layers="patch_in")
    with pytest.raises(ValueError, match="bool"):
        nv.enable_nvfp4(Model(), fused_norms=1)
    with pytest.raises(ValueError, match="E4M3 masters"):
        nv.enable_nvfp4(Model(), profile="experimental_fp8_master", fp8_layers=["patch_in"])
    tied = nn.Sequential(nn.Linear(96, 96), nn.Linear(96, 96))
    tied[1].weight = tied[0].weight
    with pytest.raises(ValueError, match="tied"):
        nv.enable_nvfp4(tied, fp8_layers=["0"])


def test_every_layer_at_8_bits():
    torch.manual_seed(0)
    model = nv.enable_nvfp4(Model(), profile="balanced", lr=1e-3, fp8_layers=["*"])
    x, y = batch()
    with nv.capture_step(model, loss_fn, x, y, steps=3) as graph:
        losses = [graph.step(x, y).item() for _ in range(3)]
    nv.check_finite(model)
    assert all(l == l for l in losses)


def test_data_parallel_slots_of_one_rank(tmp_path):
    """One rank of a data-parallel job: the 8-bit layers write their gradients into the reducer's slots, and with one rank the
    updates are those of the model without it."""
    import torch.distributed as dist
    x, y = batch()

    def all_fp8():
        torch.manual_seed(3)
        return nv.enable_nvfp4(Model(), profile="balanced", lr=1e-3, fp8_layers=["*"])
    alone = all_fp8()
    want = [nv.train_step(alone, loss_fn, x, y).item() for _ in range(3)]
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        model = nv.enable_data_parallel(all_fp8())
        assert model.nvfp4_optimizer.reducer.has_slot(model.up.weight)
        assert [nv.train_step(model, loss_fn, x, y).item() for _ in range(3)] == want
        assert all(torch.equal(a, b) for a, b in zip(model.parameters(), alone.parameters()))
    finally:
        dist.destroy_process_group()
