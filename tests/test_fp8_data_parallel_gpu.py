"""8-bit layers in a data-parallel job of one rank, whose updates have to be those of the model without it."""
import pytest
import torch
import torch.distributed as dist
from torch import nn
from torch.nn import functional as F

import nvfp4_training as nv

pytestmark = pytest.mark.gpu


class Twice(nn.Module):
    def __init__(self):
        super().__init__()
        self.a = nn.Linear(96, 96, bias=False)
        self.b = nn.Linear(96, 96)

    def forward(self, x):
        return self.b(self.a(F.gelu(self.a(x))))


def loss_fn(model, x, y):
    return F.mse_loss(model(x).float(), y)


def batch():
    g = torch.Generator(device="cuda").manual_seed(9)
    return torch.randn(300, 96, device="cuda", generator=g), torch.randn(300, 96, device="cuda", generator=g)


def fresh(profile):
    torch.manual_seed(1)
    return nv.enable_nvfp4(Twice(), profile=profile, lr=1e-3, fp8_layers=["*"])


@pytest.fixture
def one_rank(tmp_path):
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    yield
    dist.destroy_process_group()


def train(model):
    x, y = batch()
    losses = [nv.train_step(model, loss_fn, x, y).item() for _ in range(3)]
    nv.check_finite(model)
    return losses, [p.detach().float() for p in model.parameters()]


@pytest.mark.parametrize("profile", ["balanced", "conservative", "same_as_v5"])
def test_layer_applied_twice(one_rank, profile):
    """The slot holds the first gradient, autograd the second, in the slot's and the master's types; without data parallel the two are
    added in FP32.  Gradients therefore differ by 2^-8 of themselves at most, and an 8-bit moment by a step, 1/127 of its block's
    largest, in the share of elements that this carries over a border (a quarter for the largest of them): 3/127 of a typical
    moment in a half of the root mean square, 1.2 % a step.  5 % of the way that the weights moved covers three steps."""
    want_losses, want = train(fresh(profile))
    start = [p.detach().float() for p in fresh(profile).parameters()]
    losses, got = train(nv.enable_data_parallel(fresh(profile)))
    assert losses[0] == want_losses[0]
    for g, w, s in zip(got, want, start):
        assert (g - w).norm() <= 0.05 * (w - s).norm()


@pytest.mark.parametrize("profile", ["balanced", "conservative", "same_as_v5"])
def test_one_rank_updates_as_without_data_parallel(one_rank, profile):
    """Gradients keep their types in the slots, FP32 ones too.  (Eager steps: gloo's collectives cannot be captured.)"""
    class Once(nn.Module):
        def __init__(self):
            super().__init__()
            self.a, self.b = nn.Linear(96, 128), nn.Linear(128, 96, bias=False)

        def forward(self, x):
            return self.b(F.gelu(self.a(x)))

    def make():
        torch.manual_seed(1)
        return nv.enable_nvfp4(Once(), profile=profile, lr=1e-3, fp8_layers=["*"])
    want_losses, want = train(make())
    losses, got = train(nv.enable_data_parallel(make()))
    assert losses == want_losses and all(torch.equal(g, w) for g, w in zip(got, want))
