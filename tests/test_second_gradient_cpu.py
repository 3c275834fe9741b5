"""A parameter whose layer ran twice in a step has two gradients: one that the optimizer collected from the layer, and one that autograd
left in .grad, in the parameter's dtype.  The update kernels read the second one as FP32."""
import pytest
import torch

from nvfp4_training import _native as nat
from nvfp4_training._backend.optimizer import AdamW, AdamW6


@pytest.mark.parametrize("dtype,fmt", [(torch.float16, "half16_v8"), (torch.bfloat16, "sr16_v8"), (torch.float32, "tile32"), (torch.float32, None)])
def test_second_gradient_reaches_the_kernel_in_fp32(monkeypatch, dtype, fmt):
    p = torch.nn.Parameter(torch.zeros(64, 80, dtype=dtype))
    opt = AdamW([p]) if fmt is None else AdamW6([p], fmt)
    seen = []
    monkeypatch.setattr(nat, "adamw_step", lambda *a, extra=None, **k: seen.append(extra))
    monkeypatch.setattr(torch.cuda, "device", lambda d: __import__("contextlib").nullcontext())
    first = torch.ones(64, 80)
    p.grad = torch.full_like(p, 0.25)
    with torch.no_grad():
        opt._update_param(p, opt.param_groups[0], (first, None, None))
    assert seen[0].dtype == torch.float32 and seen[0].numel() == p.numel() and bool((seen[0] == 0.25).all())
    p.grad = None
    with torch.no_grad():
        opt._update_param(p, opt.param_groups[0], (first, None, None))
    assert seen[1] is None
