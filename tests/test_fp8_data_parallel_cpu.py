"""What an 8-bit layer hands to the data-parallel reducer, on gloo ranks: weight gradients go into the reducer's slots whatever a
rank's batch holds, so that every rank takes the same collective steps in the same order.  The products themselves need a GPU; a
rank's gradient is written here as the backward pass writes it, into the tensor that the layer names."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _free_port():
    with socket.socket() as s:
        s.bind(("127.0.0.1", 0))
        return s.getsockname()[1]


def _begin(rank, world, port):
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=world)
    import sys
    from pathlib import Path
    sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "sm120-nvfp4-training_b200"))
    from nvfp4_training import fp8
    from nvfp4_training.distributed import GradientReducer
    fp8._check_device = lambda t: None
    return fp8, GradientReducer


def _collecting(params, reducer):
    """As backward_step prepares the weights: their gradients are collected, and by whom."""
    pending = {}
    for p in params:
        p._v4_pending, p._dp_reducer = pending, reducer
    reducer.begin(params)
    return pending


def _no_rows_worker(rank, world, port, results):
    try:
        fp8, GradientReducer = _begin(rank, world, port)
        weights = [torch.nn.Parameter(torch.zeros(64, 80, dtype=torch.bfloat16)) for _ in range(3)]
        for p in weights:
            p._v6_defer_dense = True
        reducer = GradientReducer(weights)
        pending = _collecting(weights, reducer)
        bias = torch.nn.Parameter(torch.zeros(64))
        if rank == 0:                                       # this rank has rows
            for i, p in enumerate(weights):
                into, taken = fp8._weight_gradient_into(p)
                into.fill_(float(i + 1))
                taken(into)
        else:
            x = torch.zeros(0, 80, dtype=torch.bfloat16, requires_grad=True)
            for p in weights:
                fp8.fp8_linear(x, p, bias).sum().backward()
            assert x.grad.shape == (0, 80) and not bias.grad.any()
        assert all(p.grad is None for p in weights)         # nothing is left for a collective of its own
        reducer.finish(weights)
        assert list(pending) == weights and [reducer.launched[i] is weights[i] for i in range(3)] == [True] * 3
        assert all(bool((reducer.slot(p) == i + 1).all()) and pending[p][0] is reducer.slot(p) for i, p in enumerate(weights))
        results[rank] = "ok"
    except Exception as e:  # pragma: no cover - reported to the parent
        results[rank] = repr(e)
    finally:
        dist.destroy_process_group()


def _two_ranks(worker):
    results = mp.Manager().dict()
    mp.spawn(worker, args=(2, _free_port(), results), nprocs=2, join=True)
    assert dict(results) == {0: "ok", 1: "ok"}


def test_rank_without_rows_takes_part_in_the_collectives():
    _two_ranks(_no_rows_worker)


def _twice_worker(rank, world, port, results):
    try:
        fp8, GradientReducer = _begin(rank, world, port)
        weight = torch.nn.Parameter(torch.zeros(64, 80, dtype=torch.bfloat16))
        weight._v6_defer_dense = True
        reducer = GradientReducer([weight])
        pending = _collecting([weight], reducer)
        parts = []
        for value in (1.0, 10.0, 100.0):                    # three applications of the layer in one step
            into, taken = fp8._weight_gradient_into(weight)
            into.fill_(value * (rank + 1))
            if taken is None:
                assert into.dtype == weight.dtype and into.shape == weight.shape
                parts.append(into)                          # autograd adds up what it is given
            else:
                taken(into)
        assert len(parts) == 2 and pending[weight][0] is reducer.slot(weight)
        weight.grad = sum(parts)
        reducer.finish([weight])
        assert bool((reducer.slot(weight) == 3).all()) and bool((weight.grad == 330).all())
        results[rank] = "ok"
    except Exception as e:  # pragma: no cover - reported to the parent
        results[rank] = repr(e)
    finally:
        dist.destroy_process_group()


def test_layer_applied_more_than_once():
    """The slot takes the first gradient, autograd the others, as for the NVFP4 layers; the optimizer adds the two."""
    _two_ranks(_twice_worker)


def test_slots_have_the_gradients_types(tmp_path):
    from nvfp4_training.distributed import GradientReducer
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    try:
        nvfp4, *fp8 = (torch.nn.Parameter(torch.zeros(5000, dtype=t)) for t in (torch.float32, torch.float32, torch.float16, torch.bfloat16))
        nvfp4._v4_request_scale = True
        for p in fp8:
            p._v6_defer_dense = True
        reducer = GradientReducer([nvfp4, *fp8])
        assert [reducer.slot(p).dtype for p in (nvfp4, *fp8)] == [torch.bfloat16, torch.float32, torch.bfloat16, torch.bfloat16]
        # ranks whose slots have one size but two types would pair wrong buffers
        wide, narrow = GradientReducer(fp8[:1]).layout(), GradientReducer(fp8[1:2]).layout()
        assert wide[0] == narrow[0] and wide != narrow
    finally:
        dist.destroy_process_group()
