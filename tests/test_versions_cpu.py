"""Version counters of the pools, on fake tensors: no GPU needed."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


@pytest.mark.parametrize("mode", [torch.enable_grad, torch.no_grad, torch.inference_mode])
@pytest.mark.parametrize("op", ["append_kv_", "write_prefix_"])
def test_the_pools_counters_move_once_a_call(op, mode):
    """In inference mode too, as those of torch's own in-place operations do
    for tensors that were made outside it."""
    import branchcraft_torch as bt
    with FakeTensorMode():
        def half(*shape):
            return torch.zeros(shape, device="cuda", dtype=torch.float16)

        k, v, rows = half(4, 16, 2, 64), half(4, 16, 2, 64), half(7, 2, 64)
        where = torch.zeros(7, device="cuda", dtype=torch.int32) if op == "append_kv_" else [0]
        for calls in (1, 2):
            with mode():
                getattr(bt, op)(k, v, rows, rows, where)
            assert [x._version for x in (k, v, rows)] == [calls, calls, 0]
        with torch.inference_mode():  # made inside: they have no counter
            inner = half(4, 16, 2, 64), half(4, 16, 2, 64)
            getattr(bt, op)(*inner, rows, rows, where)
