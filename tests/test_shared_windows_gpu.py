"""Attention within windows over an 8-bit cache and of requests that begin alike: what
a call takes from the allocator, and the kernels that read shared pages once, at the
windows, groups and sizes where they can go wrong."""

import pytest
import torch

import chunk_helpers as C
import fp8_helpers as F

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def taken(call):
    """Bytes that a call has from the allocator at most, its output among them."""
    call()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    most = torch.cuda.max_memory_allocated() - before
    return out, most


@pytest.mark.parametrize("window,new", [(1024, 1), (512, 90)])
def test_no_workspace_where_a_window_is_not_cut(window, new):
    """Long tables, of which the rows see as much as tables have that are not cut."""
    import branchcraft_torch as bt
    fix, groups, shared = F.forks([(1100, [(new + i, new) for i in range(3)])], 4, 2, 64, BF16, seed=1)
    assert fix["pages"].shape[1] > 4096 // 16 and not F.pays(fix, window)
    pool, same = F.pools(fix)
    dev, pool = C.on_gpu(fix), [x.cuda() for x in pool]
    meta = [dev[n] for n in ("pages", "lengths", "starts")]
    groups, shared = groups.cuda(), shared.cuda()
    calls = [(same, lambda **k: bt.fp8_chunk_attention(dev["q"], *pool, *meta, **k)),
             (fix, lambda **k: bt.shared_chunk_attention(dev["q"], dev["k"], dev["v"], *meta, groups, shared, **k))]
    for held, call in calls:
        out, most = taken(lambda: call(window=window))
        assert most <= -(-out.numel() * 2 // 512) * 512
        want, tol = C.reference(**held, window=window)
        C.check(out, want, tol)
        assert taken(call)[1] > 10 << 20  # without a window it takes one
