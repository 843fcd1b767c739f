"""The chunk operators at the edges of what they accept."""

import pytest
import torch

import chunk_helpers as C

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def test_starts_that_decrease_leave_only_written_records():
    """Eighty requests over the same 1024 rows plan more tiles than the rows
    have workgroups, so that a split request behind them is never run.  The
    workspace starts as zeros: a record that is counted but not written has no
    parts.  Counted are the first request's two tiles, which are run; every
    record lies inside the step; nothing around the output changes."""
    import branchcraft_capi as capi
    import gpu_helpers as G
    hq, hkv, d, t, width, batch = 32, 8, 128, 1024, 2048, 82
    starts = [0, 40] + [t, 0] * 40 + [40]
    lengths = [16 * width] + [64] * 80 + [16 * width]
    g = torch.Generator("cuda").manual_seed(1)
    q = torch.randn((t, hq, d), generator=g, device="cuda").to(BF16)
    k, v = (torch.randn((8, 16, hkv, d), generator=g, device="cuda").to(BF16) for _ in range(2))
    pages = torch.randint(0, 8, (batch, width), generator=g, device="cuda", dtype=torch.int32)
    ints = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (lengths, starts)]
    shape = capi.Shape(batch, hq, hkv, d, width, 8)
    need = G.lib().bc_chunk_attention_workspace_size(shape, t)
    most = 2 * (2 * torch.cuda.get_device_properties(0).multi_processor_count) // hkv
    at = need - 16 * (1 + 2 * (most // 2 + batch))  # the records, behind the partials
    assert at > 0 and at % 16 == 0
    ws = torch.zeros(need, device="cuda", dtype=torch.uint8)
    whole = torch.full((t + 128, hq, d), 7.0, device="cuda", dtype=BF16)
    strides = capi.PoolStrides(16 * hkv * d, hkv * d, d)
    ins = capi.ChunkInputs(q.data_ptr(), k.data_ptr(), v.data_ptr(), pages.data_ptr(), ints[0].data_ptr(),
                           ints[1].data_ptr(), None, None, None, whole[64:].data_ptr(),
                           capi.RowStrides(hq * d, d), strides, strides, t, capi.BC_BFLOAT16, 1, 0, d ** -0.5, 0.0)
    G.check(G.lib().bc_chunk_attention(shape, ins, ws.data_ptr(), need, G.stream()), "bc_chunk_attention")
    torch.cuda.synchronize()
    records = ws[at:].cpu().view(torch.int32).view(-1, 4)
    split, narrow = records[0, :2].tolist()
    assert (split, narrow) == (2, 0)
    for start, row0, rows, parts in records[1:1 + 2 * split:2].tolist():
        assert parts >= 2 and 0 <= start and 0 < rows <= 128 and start + -(-(row0 + rows) // (hq // hkv)) <= t
    assert bool((whole[:64] == 7).all()) and bool((whole[64 + t:] == 7).all())
