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


FAR = (1 << 24) + 100  # rows that as many workgroups of 256 threads would take past 2^32 threads


def one_off(*shape, dtype=F16, seed=2):
    """Random values one element off the allocator's alignment."""
    g = torch.Generator("cuda").manual_seed(seed)
    n = 1
    for x in shape:
        n *= x
    return torch.randn(n + 1, generator=g, device="cuda").to(dtype)[1:].view(shape)


def test_append_of_more_rows_than_a_launch_has_workgroups():
    import branchcraft_torch as bt
    k, v = one_off(1, 4, 64), one_off(1, 4, 64, seed=3)
    pools = [torch.zeros((3, 16, 4, 64), device="cuda", dtype=F16) for _ in range(2)]
    slots = torch.full((FAR,), -1, device="cuda", dtype=torch.int32)
    rows = [0, 5, (1 << 24) - 2, (1 << 24) - 1, 1 << 24, FAR - 2, FAR - 1]
    slots[torch.tensor(rows, device="cuda")] = torch.arange(20, 20 + len(rows), device="cuda", dtype=torch.int32)
    bt.append_kv_(*pools, k.expand(FAR, 4, 64), v.expand(FAR, 4, 64), slots)
    for pool, x in zip(pools, (k, v)):
        flat = pool.view(-1, 4, 64)
        assert torch.equal(flat[20:20 + len(rows)], x.expand(len(rows), 4, 64))
        assert not flat[:20].any() and not flat[20 + len(rows):].any()


def test_rows_of_more_rows_than_a_launch_has_workgroups():
    """The form without 16-byte loads; the request is the last three rows."""
    import branchcraft_torch as bt
    q, k, v = one_off(1, 1, 64), one_off(4, 16, 1, 64, seed=4), one_off(4, 16, 1, 64, seed=5)
    meta = [torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([[2, 0, 3]], [40], [FAR - 3, FAR])]
    got = bt.chunk_attention(q.expand(FAR, 1, 64), k, v, *meta)
    want, tol = C.reference(q.expand(3, 1, 64).cpu(), k.cpu(), v.cpu(), meta[0].cpu(), meta[1].cpu(),
                            torch.tensor([0, 3]))
    C.check(got[-3:], want, tol)
    assert not got[:-3].any()


def test_tiles_of_more_heads_and_requests_than_a_launch_has_workgroups():
    """4096 requests of one token for each of 4096 KV heads: row by row."""
    import branchcraft_torch as bt
    heads = batch = 4096
    g = torch.Generator("cuda").manual_seed(6)
    q = torch.randn((1, heads, 64), generator=g, device="cuda").to(BF16)
    k, v = (torch.randn((2, 16, heads, 64), generator=g, device="cuda").to(BF16) for _ in range(2))
    lengths = 1 + torch.arange(batch, device="cuda", dtype=torch.int32) % 16
    pages = (torch.arange(batch, device="cuda", dtype=torch.int32) % 2)[:, None].contiguous()
    starts = torch.arange(batch + 1, device="cuda", dtype=torch.int32)
    got = bt.chunk_attention(q.expand(batch, heads, 64), k, v, pages, lengths, starts)
    some = [0, 1, 6, 4095]
    for h in (slice(0, 2), slice(4094, 4096)):
        want, tol = C.reference(q[:, h].expand(4, 2, 64).cpu(), k[:, :, h].cpu(), v[:, :, h].cpu(),
                                pages[some].cpu(), lengths[some].cpu(), torch.arange(5))
        C.check(got[some][:, h], want, tol)


def both(fix, **options):
    import branchcraft_torch as bt
    dev = C.on_gpu(fix)
    want, tol = C.reference(**fix, **options)
    C.check(bt.chunk_attention(*(dev[n] for n in ("q", "k", "v", "pages", "lengths", "starts")), **options),
            want, tol)


@pytest.mark.parametrize("shape", [([40, 3], [35, 1]), ([1100, 70], [34, 2])], ids=["short", "split"])
def test_more_than_64_kv_heads(shape):
    both(C.batch(*shape, 73, 73, 64, F16, seed=30))
    both(C.batch(*shape, 146, 73, 64, BF16, seed=31), window=30)


@pytest.mark.parametrize("lengths", [[1, 40, 300], [2100, 5, 900]], ids=["short", "split"])
@pytest.mark.parametrize("hq,hkv,d,dtype", [(33, 1, 128, F16), (80, 2, 64, BF16), (129, 1, 64, F16)])
def test_groups_of_more_rows_than_the_narrow_form_takes(hq, hkv, d, dtype, lengths):
    """Single tokens whose query heads alone fill a tile."""
    both(C.batch(lengths, [1, 1, 1], hq, hkv, d, dtype, seed=32))


def test_groups_whose_products_pass_32_bits():
    """256 new tokens of 4096 query heads over one KV head."""
    import branchcraft_torch as bt
    fix = C.on_gpu(C.batch([300], [256], 4096, 1, 64, BF16, seed=33))
    meta = [fix[n] for n in ("pages", "lengths", "starts")]
    got = bt.chunk_attention(fix["q"], fix["k"], fix["v"], *meta)
    for heads in ([0, 1], [2047, 4095]):
        want, tol = C.reference(fix["q"][:, heads].cpu(), fix["k"].cpu(), fix["v"].cpu(),
                                *(x.cpu() for x in meta))
        C.check(got[:, heads], want, tol)


def test_inference_mode():
    import branchcraft_torch as bt
    fix = C.on_gpu(C.batch([90, 40], [33, 2], 4, 2, 64, F16, seed=34))
    args = [fix[n] for n in ("q", "k", "v", "pages", "lengths", "starts")]
    want = bt.chunk_attention(*args, cap=4.0)
    q = args[0].clone().requires_grad_()
    with torch.inference_mode():
        assert torch.equal(bt.chunk_attention(*args, cap=4.0), want)
        assert torch.equal(bt.chunk_attention(q, *args[1:], cap=4.0), want)


def test_a_step_of_too_few_rows():
    """Capacity for four rows of six: tables and slots are those of the tokens
    that fit, and so is the attention of every request that fits whole."""
    import branchcraft_torch as bt
    fix = C.batch([20, 37, 9], [2, 3, 1], 4, 2, 64, F16, seed=35)
    dev = C.on_gpu(fix)
    ids = fix["pages"][fix["pages"] >= 0].cuda()
    counts = torch.tensor([2, 3, 1], dtype=torch.int32, device="cuda")
    pages, starts, slots, positions = bt.build_tables(ids, dev["lengths"], counts, fix["pages"].shape[1], 4)
    assert torch.equal(pages, dev["pages"])
    assert starts.tolist() == [0, 2, 4, 4] and positions.tolist() == [18, 19, 34, 35]
    want, tol = C.reference(**fix)
    got = bt.chunk_attention(dev["q"][:4], dev["k"], dev["v"], pages, dev["lengths"], starts)
    C.check(got[:2], want[:2], tol[:2])
