"""Shared prefixes at the edges of what they accept: many requests and groups, layouts,
far pages, captured steps, streams, refusals, and extend over forks."""

import pytest
import torch

import chunk_helpers as C
import fp8_helpers as F
import test_chunk_gpu as K
from test_shared_gpu import attend, both

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


@pytest.mark.parametrize("shape", ["many groups", "one of many", "across blocks"])
def test_more_requests_and_groups_than_a_wave_has_lanes(shape):
    groups = {"many groups": [(16 + g % 5 * 16, [(1 + g % 3, 1)] * 3) for g in range(70)],
              "one of many": [(80, [(1 + i % 20, 1 + i % 2) if i % 20 else (2, 2) for i in range(200)])],
              "across blocks": [(33, [(9, 1)] * 50), (96, [(2, 1)] * 100), (48, [(5, 5)] * 30)]}[shape]
    fix, bounds, shared = F.forks(groups, 2, 1, 64, F16, seed=3)
    both(fix, bounds, shared)


@pytest.mark.parametrize("sizes", ["pairs", "after a large one", "with empty ones"])
def test_groups_beyond_the_first_64_of_requests_in_blocks(sizes):
    """A request's group is found among up to thousands: pairs, one group over several
    blocks of 64 requests before them, and groups of none between them."""
    pairs = [(16 + g % 4 * 16, [(1 + g % 3, 1), (2, 1)]) for g in range(150)]
    if sizes == "after a large one":
        pairs = pairs[:70] + [(64, [(2, 1)] * 150)] + pairs[70:]
    fix, bounds, shared = F.forks(pairs, 2, 1, 64, F16, seed=12, lone_ends=1)
    if sizes == "with empty ones":  # three of no request before every eighth
        at = [i for i in range(len(shared)) for _ in range(4 if i % 8 == 7 else 1)]
        bounds, shared = torch.cat((bounds[at], bounds[-1:])), shared[at]
        assert len(shared) > 192 and (bounds[1:] >= bounds[:-1]).all()
    both(fix, bounds, shared)


@pytest.mark.parametrize("hq,hkv", [(73, 73), (129, 1), (146, 73)])
def test_many_kv_heads_and_wide_groups(hq, hkv):
    fix, bounds, shared = F.forks([(160, [(3, 1)] * 9), (40, [(20, 1)] * 2)], hq, hkv, 64, BF16, seed=4)
    if hq // hkv < 80:
        both(fix, bounds, shared)
    else:  # rows that fill tiles by themselves: every request reads its own
        assert not F.pays(fix)
        want, tol = C.reference(**fix)
        C.check(attend(fix, bounds, shared), want, tol)


def test_layouts():
    """Packed pools, heads before slots, strided and unaligned queries."""
    import branchcraft_torch as bt
    fix, bounds, shared = F.forks([(300, [(5, 2)] * 6), (100, [(30, 9)] * 2)], 4, 2, 64, F16, seed=6)
    want, tol = C.reference(**fix)
    k, v, q = (fix[n].cuda() for n in ("k", "v", "q"))
    meta = [fix[n].cuda() for n in ("pages", "lengths", "starts")] + [bounds.cuda(), shared.cuda()]
    whole = torch.stack((k, v), 1)
    heads = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    fused = torch.cat((q, q[:, :2]), 1)[:, :4]
    off = torch.cat((q.new_zeros(1), q.flatten()))[1:].view(q.shape)
    for query, kv in ((q, (whole[:, 0], whole[:, 1])), (q, heads), (fused, (k, v)), (off, (k, v)),
                      (q.transpose(0, 1).contiguous().transpose(0, 1), (k, heads[1]))):
        C.check(bt.shared_chunk_attention(query, *kv, *meta), want, tol)


def test_the_first_members_pages_are_read():
    """What the others' tables say of the shared tokens is not looked at: pages of
    NaN there, of the same contents as far as the call is told."""
    fix, bounds, shared = F.forks([(320, [(5, 1)] * 9)], 4, 2, 64, F16, seed=7)
    want, tol = C.reference(**fix)
    spare = min({*range(fix["k"].shape[0])} - {*fix["pages"].flatten().tolist()})
    fix["k"][spare] = fix["v"][spare] = float("nan")
    fix["pages"][1:, :20] = spare
    C.check(attend(fix, bounds, shared), want, tol)


def test_pool_past_32_bits():
    import branchcraft_torch as bt
    hkv, d, pool = 8, 128, 270000
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.empty((pool, 16, hkv, d), device="cuda", dtype=BF16) for _ in range(2))
    ids = [pool - 1, 5, 262143, 131072, pool - 9, 131071, 9]
    rows = [torch.randn((7, 16, hkv, d), generator=g, device="cuda").to(BF16) for _ in range(2)]
    for x, r in zip((k, v), rows):
        x[torch.tensor(ids, device="cuda")] = r
    width = 1800
    table, small = (torch.full((3, width), -1, dtype=torch.int32) for _ in range(2))
    for b in range(3):
        order = [0, 1, 2, 3, 4 + b]
        small[b, :5] = torch.tensor(order)
        table[b, :5] = torch.tensor(ids)[order]
    lengths = torch.tensor([70, 65, 80], dtype=torch.int32)
    starts = torch.tensor([0, 1, 2, 4], dtype=torch.int32)
    q = torch.randn((4, 16, d), generator=g, device="cuda").to(BF16)
    fix = dict(q=q.cpu(), k=rows[0].cpu(), v=rows[1].cpu(), pages=small, lengths=lengths, starts=starts)
    assert F.pays(fix)
    want, tol = C.reference(**fix)
    got = bt.shared_chunk_attention(q, k, v, table.cuda(), lengths.cuda(), starts.cuda(),
                                    torch.tensor([0, 3], dtype=torch.int32).cuda(), torch.tensor([64], dtype=torch.int32).cuda())
    C.check(got, want, tol)


def test_workspace_refused_or_short_gives_the_same():
    import branchcraft_capi as capi
    import gpu_helpers as G
    fix, bounds, shared = F.forks([(700, [(5, 1)] * 6)], 4, 2, 128, F16, seed=15)
    assert F.pays(fix)
    want, tol = C.reference(**fix)
    dev = C.on_gpu(fix)
    (t, hq, d), (pool, _, hkv, _) = dev["q"].shape, dev["k"].shape
    shape = capi.Shape(6, hq, hkv, d, dev["pages"].shape[1], pool)
    need = G.lib().bc_shared_chunk_attention_workspace_size(shape, t, 1)
    assert need > 0
    ws = torch.empty(need + 16, device="cuda", dtype=torch.uint8)
    strides = capi.PoolStrides(16 * hkv * d, hkv * d, d)
    groups = bounds.cuda(), shared.cuda()
    for at, size in ((None, 0), (ws.data_ptr(), need // 4), (ws.data_ptr() + 4, need), (ws.data_ptr(), need)):
        out = torch.full_like(dev["q"], float("nan"))
        ins = capi.ChunkInputs(*(dev[n].data_ptr() for n in ("q", "k", "v", "pages", "lengths", "starts")),
                               None, None, None, out.data_ptr(), capi.RowStrides(hq * d, d), strides, strides,
                               t, capi.BC_FLOAT16, 1, 0, d ** -0.5, 0.0)
        ws.fill_(0xff)  # nothing in it is taken for written
        G.check(G.lib().bc_shared_chunk_attention(shape, ins, *(x.data_ptr() for x in groups), 1, at, size, G.stream()),
                "bc_shared_chunk_attention")
        C.check(out, want, tol, f"workspace {size}")


def test_captured_steps_follow_the_lengths():
    """Captured once and replayed while own lengths, rows and what is shared change in
    place, with eager calls between; every replay equals the eager call."""
    import branchcraft_torch as bt
    fix, bounds, shared = F.forks([(640, [(90, 2)] * 6), (200, [(60, 1)] * 5)], 8, 2, 64, F16, seed=9)
    dev = C.on_gpu(fix)
    for n in ("k", "v"):
        dev[n].nan_to_num_(0.5)
    args = [dev[n] for n in ("q", "k", "v", "pages", "lengths", "starts")] + [bounds.cuda(), shared.cuda()]
    g = torch.Generator("cuda").manual_seed(6)
    full, most = dev["lengths"].clone(), shared.cuda()
    bt.shared_chunk_attention(*args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = bt.shared_chunk_attention(*args)
    for n in range(6):
        dev["lengths"].copy_(full - 9 * n)
        args[7].copy_(most - torch.tensor([100 * n, 200 if n == 4 else n], dtype=torch.int32, device="cuda"))
        dev["q"].copy_(torch.randn(dev["q"].shape, generator=g, device="cuda"))
        want = bt.shared_chunk_attention(*args).clone()
        plain = bt.chunk_attention(*args[:6])
        torch.cuda.synchronize()
        out.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
        assert bool((out.float() - plain.float()).abs().max() < 0.02)


def test_two_streams_at_once_and_the_same_bits():
    import branchcraft_torch as bt
    args = []
    for s in (20, 21):
        fix, bounds, shared = F.forks([(1500, [(70, 1)] * 12), (300, [(50, 20), (3, 1), (2, 2)])], 8, 2, 128, F16, seed=s)
        args.append([fix[n].cuda() for n in ("q", "k", "v", "pages", "lengths", "starts")] + [bounds.cuda(), shared.cuda()])
    want = [bt.shared_chunk_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(bt.shared_chunk_attention(*args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_compile():
    import branchcraft_torch as bt
    fix, bounds, shared = F.forks([(160, [(5, 1)] * 8)], 4, 2, 64, F16, seed=23)
    args = tuple(fix[n].cuda() for n in ("q", "k", "v", "pages", "lengths", "starts")) + (bounds.cuda(), shared.cuda())
    whole = torch.compile(lambda *a: bt.shared_chunk_attention(*a) * 2, fullgraph=True)
    assert torch.equal(whole(*args), bt.shared_chunk_attention(*args) * 2)


REFUSALS = {
    "group type": dict(groups=lambda x: x.long()), "group rank": dict(groups=lambda x: x[None]),
    "too few bounds": dict(groups=lambda x: x[:1]), "shared type": dict(shared=lambda x: x.float()),
    "host groups": dict(groups=lambda x: x.cpu()), "host shared": dict(shared=lambda x: x.cpu()),
    "more groups than requests": dict(groups=lambda x: torch.zeros(10, dtype=torch.int32).cuda(),
                                      shared=lambda x: torch.zeros(9, dtype=torch.int32).cuda()),
    "strided": dict(groups=lambda x: torch.stack((x, x), 1)[:, 0]), "k type": dict(k=lambda x: x.bfloat16()),
    "q rank": dict(q=lambda x: x[0]), "starts": dict(starts=lambda x: x[:-1]), "table rows": dict(pages=lambda x: x[:1]),
}


@pytest.mark.parametrize("what", REFUSALS)
def test_refusals(what):
    import branchcraft_torch as bt
    fix, bounds, shared = F.forks([(160, [(5, 1)] * 8)], 4, 2, 64, F16, seed=23)
    case = C.on_gpu(fix) | dict(groups=bounds.cuda(), shared=shared.cuda())
    names = ("q", "k", "v", "pages", "lengths", "starts", "groups", "shared")
    bt.shared_chunk_attention(*(case[n] for n in names))
    for name, change in REFUSALS[what].items():
        case[name] = change(case[name])
    with pytest.raises((RuntimeError, NotImplementedError)):
        bt.shared_chunk_attention(*(case[n] for n in names))


def test_extend_over_forks():
    """Samples of one prompt that grow apart, a second prompt's, and a request alone:
    the same pages and lengths as without sharing, outputs against the definition."""
    from branchcraft_torch.transaction import PagedTreeCache
    outs, caches = [], []
    for share in (False, True):
        g = torch.Generator("cuda").manual_seed(4)

        def rand(n, heads):
            return torch.randn((n, heads, 64), generator=g, device="cuda", dtype=F16)

        cache = PagedTreeCache(1400, 8, 64)
        a = cache.new(rand(6007, 8), rand(6007, 8))
        b = cache.new(rand(1111, 8), rand(1111, 8))
        who = [a] + [cache.fork(a) for _ in range(6)] + [b, cache.fork(b), cache.new(rand(70, 8), rand(70, 8))]
        mine = []
        for turn, counts in enumerate(([2] * 7 + [3, 1, 30], [1] * 10, [1, 0, 1, 5, 1, 1, 1, 0, 0, 2])):
            total = sum(counts)
            q, k, v = rand(total, 16), rand(total, 8), rand(total, 8)
            options = [{}, dict(cap=20.0), dict(slopes=torch.rand(16, generator=g, device="cuda"))][turn]
            mine.append((q, counts, options, cache.extend(who, counts, q, k, v, share=share, **options)))
        outs.append(mine)
        caches.append((cache, who))
    (plain, _), (cache, who) = caches
    assert plain.pages == cache.pages and plain.lengths == cache.lengths and plain.free == cache.free
    assert torch.equal(plain.k, cache.k) and torch.equal(plain.v, cache.v)
    bounds, tokens = cache.owner.shared_prefixes(who)
    assert bounds == [0, 7, 9, 10] and tokens[:2] == [6007 // 16 * 16, 1111 // 16 * 16]
    for (q, counts, options, x), (_, _, _, y) in zip(*outs):
        assert float((x.float() - y.float()).abs().max()) < 0.02
    q, counts, options, got = outs[1][-1]
    lists = [cache.pages[x] for x in who]
    table = torch.full((len(who), max(map(len, lists))), -1, dtype=torch.int32)
    for i, pages in enumerate(lists):
        table[i, :len(pages)] = torch.tensor(pages)
    starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
    fix = dict(q=q.cpu(), k=cache.k.cpu(), v=cache.v.cpu(), pages=table, starts=starts,
               lengths=torch.tensor([cache.lengths[x] for x in who], dtype=torch.int32))
    assert F.pays(fix)
    want, tol = C.reference(**fix, **{n: x.cpu() for n, x in options.items()})
    C.check(got, want, tol)
