"""build_tables, append_kv_ and PagedTreeCache.extend: whole numbers and bits
equal to what plain Python makes of the same lists, and the three together
against the definition of the attention in 64 bits."""

import random

import pytest
import torch

import chunk_helpers as C

pytestmark = pytest.mark.gpu


def plain_tables(ids, lengths, counts, width, tokens):
    table, starts, slots, positions = [], [], [], []
    at = 0
    for n, new in zip((max(x, 0) for x in lengths), (max(x, 0) for x in counts)):
        held = ids[at:at + C.pages_of(n)][:width]
        at += C.pages_of(n)
        table.append(held + [-1] * (width - len(held)))
        starts.append(min(len(slots), tokens))
        for pos in range(n - new, n):
            positions.append(max(pos, -1))
            page = held[pos // 16] if 0 <= pos and pos // 16 < len(held) else -1
            slots.append(16 * page + pos % 16 if 0 <= page < 2**27 else -1)
    starts.append(min(len(slots), tokens))
    slots, positions = (x[:tokens] + [-1] * (tokens - len(x)) for x in (slots, positions))
    return [torch.tensor(x, dtype=torch.int32) for x in (table, starts, slots, positions)]


def gpu_ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


CASES = [
    # lengths, counts, more table columns, more rows than new tokens
    ([1], [1], 0, 0),
    ([16, 17, 15], [1, 1, 1], 2, 0),
    ([40, 0, 7], [5, 0, 7], 0, 9),
    ([0, 0], [0, 0], 1, 3),
    ([300, 2, 77], [300, 1, 30], 0, 0),
    ([50, -4, 20], [70, 3, -2], 1, 5),     # more new tokens than tokens; negative
    ([5000, 33], [4999, 2], 0, 4000),      # several slices of rows
    ([40000, 9], [3, 1], 0, 0),            # several slices of the table
]


@pytest.mark.parametrize("case", range(len(CASES)))
def test_build_tables(case):
    import branchcraft_torch as bt
    lengths, counts, cols, rows = CASES[case]
    r = random.Random(case)
    held = sum(C.pages_of(max(n, 0)) for n in lengths)
    ids = r.sample(range(held + 50), held)
    width = max(max(C.pages_of(max(n, 0)) for n in lengths), 1) + cols
    tokens = sum(max(n, 0) for n in counts) + rows
    want = plain_tables(ids, lengths, counts, width, tokens)
    got = bt.build_tables(gpu_ints(ids), gpu_ints(lengths), gpu_ints(counts), width, tokens)
    for a, b in zip(got, want):
        assert torch.equal(a.cpu(), b)


def test_build_tables_many_requests_and_short_inputs():
    """Over a wave and a workgroup of requests; a table, a list of ids and a
    row count that are too small; ids that no slot can hold."""
    import branchcraft_torch as bt
    r = random.Random(1)
    for batch in (63, 257, 1500):
        lengths = [r.randint(0, 70) for _ in range(batch)]
        counts = [r.randint(0, n) for n in lengths]
        ids = [r.randint(-2, 2**27 + 5) if r.random() < 0.1 else r.randint(0, 9999)
               for _ in range(sum(map(C.pages_of, lengths)))]
        for width, drop, tokens in ((5, 0, sum(counts)), (2, 0, sum(counts)), (5, 40, sum(counts)),
                                    (5, 0, sum(counts) // 2), (5, len(ids), 0)):
            held = ids[:len(ids) - drop]
            want = plain_tables(held, lengths, counts, width, tokens)
            got = bt.build_tables(gpu_ints(held), gpu_ints(lengths), gpu_ints(counts), width, tokens)
            for a, b in zip(got, want):
                assert torch.equal(a.cpu(), b), (batch, width, drop, tokens)


def bits(x):
    return x.contiguous().view(torch.int16)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("tokens,hkv,d", [(1, 8, 128), (3, 1, 64), (17, 3, 64), (300, 8, 128), (70, 40, 128)])
@pytest.mark.parametrize("form", ["plain", "fused", "heads_first", "unaligned", "expanded", "packed pool",
                                  "odd pool"])
def test_append_kv(tokens, hkv, d, form, dtype):
    import branchcraft_torch as bt
    torch.manual_seed(tokens + d)

    def rand(*shape):
        return torch.randn(shape, device="cuda").to(dtype)

    k, v = rand(tokens, hkv, d), rand(tokens, hkv, d)
    if form == "fused":
        rows = rand(tokens, 3, hkv, d)
        k, v = rows[:, 1], rows[:, 2]
    elif form == "heads_first":
        k = rand(hkv, tokens, d).transpose(0, 1)
    elif form == "unaligned":
        k = rand(tokens * hkv * d + 1)[1:].view(tokens, hkv, d)
    elif form == "expanded":
        k, v = rand(1, hkv, d).expand(tokens, hkv, d), rand(tokens, 1, d).expand(tokens, hkv, d)
    pages = tokens // 16 + 4
    if form == "packed pool":
        whole = rand(pages, 2, 16, hkv, d)
        ck, cv = whole[:, 0], whole[:, 1]
    elif form == "odd pool":
        whole = rand(pages, hkv, 16, 2 * d + 1)
        ck, cv = whole[..., :d].transpose(1, 2), whole[..., d + 1:].transpose(1, 2)
    else:
        ck, cv = rand(pages, 16, hkv, d), rand(pages, 16, hkv, d)
    slots = torch.randperm(pages * 16)[:tokens].to(torch.int32)
    slots[::5] = torch.tensor([-1, pages * 16, -2**31, 2**31 - 1])[torch.arange(len(slots[::5])) % 4].int()
    want_k, want_v = ck.clone(), cv.clone()
    for t, slot in enumerate(slots.tolist()):
        if 0 <= slot < pages * 16:
            want_k[slot // 16, slot % 16], want_v[slot // 16, slot % 16] = k[t], v[t]
    versions = ck._version, cv._version
    bt.append_kv_(ck, cv, k, v, slots.cuda())
    assert torch.equal(bits(ck), bits(want_k)) and torch.equal(bits(cv), bits(want_v))
    assert ck._version > versions[0] and cv._version > versions[1]


def test_append_keeps_every_bit():
    """NaN payloads, infinities, signed zeros and subnormals."""
    import branchcraft_torch as bt
    every = torch.arange(-2**15, 2**15, device="cuda").to(torch.int16).view(torch.float16).view(64, 8, 128)
    ck, cv = (torch.zeros(4, 16, 8, 128, device="cuda", dtype=torch.float16) for _ in range(2))
    bt.append_kv_(ck, cv, every, every.flip(0), torch.arange(64, device="cuda", dtype=torch.int32))
    assert torch.equal(bits(ck).view(64, 8, 128), bits(every))
    assert torch.equal(bits(cv).view(64, 8, 128), bits(every.flip(0)))


def random_rows(g, n, heads, d):
    return torch.randn((n, heads, d), generator=g, device="cuda", dtype=torch.float16)


def test_extend_runs_the_whole_step():
    """Prompt chunks, turns and single tokens of requests that share pages,
    step after step: outputs, pages and untouched siblings."""
    from branchcraft_torch.transaction import PagedTreeCache
    hq, hkv, d = 8, 2, 64
    g = torch.Generator("cuda").manual_seed(2)
    r = random.Random(2)
    cache = PagedTreeCache(300, hkv, d)
    rows = {}  # request -> its K and V, as they should be

    def new(n):
        k, v = random_rows(g, n, hkv, d), random_rows(g, n, hkv, d)
        request = cache.new(k, v)
        rows[request] = (k, v)
        return request

    requests = [new(37), new(0), new(16)]
    for source in (requests[0], requests[0], requests[2]):
        requests.append(cache.fork(source))
        rows[requests[-1]] = rows[source]
    sibling = cache.fork(requests[0])  # never extended
    rows[sibling] = rows[requests[0]]
    for step in range(4):
        counts = [r.choice((0, 1, 1, 2, 15, 16, 40)) for _ in requests]
        counts[step % len(counts)] = 33
        total = sum(counts)
        q, k, v = random_rows(g, total, hq, d), random_rows(g, total, hkv, d), random_rows(g, total, hkv, d)
        options = [dict(), dict(cap=4.0), dict(window=20),
                   dict(slopes=torch.rand(hq, generator=g, device="cuda"))][step]
        out = cache.extend(requests, counts, q, k, v, **options)
        at = 0
        for request, n in zip(requests, counts):
            rows[request] = tuple(torch.cat((old, x[at:at + n])) for old, x in zip(rows[request], (k, v)))
            at += n
        cache.owner.check_invariants()
        lengths = [len(rows[x][0]) for x in requests]
        width = max(map(C.pages_of, lengths))
        table = torch.tensor([cache.pages[x] + [-1] * (width - len(cache.pages[x])) for x in requests])
        starts = torch.tensor([0] + torch.tensor(counts).cumsum(0).tolist())
        cpu = {n: x.cpu() if isinstance(x, torch.Tensor) else x for n, x in options.items()}
        want, tol = C.reference(q.cpu(), cache.k.cpu(), cache.v.cpu(), table, torch.tensor(lengths), starts, **cpu)
        C.check(out, want, tol, f"step {step}")
        for request in requests + [sibling]:
            n = len(rows[request][0])
            assert cache.lengths[request] == n
            ids = torch.tensor(cache.pages[request], dtype=torch.long, device="cuda")
            for pool, x in zip((cache.k, cache.v), rows[request]):
                assert torch.equal(bits(pool[ids].flatten(0, 1)[:n]), bits(x))


def test_extend_matches_commits_of_the_same_tokens():
    """Pages and tables as consecutive commits leave them."""
    from branchcraft_torch.transaction import PagedTreeCache
    g = torch.Generator("cuda").manual_seed(3)
    k, v = random_rows(g, 21, 2, 64), random_rows(g, 21, 2, 64)
    dk, dv = random_rows(g, 10, 2, 64), random_rows(g, 10, 2, 64)
    caches = [PagedTreeCache(20, 2, 64) for _ in range(2)]
    for cache in caches:
        first = cache.new(k, v)
        cache.fork(first)
    caches[0].extend([0, 1], [5, 5], random_rows(g, 10, 2, 64), dk, dv)
    for request in (0, 1):
        part = slice(5 * request, 5 * request + 5)
        caches[1].commit(request, [0, 1, 2, 3, 4], dk[None, part].contiguous(), dv[None, part].contiguous())
    assert caches[0].pages == caches[1].pages and caches[0].lengths == caches[1].lengths
    assert torch.equal(bits(caches[0].k), bits(caches[1].k)) and torch.equal(bits(caches[0].v), bits(caches[1].v))


def test_extend_refuses_before_anything_changes():
    from branchcraft_torch.transaction import PagedTreeCache
    g = torch.Generator("cuda").manual_seed(4)
    cache = PagedTreeCache(4, 2, 64)
    a = cache.new(random_rows(g, 20, 2, 64), random_rows(g, 20, 2, 64))
    b = cache.fork(a)
    q, k = random_rows(g, 30, 4, 64), random_rows(g, 30, 2, 64)

    def state():
        return ({x: list(p) for x, p in cache.pages.items()}, dict(cache.lengths), list(cache.free),
                list(cache.refcount))

    before = state()
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.extend([a, b], [29, 1], q, k, k)  # 20 + 29 tokens: two more pages and a clone; two are free
    refusals = [([a, a], [15, 15], q, k, {}), ([a], [30, 0], q, k, {}), ([], [], q[:0], k[:0], {}),
                ([a, b], [31, -1], q, k, {}),
                ([a], [5], q[:5, :1].expand(5, 4098, 64), k[:5], {}), ([a], [29], q, k, {}), ([a], [30], q[:, :3], k, {}),
                ([a], [30], q.bfloat16(), k, {}), ([a], [30], q, k.cpu(), {}),
                ([a], [5], q[:5], k[:5].clone().requires_grad_(), {}),
                ([a], [5], q[:5].clone().requires_grad_(), k[:5], {}),
                ([a], [5], q[:5], k[:5], dict(cap=-1.0)), ([a], [5], q[:5], k[:5], dict(windows=1)),
                ([a], [5], q[:5], k[:5], dict(first=torch.zeros(4, device="cuda", dtype=torch.int32)))]
    for requests, counts, qq, kk, options in refusals:
        with pytest.raises((ValueError, RuntimeError, TypeError)):
            cache.extend(requests, counts, qq, kk, kk.detach(), **options)
        assert state() == before
    assert cache.extend([a, b], [12, 3], q[:15], k[:15], k[:15]).shape == (15, 4, 64)


def test_extend_refuses_a_tangent_before_anything_changes():
    from torch.autograd import forward_ad
    from branchcraft_torch.transaction import PagedTreeCache
    g = torch.Generator("cuda").manual_seed(6)
    cache = PagedTreeCache(4, 2, 64)
    a = cache.new(random_rows(g, 20, 2, 64), random_rows(g, 20, 2, 64))
    rows = random_rows(g, 5, 2, 64)
    with forward_ad.dual_level():
        with pytest.raises(ValueError, match="differentiable"):
            cache.extend([a], [5], rows, rows, forward_ad.make_dual(rows, rows))
    assert cache.lengths[a] == 20 and len(cache.pages[a]) == 2


def test_extend_with_rows_of_the_pool_itself():
    """Another request's tokens once more, as views of its pages."""
    from branchcraft_torch.transaction import PagedTreeCache
    g = torch.Generator("cuda").manual_seed(5)
    caches = [PagedTreeCache(8, 2, 64) for _ in range(2)]
    k, v, q = random_rows(g, 40, 2, 64), random_rows(g, 40, 2, 64), random_rows(g, 12, 4, 64)
    outs = []
    for cache in caches:
        a, b = cache.new(k, v), cache.new(k[:5], v[:5])
        page = cache.pages[a][1]
        rows = [pool[page, 2:14] for pool in (cache.k, cache.v)]
        if cache is caches[1]:
            rows = [x.clone() for x in rows]
        outs.append(cache.extend([b, a], [5, 7], q, *rows))
    assert torch.equal(bits(outs[0]), bits(outs[1]))
    assert torch.equal(bits(caches[0].k), bits(caches[1].k)) and torch.equal(bits(caches[0].v), bits(caches[1].v))
