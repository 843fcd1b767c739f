"""The 8-bit cache at the edges of what it accepts: layouts, far pages, captured steps,
streams, refusals, and the cache class over a whole run."""

import pytest
import torch

import chunk_helpers as C
import fp8_helpers as F
import test_chunk_gpu as K
from test_fp8_gpu import attend, raw, rows

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def bytes_as(x, change):
    """A view or copy of codes, made on their bytes."""
    return change(x.view(torch.uint8)).view(F.E4M3)


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("shape", [([200, 31, 90], [60, 1, 4]), ([2100, 40], [3, 2])], ids=["short", "split"])
def test_layouts(dtype, d, shape):
    """Packed pools, heads before slots, strided and unaligned queries."""
    import branchcraft_torch as bt
    fix = C.batch(*shape, 4, 2, d, dtype, seed=3)
    pool, same = F.pools(fix)
    want, tol = C.reference(**same)
    k, sk, v, sv = (x.cuda() for x in pool)
    meta = [fix[n].cuda() for n in ("pages", "lengths", "starts")]
    q = fix["q"].cuda()
    whole = torch.stack((k.view(torch.uint8), v.view(torch.uint8)), 1)
    heads = [bytes_as(x, lambda y: y.transpose(1, 2).contiguous().transpose(1, 2)) for x in (k, v)]
    fused = torch.cat((q, q[:, :2]), 1)[:, :4]
    off = torch.cat((q.new_zeros(1), q.flatten()))[1:].view(q.shape)
    for query, kv in ((q, (whole[:, 0].view(F.E4M3), whole[:, 1].view(F.E4M3))), (q, heads), (fused, (k, v)), (off, (k, v)),
                      (q.transpose(0, 1).contiguous().transpose(0, 1), (k, heads[1]))):
        C.check(bt.fp8_chunk_attention(query, kv[0], sk, kv[1], sv, *meta), want, tol)


def test_pool_past_32_bits():
    """Pages whose codes' byte offsets pass 32 bits."""
    import branchcraft_torch as bt
    hkv, d, pool = 64, 128, 40000  # 5.2e9 bytes each of K and V
    k, v = (torch.empty((pool, 16, hkv, d), device="cuda", dtype=torch.uint8).view(F.E4M3) for _ in range(2))
    sk, sv = (torch.empty((pool, hkv, 16, d // 32), device="cuda", dtype=torch.uint8).view(F.E8M0) for _ in range(2))
    g = torch.Generator("cuda").manual_seed(3)
    ids = torch.tensor([pool - 1, 5, pool - 7, 1, 16383, 16384, 32768], dtype=torch.int32, device="cuda")
    lengths = torch.tensor([40, 50], dtype=torch.int32, device="cuda")
    new = [torch.randn((90, hkv, d), generator=g, device="cuda").to(BF16) for _ in range(2)]
    pages, _, slots, _ = bt.build_tables(ids, lengths, lengths, 4, 90)
    bt.append_fp8_kv_(k, sk, v, sv, *new, slots)
    back = bt.read_fp8_kv(k, sk, v, sv, slots, BF16)
    held = [F.values(*F.to_fp8(x.cpu())) for x in new]
    for got, want in zip(back, held):
        assert torch.equal(got.cpu().double(), want)
    starts = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda")
    q = torch.randn((4, 64, d), generator=g, device="cuda").to(BF16)
    got = bt.fp8_chunk_attention(q, k, sk, v, sv, pages, lengths, starts)
    small = [torch.zeros((7, 16, hkv, d), dtype=BF16) for _ in range(2)]
    table = torch.tensor([[0, 1, 2, -1], [3, 4, 5, 6]], dtype=torch.int32)
    for x, want in zip(small, held):
        x[:3].view(-1, hkv, d)[:40] = want[:40].to(BF16)
        x[3:].view(-1, hkv, d)[:50] = want[40:].to(BF16)
    some = [0, 1, 62, 63]
    want, tol = C.reference(q[:, some].cpu(), *(x[:, :, some].contiguous() for x in small), table, lengths.cpu(), starts.cpu())
    C.check(got[:, some], want, tol)


def test_powers_past_32_bits():
    """One page of codes for all, and powers whose byte offsets pass 32 bits."""
    import branchcraft_torch as bt
    hkv, d, pool = 64, 128, 1100000  # 4.5e9 bytes of powers
    g = torch.Generator("cuda").manual_seed(4)
    codes, power = F.to_fp8(torch.randn((1, 16, hkv, d), generator=g, device="cuda").to(BF16).cpu())
    k = codes.cuda().view(torch.uint8).expand(pool, 16, hkv, d).view(F.E4M3)
    scale = torch.full((pool, hkv, 16, d // 32), 60, device="cuda", dtype=torch.uint8)
    ids = [pool - 1, 1048575, 1048576, 3]
    base = power.view(torch.uint8).transpose(1, 2)[0].cuda()
    for i, page in enumerate(ids):
        scale[page] = base + i % 2  # every other page twice the values
    scale = scale.view(F.E8M0)
    slots = (torch.tensor(ids, dtype=torch.int32, device="cuda")[:, None] * 16 + torch.arange(16, dtype=torch.int32, device="cuda")).flatten()
    want = F.values(codes[0], power[0])
    want = torch.cat([want * (1 + i % 2) for i in range(4)]).to(BF16)
    for got in bt.read_fp8_kv(k, scale, k, scale, slots, BF16):
        assert torch.equal(got.cpu(), want)
    q = torch.randn((1, hkv, d), generator=g, device="cuda").to(BF16)
    meta = [torch.tensor(x, dtype=torch.int32) for x in ([ids], [64], [0, 1])]
    got = bt.fp8_chunk_attention(q, k, scale, k, scale, *(x.cuda() for x in meta))
    some = [0, 31, 63]
    small = want.view(4, 16, hkv, d)[:, :, some].contiguous()
    meta[0] = torch.arange(4, dtype=torch.int32)[None]
    ref, tol = C.reference(q[:, some].cpu(), small, small, *meta)
    C.check(got[:, some], ref, tol)


def test_append_of_more_rows_than_a_launch_has_workgroups():
    """2^24 and more rows of 4 heads: several launches; all but a few are padding."""
    import branchcraft_torch as bt
    far = (1 << 27) + 50  # rows of eight threads each: past 2^24 workgroups in all, and past the first launch
    k, v = (rows(1, 1, 64, F16, s).cuda().expand(far, 1, 64) for s in (1, 2))
    pool = [torch.zeros(s, device="cuda", dtype=torch.uint8).view(t)
            for s, t in (((3, 16, 1, 64), F.E4M3), ((3, 1, 16, 2), F.E8M0)) * 2]
    slots = torch.full((far,), -1, device="cuda", dtype=torch.int32)
    at = torch.tensor([0, 5, far - 60, far - 2, far - 1], device="cuda")
    slots[at] = torch.arange(20, 25, device="cuda", dtype=torch.int32)
    bt.append_fp8_kv_(*pool, k, v, slots)
    for x, codes, scale in ((k, *pool[:2]), (v, *pool[2:])):
        c, s = F.to_fp8(x[:1].cpu())
        flat, powers = raw(codes).view(-1, 1, 64).cpu(), raw(scale)[:, 0].reshape(-1, 2).cpu()
        same = (c.view(torch.uint8) & 0x7f) != 0x7f
        assert torch.equal((flat[20:25] * same), (c.view(torch.uint8) * same).expand(5, 1, 64))
        assert torch.equal(powers[20:25], s.view(torch.uint8)[:, 0].expand(5, 2))
        assert not flat[:20].any() and not flat[25:].any() and not powers[:20].any() and not powers[25:].any()


def test_captured_steps_follow_the_lengths():
    """A whole step captured and replayed while lengths, tables and rows change in
    place, with eager calls between; every replay equals the eager call."""
    import branchcraft_torch as bt
    hq, hkv, d, batch, width = 8, 2, 64, 3, 130
    g = torch.Generator("cuda").manual_seed(6)
    pool = batch * width + 1
    cache = [torch.zeros(s, device="cuda", dtype=torch.uint8).view(t)
             for s, t in (((pool, 16, hkv, d), F.E4M3), ((pool, hkv, 16, d // 32), F.E8M0)) * 2]
    ids = torch.randperm(pool, generator=g, device="cuda")[:batch * width].to(torch.int32)
    lengths = torch.tensor([1, 1900, 40], dtype=torch.int32, device="cuda")
    counts = torch.ones(batch, dtype=torch.int32, device="cuda")
    held = torch.empty(batch * width, dtype=torch.int32, device="cuda")
    q = torch.zeros((5, hq, d), device="cuda", dtype=F16)
    nk, nv = (torch.zeros((5, hkv, d), device="cuda", dtype=F16) for _ in range(2))

    def set_step(n):
        lengths.copy_(torch.tensor([n, 1900 + n, 40 + 3 * n], dtype=torch.int32))
        counts.copy_(torch.tensor([1, 2, 1] if n % 2 else [1, 1, 1], dtype=torch.int32))
        at = 0
        for b, m in enumerate(lengths.tolist()):
            c = C.pages_of(m)
            held[at:at + c] = ids[b * width:b * width + c]
            at += c
        for x in (q, nk, nv):
            x.copy_(torch.randn(x.shape, generator=g, device="cuda"))

    def step():
        pages, starts, slots, _ = bt.build_tables(held, lengths, counts, width, 5)
        bt.append_fp8_kv_(*cache, nk, nv, slots)
        return bt.fp8_chunk_attention(q, *cache, pages, lengths, starts), *bt.read_fp8_kv(*cache, slots, F16)

    set_step(1)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(1, 6):
        set_step(n)
        want = [x.clone() for x in step()]
        torch.cuda.synchronize()
        for x in out:
            x.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n
        assert not out[0][int(counts.sum()):].any() and not out[1][int(counts.sum()):].any()


def test_two_streams_at_once_and_the_same_bits():
    import branchcraft_torch as bt
    args = []
    for s in (20, 21):
        fix = C.batch([2100, 900, 50], [3, 40, 50], 8, 2, 128, F16, seed=s)
        pool, _ = F.pools(fix)
        args.append([fix["q"].cuda(), *(x.cuda() for x in pool), *(fix[n].cuda() for n in ("pages", "lengths", "starts"))])
    want = [bt.fp8_chunk_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(bt.fp8_chunk_attention(*args[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


@pytest.mark.parametrize("shape", [([40, 3], [35, 1]), ([1100, 70], [34, 2])], ids=["short", "split"])
def test_many_kv_heads_and_wide_groups(shape):
    for heads, d, dtype in (((73, 73), 64, F16), ((129, 1), 128, BF16)):
        fix = C.batch(*shape, *heads, d, dtype, seed=30)
        pool, same = F.pools(fix)
        want, tol = C.reference(**same, window=30)
        C.check(attend(fix, pool, window=30), want, tol)


def test_lengths_past_the_table_and_rows_before_the_request():
    fix = C.batch([100, 3, 60], [5, 3, 60], 4, 2, 64, F16, seed=7)
    fix["pages"] = fix["pages"][:, :4].contiguous()
    fix["lengths"] = torch.tensor([100, 1, -5], dtype=torch.int32)
    pool, same = F.pools(fix)
    want, tol = C.reference(**same)
    C.check(attend(fix, pool), want, tol)


def test_an_empty_pool_is_zeros():
    """Codes and powers of zero bytes: scores of zero, outputs of zero."""
    fix = C.batch([70], [3], 4, 2, 64, BF16, seed=1)
    zero = [torch.zeros_like(x.view(torch.uint8)).view(x.dtype) for x in F.pools(fix)[0]]
    assert not attend(fix, zero).any()


def test_dispatcher_checks_and_compile():
    import branchcraft_torch as bt
    fix = C.batch([90, 40], [3, 40], 4, 2, 64, F16, seed=23)
    pool = [x.cuda() for x in F.pools(fix)[0]]
    args = (fix["q"].cuda(), *pool, *(fix[n].cuda() for n in ("pages", "lengths", "starts")))
    whole = torch.compile(lambda *a: bt.fp8_chunk_attention(*a, window=9) * 2, fullgraph=True)
    assert torch.equal(whole(*args), bt.fp8_chunk_attention(*args, window=9) * 2)
    slots = torch.arange(5, dtype=torch.int32, device="cuda")
    both = torch.compile(lambda *a: bt.read_fp8_kv(*a, F16), fullgraph=True)
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num())
               for a, b in zip(both(*pool, slots), bt.read_fp8_kv(*pool, slots, F16)))


def _case():
    fix = C.batch([90, 40], [3, 4], 4, 2, 64, F16, seed=24)
    pool = [x.cuda() for x in F.pools(fix)[0]]
    return dict(q=fix["q"].cuda(), k=pool[0], sk=pool[1], v=pool[2], sv=pool[3],
                **{n: fix[n].cuda() for n in ("pages", "lengths", "starts")})


REFUSALS = {
    "k type": dict(k=lambda x: x.half()), "k bytes": dict(k=lambda x: x.view(torch.uint8)),
    "scale type": dict(sk=lambda x: x.view(torch.uint8)), "scale shape": dict(sv=lambda x: bytes_scale(x, lambda y: y[:, :1])),
    "scale order": dict(sk=lambda x: bytes_scale(x, lambda y: y.transpose(1, 2))),
    "scale strides": dict(sk=lambda x: bytes_scale(x, lambda y: torch.stack((y, y), -1)[..., 0])),
    "host scale": dict(sk=lambda x: x.cpu()), "v shape": dict(v=lambda x: x[:-1]),
    "unaligned": dict(k=lambda x: bytes_as(x, lambda y: torch.cat((y.flatten()[:8], y.flatten()))[8:].view(y.shape))),
    "odd strides": dict(k=lambda x: bytes_as(x, lambda y: torch.cat((y, y[..., :8]), -1)[..., :64])),
    "page size": dict(k=lambda x: bytes_as(x, lambda y: y[:, :8])), "q type": dict(q=lambda x: x.float()),
    "head dim": dict(q=lambda x: x[..., :32].contiguous()), "heads": dict(q=lambda x: x[:, :3]),
    "starts": dict(starts=lambda x: x[:-1]), "table type": dict(pages=lambda x: x.long()),
}


def bytes_scale(x, change):
    return change(x.view(torch.uint8)).view(F.E8M0)


@pytest.mark.parametrize("what", [*REFUSALS, "scale", "window", "cap", "prefix without causal"])
def test_refusals(what):
    import branchcraft_torch as bt
    case, options = _case(), {}
    for name, change in REFUSALS.get(what, {}).items():
        case[name] = change(case[name])
    if what not in REFUSALS:
        options = {"scale": dict(scale=0.0), "window": dict(window=-1), "cap": dict(cap=-1.0),
                   "prefix without causal": dict(causal=False, prefix=torch.zeros(2, dtype=torch.int32).cuda())}[what]
    with pytest.raises((RuntimeError, NotImplementedError)):
        bt.fp8_chunk_attention(*(case[n] for n in ("q", "k", "sk", "v", "sv", "pages", "lengths", "starts")), **options)


def test_row_refusals():
    import branchcraft_torch as bt
    case = _case()
    pool = [case[n] for n in ("k", "sk", "v", "sv")]
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    r = torch.zeros((3, 2, 64), dtype=F16, device="cuda")
    bt.append_fp8_kv_(*pool, r, r, slots)
    bad = [(*pool, r, r.bfloat16(), slots), (*pool, r, r, slots[:2]), (*pool, r, r, slots.long()), (*pool, r[:, :1], r[:, :1], slots),
           (*pool, r.float(), r.float(), slots), (pool[0], pool[1], pool[0], pool[3], r, r, slots),
           (pool[0], pool[1], pool[2], pool[1], r, r, slots), (pool[0].half(), *pool[1:], r, r, slots),
           (pool[0], pool[1].view(torch.uint8), *pool[2:], r, r, slots), (pool[0][:-1], *pool[1:], r, r, slots),
           (*pool, r[..., ::2], r[..., ::2], slots), (*pool, r.cpu(), r, slots)]
    for args in bad:
        with pytest.raises((RuntimeError, NotImplementedError)):
            bt.append_fp8_kv_(*args)
    for args in [(*pool, slots.long(), F16), (*pool, slots, torch.float32), (*pool, slots[None], F16),
                 (pool[0].half(), *pool[1:], slots, F16), (pool[0], pool[1][:-1], *pool[2:], slots, F16)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            bt.read_fp8_kv(*args)
    for args in [(*pool, slots, slots[:2]), (*pool, slots.long(), slots), (*pool, slots, slots.cpu()), (*pool, slots[None], slots[None]),
                 (pool[0], pool[1], pool[0], pool[3], slots, slots), (pool[0].half(), *pool[1:], slots, slots)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            bt.copy_fp8_pages_(*args)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_a_cache_in_8_bits(dtype):
    """Prompts, forks, turns and a rollback: rows and attention as of the values that
    the rows were rounded to, pages shared until they are written."""
    from branchcraft_torch.transaction import Fp8Cache
    g = torch.Generator("cuda").manual_seed(4)

    def rand(n, heads):
        return torch.randn((n, heads, 64), generator=g, device="cuda").to(dtype)

    def held(x):
        return F.values(*F.to_fp8(x.cpu())).to(dtype)

    cache = Fp8Cache(40, 2, 64, dtype)
    kv = {}
    prompt = rand(37, 2), rand(37, 2)
    a = cache.new(*prompt)
    kv[a] = [held(x) for x in prompt]
    empty = cache.new(rand(0, 2), rand(0, 2))
    kv[empty] = [held(rand(0, 2)) for _ in range(2)]
    b = cache.fork(a)
    kv[b] = [x.clone() for x in kv[a]]
    shot = cache.checkpoint(b)
    for turn, counts in enumerate(([3, 20, 5], [1, 1, 1], [0, 30, 2])):
        who = [a, b, empty]
        total = sum(counts)
        q, k, v = rand(total, 4), rand(total, 2), rand(total, 2)
        got = cache.extend(who, counts, q, k, v, **({"cap": 9.0} if turn == 1 else {}))
        at = 0
        for x, n in zip(who, counts):
            kv[x] = [torch.cat((old, held(new[at:at + n]))) for old, new in zip(kv[x], (k, v))]
            at += n
        for x in who:
            for have, want in zip(cache.read(x), kv[x]):
                assert torch.equal(have.cpu(), want)
        lengths = [cache.lengths[x] for x in who]
        width = max(C.pages_of(n) for n in lengths)
        table = torch.full((3, width), -1, dtype=torch.int32)
        pools = [torch.zeros((3 * width, 16, 2, 64), dtype=dtype) for _ in range(2)]
        for i, (x, n) in enumerate(zip(who, lengths)):
            table[i, :C.pages_of(n)] = torch.arange(i * width, i * width + C.pages_of(n))
            for pool, rows_ in zip(pools, kv[x]):
                pool[i * width:(i + 1) * width].view(-1, 2, 64)[:n] = rows_
        starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
        want, tol = C.reference(q.cpu(), *pools, table, torch.tensor(lengths, dtype=torch.int32), starts,
                                cap=9.0 if turn == 1 else 0.0)
        C.check(got, want, tol)
        cache.owner.check_invariants()
    cache.rollback(shot)
    for have, want in zip(cache.read(b), (held(x) for x in prompt)):
        assert torch.equal(have.cpu(), want)
    if dtype == F16:  # what it holds enters a 16-bit pool for trees
        from branchcraft_torch.transaction import PagedTreeCache
        wide = PagedTreeCache(8, 2, 64)
        c = wide.new(*cache.read(a))
        flat = wide.k[wide.pages[c]].view(-1, 2, 64)[:wide.lengths[c]]
        assert torch.equal(flat.cpu(), kv[a][0])
    before = ({x: list(p) for x, p in cache.pages.items()}, list(cache.free))
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.extend([a], [700], rand(700, 4), rand(700, 2), rand(700, 2))
    with pytest.raises(RuntimeError, match="exhausted"):
        cache.new(rand(700, 2), rand(700, 2))
    assert ({x: list(p) for x, p in cache.pages.items()}, list(cache.free)) == before
