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


# ---------------------------------------------------------------------------
# Shared pages read once


def attend(fix, groups, shared, **options):
    """The call where only the first member of each group has the shared pages: the
    others' tables name a page of NaN in their place, which a call that reads each
    request's own pages would meet."""
    import branchcraft_torch as bt
    spare = min({*range(fix["k"].shape[0])} - {*fix["pages"].flatten().tolist()})
    table = fix["pages"].clone()
    for a, b, n in zip(groups.tolist(), groups.tolist()[1:], shared.tolist()):
        table[a + 1:b, :n // C.PAGE] = spare
    dev = C.on_gpu(fix | dict(pages=table))
    dev["k"][spare] = dev["v"][spare] = float("nan")
    options = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in options.items()}
    return bt.shared_chunk_attention(dev["q"], dev["k"], dev["v"], dev["pages"], dev["lengths"], dev["starts"],
                                     groups.cuda(), shared.cuda(), **options)


# Groups of up to 32 rows (query heads per KV head times new tokens), of a few more and
# of more than a tile; what they share is shorter and longer than a window, and
# members' lengths differ by more than one, so that of some all of it is out of sight.
SIZES = [(2, 900), (3, 1500), (8, 333), (9, 700), (16, 64), (17, 1300), (31, 650)]
LAYOUTS = {
    "64 over 32, D = 64": (64, 32, 64, BF16, 600),
    "32 over 8, D = 128": (32, 8, 128, F16, 1200),
}
FORMS = {
    "window": {}, "bias": dict(slopes=True), "cap": dict(cap=4.0), "full": dict(causal=False),
    "prefix bias": dict(prefix=True, slopes=True), "documents": dict(first=True),
}
_made = {}


def windows_of(layout):
    if layout not in _made:
        hq, hkv, d, dtype, window = LAYOUTS[layout]
        groups, i = [], 0
        for members, n in SIZES:
            own = [(2 + 37 * j * j % (window + 300), 1 + (j % 5 == 4)) for j in range(i, i + members)]
            groups.append((n, own))
            i += members
        _made.clear()
        _made[layout] = (*F.forks(groups, hq, hkv, d, dtype, seed=11), window)
    return _made[layout]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("layout", LAYOUTS)
def test_windows_over_shared_pages(layout, form):
    fix, groups, shared, window = windows_of(layout)
    rows = fix["starts"][groups[1:].long()] - fix["starts"][groups[:-1].long()]
    rows = rows * (fix["q"].shape[1] // fix["k"].shape[2])
    assert rows.min() <= 32 < rows.max() and window < fix["pages"].shape[1] * C.PAGE
    lengths = fix["lengths"]
    assert any(int(lengths[a:b].max() - lengths[a:b].min()) > window for a, b in zip(groups, groups[1:]))
    assert F.pays(fix, window)
    options = dict(FORMS[form], window=window)
    g = torch.Generator().manual_seed(5)
    if "slopes" in options:
        options["slopes"] = (torch.rand(fix["q"].shape[1], generator=g) - 0.25) / 16
    if "prefix" in options:  # from none to more than the request holds
        options["prefix"] = torch.tensor([int(torch.randint(-1, int(n) + 20, (1,), generator=g)) for n in lengths],
                                         dtype=torch.int32)
    if "first" in options:  # from before the request to past it: rows that see nothing
        options["first"] = torch.tensor([int(torch.randint(-3, int(n) + 3, (1,), generator=g))
                                         for n, c in zip(lengths, fix["starts"].diff()) for _ in range(int(c))],
                                        dtype=torch.int32)
    want, tol = C.reference(**fix, **options)
    C.check(attend(fix, groups, shared, **options), want, tol, form)


def test_a_tile_under_a_window_in_several_parts():
    """One group of two tiles and little else to fill the card with, of which a tile's
    27 steps of 64 tokens are cut into parts of four."""
    fix, groups, shared = F.forks([(1700, [(1 + i % 7, 1) for i in range(64)])], 32, 8, 128, BF16, seed=12)
    window = 1600
    assert fix["pages"].shape[1] * C.PAGE > window and F.pays(fix, window)
    want, tol = C.reference(**fix, window=window)
    C.check(attend(fix, groups, shared, window=window), want, tol)


# ---------------------------------------------------------------------------
# The join where a wave has several rows of a token, and several tokens


def by_rows(fix):
    """C.reference of the causal form, all heads of a row at once."""
    q, k, v, pages, lengths, starts = (fix[n] for n in ("q", "k", "v", "pages", "lengths", "starts"))
    t, hq, d = q.shape
    hkv = k.shape[2]
    scale, u = d ** -0.5, torch.finfo(q.dtype).eps / 2
    out = torch.zeros((t, hq, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b, n in enumerate(lengths.tolist()):
        ids = pages[b, :C.pages_of(n)].long()
        kk, vv = (x[ids].flatten(0, 1)[:n].double().transpose(0, 1) for x in (k, v))  # [Hkv, n, D]
        lo, hi = starts[b:b + 2].tolist()
        for row in range(lo, hi):
            p = n - (hi - row) + 1
            qq = q[row].double().view(hkv, -1, d)
            keys, values = kk[:, :p].transpose(1, 2), vv[:, :p]
            w = torch.softmax(scale * (qq @ keys), -1)
            size = scale * (qq.abs() @ keys.abs()).amax(-1, keepdim=True)
            e = 2.0 ** -24 * (d + 4 * 16) * size.clamp(min=1.0)
            o, mean = w @ values, w @ values.abs()
            out[row] = o.reshape(hq, d)
            tol[row] = (u * o.abs() + (u + 2 * e) * mean + p * 2.0 ** -32 * values.abs().max()
                        + 2.0 ** -24).reshape(hq, d)
    return out, tol


@pytest.mark.parametrize("hq,hkv,d,dtype,members,new", [
    (28, 4, 64, BF16, 40, 11), (32, 8, 128, F16, 300, 1), (2560, 64, 64, F16, 130, 1), (264, 8, 128, BF16, 70, 2)])
def test_more_rows_than_the_join_has_waves(hq, hkv, d, dtype, members, new):
    fix, groups, shared = F.forks([(96, [(new + i % 40, new) for i in range(members - 30)]),
                                   (40, [(new + i % 9, new) for i in range(30)])], hq, hkv, d, dtype, seed=13)
    waves = 4 * 8 * torch.cuda.get_device_properties(0).multi_processor_count
    pairs = fix["q"].shape[0] * hkv
    assert F.pays(fix) and pairs * hq // hkv > waves  # fewer waves than rows
    want, tol = by_rows(fix)
    C.check(attend(fix, groups, shared), want, tol)


def test_the_two_references_agree():
    fix, _, _ = F.forks([(64, [(1 + i, 1 + i % 3) for i in range(5)])], 4, 2, 64, F16, seed=14)
    for x, y in zip(by_rows(fix), C.reference(**fix)):
        assert torch.allclose(x, y, rtol=1e-12, atol=1e-15)


# ---------------------------------------------------------------------------
# Whole calls


@pytest.mark.parametrize("window", [0, 3000])
def test_extend_over_forks_beside_others(window):
    """A chat, forks of a document and forks of a short note, all behind one system
    prompt; the note itself has no new tokens."""
    from branchcraft_torch.transaction import PagedTreeCache
    g = torch.Generator("cuda").manual_seed(8)
    hq, hkv, d = 32, 16, 64

    def rand(n, heads):
        return torch.randn((n, heads, d), generator=g, device="cuda", dtype=F16)

    cache = PagedTreeCache(1000, hkv, d)
    root = cache.new(rand(32, hkv), rand(32, hkv))

    def grow(x, n):
        cache.extend([x], [n], rand(n, hq), rand(n, hkv), rand(n, hkv))
        return x

    chat, document, note = (grow(cache.fork(root), n) for n in (700, 3800, 150))
    who = [chat, document] + [cache.fork(document) for _ in range(30)] + [note, cache.fork(note)]
    for turn in range(2):
        counts = [3] + [1, 2] * 15 + [1, 0] + [1]
        total = sum(counts)
        q, k, v = rand(total, hq), rand(total, hkv), rand(total, hkv)
        got = cache.extend(who, counts, q, k, v, share=True, window=window)
        lists = [cache.pages[x] for x in who]
        table = torch.full((len(who), max(map(len, lists))), -1, dtype=torch.int32)
        for i, pages in enumerate(lists):
            table[i, :len(pages)] = torch.tensor(pages)
        starts = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32)
        fix = dict(q=q.cpu(), k=cache.k.cpu(), v=cache.v.cpu(), pages=table, starts=starts,
                   lengths=torch.tensor([cache.lengths[x] for x in who], dtype=torch.int32))
        assert F.pays(fix, window)
        bounds, tokens = cache.owner.shared_prefixes(who)
        assert bounds == [0, 1, 32, 34] and tokens[1] == 3832 // 16 * 16
        want, tol = C.reference(**fix, window=window)
        C.check(got, want, tol)
