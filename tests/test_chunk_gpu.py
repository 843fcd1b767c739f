"""chunk_attention against its definition in 64 bits, at the sizes, masks and
layouts where it can go wrong.  Slots of the pool that hold no token are NaN
throughout."""

import pytest
import torch

import chunk_helpers as C

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def run(fix, **options):
    import branchcraft_torch as bt
    dev = C.on_gpu(fix)
    options = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in options.items()}
    out = bt.chunk_attention(dev["q"], dev["k"], dev["v"], dev["pages"], dev["lengths"],
                             dev["starts"], **options)
    torch.cuda.synchronize()
    assert out.dtype == fix["q"].dtype and out.is_contiguous()
    return out


def both(fix, what="", **options):
    want, tol = C.reference(**fix, **options)
    got = run(fix, **options)
    C.check(got, want, tol, what)
    return got


# One token, edges of a page (16), of a tile (32), of a step (64, 128), of a
# tile of rows; requests without new tokens or without any.
SHAPES = [
    ([1], [1]),
    ([512], [1]),
    ([15, 16, 17, 1], [1, 1, 1, 1]),
    ([31, 32, 33, 63, 64, 65], [1, 2, 3, 4, 8, 9]),
    ([127, 128, 129, 255, 257], [1, 1, 33, 255, 1]),
    ([64, 64], [64, 0]),
    ([0, 40, 0, 7], [0, 5, 0, 7]),
    ([200], [200]),
    ([333, 1, 90], [130, 1, 17]),
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (7, 1, 64), (4, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_causal(shape, hq, hkv, d, dtype):
    lengths, counts = SHAPES[shape]
    both(C.batch(lengths, counts, hq, hkv, d, dtype, seed=shape))


FORMS = {
    "full": dict(causal=False),
    "window 1": dict(window=1),
    "window 50": dict(window=50),
    "window 500": dict(window=500),
    "cap": dict(cap=3.0),
    "cap window": dict(cap=30.0, window=70),
    "cap 256": dict(cap=256.0),
    "cap 300": dict(cap=300.0),
    "cap 1e6 bias": dict(cap=1e6, slopes=True),
    "cap 1e-3": dict(cap=1e-3),
    "bias": dict(slopes=True),
    "bias full": dict(slopes=True, causal=False),
    "window full": dict(window=33, causal=False),
    "cap bias": dict(slopes=True, cap=5.0),
    "prefix": dict(prefix=True),
    "prefix bias window": dict(prefix=True, slopes=True, window=40),
    "first": dict(first=True),
    "first cap full": dict(first=True, cap=8.0, causal=False),
    "scale": dict(scale=0.5),
}


def options_of(form, fix, seed=5):
    options = dict(FORMS[form])
    g = torch.Generator().manual_seed(seed)
    lengths, counts = fix["lengths"], fix["starts"].diff()
    if "slopes" in options:
        options["slopes"] = torch.rand(fix["q"].shape[1], generator=g) - 0.25
    if "prefix" in options:  # from none to more than the request holds
        options["prefix"] = torch.tensor(
            [int(torch.randint(-1, int(n) + 20, (1,), generator=g)) for n in lengths],
            dtype=torch.int32)
    if "first" in options:  # from before the request to past it: rows that see nothing
        options["first"] = torch.tensor(
            [int(torch.randint(-3, int(n) + 3, (1,), generator=g))
             for n, c in zip(lengths, counts) for _ in range(int(c))], dtype=torch.int32)
    return options


@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 8, 2, 128), (BF16, 6, 2, 64)])
@pytest.mark.parametrize("shape", [([333, 1, 90, 64], [130, 1, 17, 40]), ([700], [1]), ([150], [150])])
@pytest.mark.parametrize("form", FORMS)
def test_forms(form, shape, dtype, hq, hkv, d):
    fix = C.batch(*shape, hq, hkv, d, dtype, seed=len(form))
    both(fix, form, **options_of(form, fix))


@pytest.mark.parametrize("form", ["scale", "window 500", "cap bias"])
def test_long_and_split(form):
    """A few rows over a long table: split over workgroups, pages in any order."""
    fix = C.batch([5000, 3, 4111], [2, 1, 9], 4, 1, 128, BF16, seed=3)
    both(fix, form, **options_of(form, fix))


def test_sharp_scores():
    """Scores far apart: the running maximum moves by much in every tile."""
    fix = C.batch([400, 300], [70, 1], 8, 2, 128, F16, seed=9, spread=12.0)
    both(fix)
    both(fix, cap=20.0)


def test_pages_outside_the_pool_are_not_seen():
    fix = C.batch([200, 90], [70, 1], 8, 2, 128, F16, seed=4)
    fix["pages"][0, 3] = -1
    fix["pages"][0, 9] = fix["k"].shape[0]
    fix["pages"][1, 0] = 2**31 - 1
    fix["pages"][1, 1:] = -7
    got = both(fix)
    assert not got[70].any()  # nothing seen
    both(fix, causal=False)


def test_lengths_past_the_table_and_rows_before_the_request():
    """A table of three pages under a length of 60; more new rows than tokens."""
    fix = C.batch([48, 5], [10, 9], 4, 2, 64, F16, seed=6, extra_cols=0)
    fix["lengths"][0] = 60
    got = both(fix)
    assert not got[10:14].any()
    fix["lengths"] = torch.tensor([-3, 2**31 - 1], dtype=torch.int32)
    got = run(fix)
    assert not got[:10].any()


def test_rows_of_no_request_are_zero():
    fix = C.batch([70, 20], [33, 5], 8, 2, 128, BF16, seed=7)
    g = torch.Generator().manual_seed(1)
    q = torch.randn((400, 8, 128), generator=g).to(BF16)
    q[2:40] = fix["q"]
    fix["q"], fix["starts"] = q, fix["starts"] + 2
    got = both(fix)
    assert not got[:2].any() and not got[40:].any()


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_row_does_not_see_stays_out(bad, dtype):
    """NaN and infinities in the K and V of later tokens, of another document
    and before the window: rows that do not see them are as without them."""
    for n, new in ((200, 140), (90, 3)):
        fix = C.batch([n], [new], 8, 2, 128, dtype, seed=8)
        clean = {name: x.clone() for name, x in fix.items()}
        at = n - new // 2 - 1  # a token in the middle of the new ones
        page, slot = int(fix["pages"][0, at // 16]), at % 16
        fix["k"][page, slot], fix["v"][page, slot, :, ::3] = bad, bad
        rows = torch.arange(n - new, n)
        for options, blind in ((dict(), rows < at),
                               (dict(window=2), (rows < at) | (rows >= at + 2)),
                               (dict(first=rows.int()), rows != at)):
            got, want = run(fix, **options), run(clean, **options)
            assert torch.equal(got[blind.cuda()], want[blind.cuda()])
            assert bool((got[~blind.cuda()] != want[~blind.cuda()]).any(-1).any(-1).all())


def layouts(fix):
    """The same pools in other places: heads before slots, the halves of a
    packed cache, rows with padding, one element off alignment."""
    k, v = fix["k"].cuda(), fix["v"].cuda()
    p, s, h, d = k.shape
    yield "heads first", [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v)]
    both = torch.stack((k, v), 1)
    yield "packed blocks", [both[:, 0], both[:, 1]]
    rows = torch.cat((k, v), -1)
    yield "packed rows", [rows[..., :d], rows[..., d:]]
    rows = torch.cat((k, v, k[..., :3]), -1)
    yield "odd rows", [rows[..., :d], rows[..., d:2 * d]]
    flat = [torch.empty(x.numel() + 1, device="cuda", dtype=x.dtype)[1:].view(x.shape).copy_(x)
            for x in (k, v)]
    yield "one off", flat
    yield "one of two off", [k, flat[1]]


@pytest.mark.parametrize("dtype,d", [(F16, 128), (BF16, 64)])
def test_layouts(dtype, d):
    import branchcraft_torch as bt
    fix = C.batch([150, 33, 290], [70, 1, 12], 8, 2, d, dtype, seed=11)
    want, tol = C.reference(**fix)
    dev = C.on_gpu(fix)
    meta = [dev[n] for n in ("pages", "lengths", "starts")]
    for name, (k, v) in layouts(fix):
        C.check(bt.chunk_attention(dev["q"], k, v, *meta), want, tol, name)
    t, hq = fix["q"].shape[:2]
    fused = torch.cat((dev["q"], dev["q"][:, :4] + 1), 1)
    C.check(bt.chunk_attention(fused[:, :hq], dev["k"], dev["v"], *meta), want, tol, "fused q")
    turned = dev["q"].transpose(0, 1).contiguous().transpose(0, 1)
    C.check(bt.chunk_attention(turned, dev["k"], dev["v"], *meta), want, tol, "q heads first")
    odd = torch.cat((dev["q"], dev["q"][..., :1]), -1)[..., :d]
    C.check(bt.chunk_attention(odd, dev["k"], dev["v"], *meta), want, tol, "q odd rows")


def test_long_documents_window_and_few_rows():
    """Ranges of the narrow form that start inside a request: behind a window,
    at a document's start, over many requests of one token or none."""
    g = torch.Generator().manual_seed(12)
    lengths = [int(x) for x in torch.randint(0, 2500, (70,), generator=g)]
    counts = [int(torch.randint(0, 4, (1,), generator=g)) for _ in lengths]
    fix = C.batch(lengths, counts, 2, 1, 64, BF16, seed=13)
    both(fix, "causal")
    both(fix, "window", window=700)
    first = torch.tensor([int(torch.randint(0, max(n, 1), (1,), generator=g))
                          for n, c in zip(lengths, counts) for _ in range(c)], dtype=torch.int32)
    both(fix, "documents", first=first)


def test_mixed_batch_with_every_form_of_work():
    """Whole tiles, split tiles and ranges in one call: chunks of several
    lengths among single tokens, and a request that only waits."""
    fix = C.batch([1500, 1300, 40, 1100, 9, 1200], [70, 1, 40, 3, 0, 300], 4, 2, 128, F16, seed=14)
    both(fix)
    both(fix, cap=5.0)
    both(fix, slopes=torch.tensor([0.5, 0.1, -0.01, 0.02]))


def test_workspace_refused_or_short_gives_the_same():
    """The C entry without a workspace, with a short one and with one that is
    not aligned: unsplit, and as exact."""
    import branchcraft_capi as capi
    import gpu_helpers as G
    fix = C.batch([3000, 2000], [2, 140], 4, 2, 128, F16, seed=15)
    want, tol = C.reference(**fix)
    dev = C.on_gpu(fix)
    (t, hq, d), (pool, _, hkv, _) = dev["q"].shape, dev["k"].shape
    shape = capi.Shape(2, hq, hkv, d, dev["pages"].shape[1], pool)
    need = G.lib().bc_chunk_attention_workspace_size(shape, t)
    assert need > 0
    ws = torch.empty(need + 16, device="cuda", dtype=torch.uint8)
    strides = capi.PoolStrides(16 * hkv * d, hkv * d, d)
    for at, size in ((None, 0), (ws.data_ptr(), need - 1), (ws.data_ptr() + 4, need), (ws.data_ptr(), need)):
        out = torch.full_like(dev["q"], float("nan"))
        ins = capi.ChunkInputs(*(dev[n].data_ptr() for n in ("q", "k", "v", "pages", "lengths", "starts")),
                               None, None, None, out.data_ptr(), capi.RowStrides(hq * d, d), strides, strides,
                               t, capi.BC_FLOAT16, 1, 0, d ** -0.5, 0.0)
        G.check(G.lib().bc_chunk_attention(shape, ins, at, size, G.stream()), "bc_chunk_attention")
        C.check(out, want, tol, f"workspace {size}")


def test_pool_past_32_bits():
    """Pages whose byte and element offsets pass 32 bits."""
    import branchcraft_torch as bt
    hkv, d, pool = 8, 128, 270000  # 4.4e9 elements, 8.8 GB each of K and V
    g = torch.Generator("cuda").manual_seed(3)
    k, v = (torch.empty((pool, 16, hkv, d), device="cuda", dtype=BF16) for _ in range(2))
    ids = [pool - 1, 5, pool - 7, 131071, 131072, 262143]
    lengths, counts = [40, 50], [40, 2]
    rows = [torch.randn((90, hkv, d), generator=g, device="cuda").to(BF16) for _ in range(2)]
    meta = [torch.tensor(x, dtype=torch.int32, device="cuda") for x in (ids[:3] + ids[2:6], lengths, lengths)]
    meta[0][3:] = torch.tensor([1, 131071, 131072, 262143], dtype=torch.int32)
    pages, _, slots, _ = bt.build_tables(*meta, 4, 90)
    bt.append_kv_(k, v, *rows, slots)
    starts = torch.tensor([0, 40, 42], dtype=torch.int32, device="cuda")
    q = torch.randn((42, 16, d), generator=g, device="cuda").to(BF16)
    got = bt.chunk_attention(q, k, v, pages, meta[1], starts)
    small = torch.arange(7, dtype=torch.int32)
    order = pages.cpu()[pages.cpu() >= 0].long()
    table = torch.full((2, 4), -1, dtype=torch.int32)
    table[0, :3], table[1, :4] = small[:3], small[3:]
    want, tol = C.reference(q.cpu(), k[order.cuda()].cpu(), v[order.cuda()].cpu(), table,
                            meta[1].cpu(), starts.cpu())
    C.check(got, want, tol)


def test_captured_steps_follow_the_lengths():
    """A whole step captured once and replayed while lengths, tables and
    inputs change in place, with eager calls between the replays; two graphs
    of the same buffers in turn; every replay equals the eager call."""
    import branchcraft_torch as bt
    hq, hkv, d, batch, width = 8, 2, 64, 3, 130
    g = torch.Generator("cuda").manual_seed(6)
    pool = batch * width + 1
    k, v = (torch.zeros((pool, 16, hkv, d), device="cuda", dtype=F16) for _ in range(2))
    ids = torch.randperm(pool, generator=g, device="cuda")[:batch * width].to(torch.int32)
    lengths = torch.tensor([1, 1900, 40], dtype=torch.int32, device="cuda")
    counts = torch.ones(batch, dtype=torch.int32, device="cuda")
    held = torch.empty(batch * width, dtype=torch.int32, device="cuda")
    q = torch.zeros((5, hq, d), device="cuda", dtype=F16)  # two rows of padding
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

    def step(window):
        pages, starts, slots, positions = bt.build_tables(held, lengths, counts, width, 5)
        bt.append_kv_(k, v, nk, nv, slots)
        return bt.chunk_attention(q, k, v, pages, lengths, starts, window=window), positions

    set_step(1)
    step(0)  # warm
    graphs = []
    for window in (0, 300):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(window)
        graphs.append((graph, out, window))
    for n in range(1, 7):
        set_step(n)
        for graph, out, window in graphs:
            want = [x.clone() for x in step(window)]
            torch.cuda.synchronize()
            for x in out:
                x.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (n, window)
            assert not out[0][int(counts.sum()):].any()


def test_two_streams_at_once():
    import branchcraft_torch as bt
    fixes = [C.on_gpu(C.batch([2100, 900, 50], [3, 40, 50], 8, 2, 128, F16, seed=s)) for s in (20, 21)]
    args = [[f[n] for n in ("q", "k", "v", "pages", "lengths", "starts")] for f in fixes]
    want = [bt.chunk_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(bt.chunk_attention(*args[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_same_inputs_give_the_same_bits():
    fix = C.batch([2500, 700, 90], [5, 300, 1], 8, 2, 128, BF16, seed=22)
    first = run(fix)
    for _ in range(5):
        assert torch.equal(run(fix), first)


def test_dispatcher_checks_and_compile():
    import branchcraft_torch as bt
    dev = C.on_gpu(C.batch([90, 40], [3, 40], 4, 2, 64, F16, seed=23))
    args = tuple(dev[n] for n in ("q", "k", "v", "pages", "lengths", "starts"))
    torch.library.opcheck(torch.ops.branchcraft.chunk_attention, args, dict(cap=3.0))
    ints = (torch.arange(9, dtype=torch.int32, device="cuda"), dev["lengths"], dev["lengths"])
    torch.library.opcheck(torch.ops.branchcraft.build_tables, (*ints, 7, 130))
    k, v = dev["k"].nan_to_num(), dev["v"].nan_to_num()
    slots = torch.arange(5, dtype=torch.int32, device="cuda")
    torch.library.opcheck(torch.ops.branchcraft.append_kv_, (k, v, k[0, :5].clone(), v[0, :5].clone(), slots))
    whole = torch.compile(lambda *a: bt.chunk_attention(*a, window=9) * 2, fullgraph=True)
    assert torch.equal(whole(*args), bt.chunk_attention(*args, window=9) * 2)


REFUSALS = {
    "q type": dict(q=lambda x: x.float()), "k type": dict(k=lambda x: x.bfloat16()),
    "q rank": dict(q=lambda x: x[0]), "head dim": dict(q=lambda x: x[..., :32].contiguous()),
    "strided head dim": dict(q=lambda x: x.repeat_interleave(2, -1)[..., ::2]),
    "heads": dict(q=lambda x: x[:, :3]), "page size": dict(k=lambda x: x[:, :8], v=lambda x: x[:, :8]),
    "v shape": dict(v=lambda x: x[:-1]), "no pages": dict(k=lambda x: x[:0], v=lambda x: x[:0]),
    "table rows": dict(pages=lambda x: x[:1]), "table columns": dict(pages=lambda x: x[:, :0].contiguous()),
    "table type": dict(pages=lambda x: x.long()), "starts": dict(starts=lambda x: x[:-1]),
    "lengths": dict(lengths=lambda x: x[:1]), "host lengths": dict(lengths=lambda x: x.cpu()),
    "scale": dict(scale=0.0), "scale nan": dict(scale=float("nan")), "cap": dict(cap=-1.0),
    "cap inf": dict(cap=float("inf")), "window": dict(window=-1),
    "slopes": dict(slopes=torch.zeros(3)), "slopes type": dict(slopes=torch.zeros(4, dtype=torch.float16)),
    "prefix": dict(prefix=torch.zeros(3, dtype=torch.int32)),
    "prefix without causal": dict(prefix=torch.zeros(2, dtype=torch.int32), causal=False),
    "first": dict(first=torch.zeros(3, dtype=torch.int32)),
}


@pytest.mark.parametrize("what", REFUSALS)
def test_refusals(what):
    import branchcraft_torch as bt
    dev = C.on_gpu(C.batch([90, 40], [3, 4], 4, 2, 64, F16, seed=24))
    options = {}
    for name, change in REFUSALS[what].items():
        if name in dev:
            dev[name] = change(dev[name])
        else:
            options[name] = change.cuda() if isinstance(change, torch.Tensor) else change
    with pytest.raises((RuntimeError, NotImplementedError)):
        bt.chunk_attention(*(dev[n] for n in ("q", "k", "v", "pages", "lengths", "starts")), **options)


def test_append_refusals():
    import branchcraft_torch as bt

    def rows(*shape, dtype=F16):
        return torch.zeros(shape, device="cuda", dtype=dtype)

    slots = torch.zeros(3, device="cuda", dtype=torch.int32)
    k, v, r = rows(4, 16, 2, 64), rows(4, 16, 2, 64), rows(3, 2, 64)
    bt.append_kv_(k, v, r, r, slots.copy_(torch.tensor([0, 1, 2])))
    one = rows(1, 16, 2, 64)
    for args in [(k, v, r, rows(3, 2, 64, dtype=BF16), slots), (k, k, r, r, slots),
                 (k, v, k[0, :3], r, slots), (one.expand(4, 16, 2, 64), v, r, r, slots),
                 (k, v, r, r, slots[:2]), (k, v, r, r, slots.long()), (k, v, rows(3, 1, 64), rows(3, 1, 64), slots),
                 (k[:0], v[:0], r, r, slots), (k.cpu(), v, r, r, slots), (k[:, :8], v[:, :8], r, r, slots)]:
        with pytest.raises((RuntimeError, NotImplementedError)):
            bt.append_kv_(*args)
    bt.append_kv_(k, v, r[:0], r[:0], slots[:0])
