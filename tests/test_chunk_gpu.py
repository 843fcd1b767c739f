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
    "bias": dict(slopes=True),
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
