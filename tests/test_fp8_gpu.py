"""The 8-bit cache: rows rounded as they enter it, bit for bit; rows of it in 16
bits, exactly; and the attention over it against its definition in 64 bits over
the values that the cache holds."""

import pytest
import torch

import chunk_helpers as C
import fp8_helpers as F
import test_chunk_gpu as K

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def raw(x):
    return x.contiguous().view(torch.uint8)


def empty_pool(pages, hkv, d, seed=0):
    """Codes and scales that a test can tell from what is written."""
    g = torch.Generator().manual_seed(seed)
    pool = []
    for _ in range(2):
        codes = torch.randint(0, 127, (pages, 16, hkv, d), generator=g, dtype=torch.uint8)
        scale = torch.randint(100, 140, (pages, hkv, 16, d // 32), generator=g, dtype=torch.uint8)
        pool += [codes.view(F.E4M3).cuda(), scale.view(F.E8M0).cuda()]
    return pool


def rows(n, hkv, d, dtype, seed=0):
    """Rows of every size: whole blocks of zeros, outliers, the types' smallest and
    largest, infinities and NaN."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((n, hkv, d), generator=g)
    x = x * torch.exp2(torch.randint(-30, 15, (n, hkv, d // 32, 1), generator=g).float()).expand(
        n, hkv, d // 32, 32).flatten(-2)
    x = torch.where(torch.rand(x.shape, generator=g) < 0.02, x * 300, x)
    x = x.clamp(-6e4, 6e4).to(dtype)
    flat = x.view(-1, 32)
    kinds = [0.0, -0.0, float("inf"), float("-inf"), float("nan"), torch.finfo(dtype).max,
             torch.finfo(dtype).tiny, torch.finfo(dtype).smallest_normal / 8, 63488.0, 57344.0, 448.0, 449.0]
    for i, v in enumerate(kinds):
        if 3 * i + 2 < flat.shape[0]:
            flat[3 * i] = v
            flat[3 * i + 1, i] = v
            flat[3 * i + 2] *= 2.0 ** -12
    return x


@pytest.mark.parametrize("hkv,d", [(1, 64), (8, 128), (3, 64), (73, 128)])
@pytest.mark.parametrize("form", ["plain", "packed pool", "heads pool"])
@pytest.mark.parametrize("count", [0, 1, 10])
def test_pages_are_copied(count, form, hkv, d):
    """Bit for bit; pairs with a page outside the pool, or of one page, do nothing."""
    import branchcraft_torch as bt
    ck, sk, cv, sv = empty_pool(20, hkv, d)
    if form == "packed pool":
        whole = torch.stack((ck.view(torch.uint8), cv.view(torch.uint8)), 1).view(F.E4M3)
        ck, cv = whole[:, 0], whole[:, 1]
    elif form == "heads pool":
        ck, cv = (x.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(F.E4M3) for x in (ck, cv))
    src = torch.tensor([3, 0, 19, 3, -1, 20, 4, 8, 2**31 - 1, 5][:count], dtype=torch.int32)
    dst = torch.tensor([7, 18, 1, 2, 9, 10, 20, 8, 11, -2**31][:count], dtype=torch.int32)
    want = [raw(x).cpu().clone() for x in (ck, sk, cv, sv)]
    for a, b in zip(src.tolist(), dst.tolist()):
        if 0 <= a < 20 and 0 <= b < 20:
            for x in want:
                x[b] = x[a]
    bt.copy_fp8_pages_(ck, sk, cv, sv, src.cuda(), dst.cuda())
    torch.cuda.synchronize()
    for x, y in zip((ck, sk, cv, sv), want):
        assert torch.equal(raw(x).cpu(), y)


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("tokens,hkv,d", [(1, 8, 128), (3, 1, 64), (17, 3, 64), (300, 8, 128), (70, 40, 128)])
@pytest.mark.parametrize("form", ["plain", "fused", "heads_first", "unaligned", "expanded", "packed pool",
                                  "heads pool"])
def test_append_and_read(tokens, hkv, d, form, dtype):
    import branchcraft_torch as bt
    k, v = rows(tokens, hkv, d, dtype, 1).cuda(), rows(tokens, hkv, d, dtype, 2).cuda()
    if form == "fused":
        whole = torch.stack((k, k, v), 1)
        k, v = whole[:, 1], whole[:, 2]
    elif form == "heads_first":
        k = k.transpose(0, 1).contiguous().transpose(0, 1)
    elif form == "unaligned":
        k = torch.cat((k.new_zeros(1), k.flatten()))[1:].view(tokens, hkv, d)
    elif form == "expanded":
        k, v = k[:1].expand(tokens, hkv, d), v[:, :1].expand(tokens, hkv, d)
    pages = tokens // 16 + 4
    ck, sk, cv, sv = empty_pool(pages, hkv, d)
    if form == "packed pool":
        whole = torch.stack((ck.view(torch.uint8), cv.view(torch.uint8)), 1).view(F.E4M3)
        ck, cv = whole[:, 0], whole[:, 1]
    elif form == "heads pool":
        ck, cv = (x.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(F.E4M3) for x in (ck, cv))
    slots = torch.randperm(pages * 16, generator=torch.Generator().manual_seed(3))[:tokens].to(torch.int32)
    slots[::5] = torch.tensor([-1, pages * 16, -2**31, 2**31 - 1])[torch.arange(len(slots[::5])) % 4].int()
    want = [x.cpu().clone() for x in (ck, sk, cv, sv)]
    back = []
    for x, codes, scale in ((k, want[0], want[1]), (v, want[2], want[3])):
        c, s = F.to_fp8(x.cpu())
        held = F.values(c, s)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages * 16:
                codes.view(torch.uint8)[slot // 16, slot % 16] = c.view(torch.uint8)[t]
                scale.view(torch.uint8)[slot // 16, :, slot % 16] = s.view(torch.uint8)[t]
            else:
                held[t] = 0
        assert torch.equal(held.to(dtype).double().nan_to_num(1e9), held.nan_to_num(1e9))  # exact in the type
        back.append(held.to(dtype))
    bt.append_fp8_kv_(ck, sk, cv, sv, k, v, slots.cuda())
    for got, w in zip((ck, sk, cv, sv), want):
        got, w = raw(got.cpu()), raw(w)
        nan = (w & 0x7f) == 0x7f  # of a NaN the sign is not held to anything
        assert torch.equal(torch.where(nan, w, got), w) and bool(((got & 0x7f) == 0x7f)[nan].all())
    for got, w in zip(bt.read_fp8_kv(ck, sk, cv, sv, slots.cuda(), dtype), back):
        assert got.dtype == dtype and got.is_contiguous()
        assert torch.equal(got.cpu().nan_to_num(1e4), w.nan_to_num(1e4))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
def test_every_code_under_every_scale(dtype):
    """Read back as the nearest value of the type, ties to even; NaN codes as NaN."""
    import branchcraft_torch as bt
    codes = torch.arange(256, dtype=torch.uint8).view(1, 1, 4, 64).expand(255, 16, 4, 64).contiguous()
    scale = torch.arange(255, dtype=torch.uint8).view(255, 1, 1, 1).expand(255, 4, 16, 2).contiguous()
    pool = codes.view(F.E4M3).cuda(), scale.view(F.E8M0).cuda()
    slots = torch.arange(255 * 16, dtype=torch.int32, device="cuda")[::16].contiguous()
    k, v = bt.read_fp8_kv(*pool, *pool, slots, dtype)
    want = codes[:, 0].view(F.E4M3).double() * torch.exp2(torch.arange(255).double() - 127)[:, None, None]
    want = want.to(dtype)
    for got in (k, v):
        assert torch.equal(got.cpu().nan_to_num(1e4), want.nan_to_num(1e4))
        assert torch.equal(got.cpu().isnan(), want.isnan())


def test_no_rows_and_rows_twice():
    import branchcraft_torch as bt
    pool = empty_pool(4, 2, 64)
    before = [raw(x).clone() for x in pool]
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    nothing = torch.zeros(0, 2, 64, dtype=F16, device="cuda")
    bt.append_fp8_kv_(*pool, nothing, nothing, none)
    assert all(torch.equal(raw(x), b) for x, b in zip(pool, before))
    assert [tuple(x.shape) for x in bt.read_fp8_kv(*pool, none, BF16)] == [(0, 2, 64)] * 2
    twice = torch.tensor([5, 5, 60], dtype=torch.int32, device="cuda")
    k, v = bt.read_fp8_kv(*pool, twice, BF16)
    assert torch.equal(k[0], k[1]) and torch.equal(v[0], v[1])


def attend(fix, pool, **options):
    import branchcraft_torch as bt
    dev = C.on_gpu(fix)
    options = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in options.items()}
    k, sk, v, sv = (x.cuda() for x in pool)
    out = bt.fp8_chunk_attention(dev["q"], k, sk, v, sv, dev["pages"], dev["lengths"], dev["starts"], **options)
    torch.cuda.synchronize()
    assert out.dtype == fix["q"].dtype and out.is_contiguous()
    return out


def both(fix, what="", **options):
    pool, same = F.pools(fix)
    want, tol = C.reference(**same, **options)
    got = attend(fix, pool, **options)
    C.check(got, want, tol, what)
    return got


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (7, 1, 64), (4, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize("shape", range(len(K.SHAPES)))
def test_causal(shape, hq, hkv, d, dtype):
    both(C.batch(*K.SHAPES[shape], hq, hkv, d, dtype, seed=shape))


@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 8, 2, 128), (BF16, 6, 2, 64)])
@pytest.mark.parametrize("shape", [([333, 1, 90, 64], [130, 1, 17, 40]), ([700], [1])])
@pytest.mark.parametrize("form", K.FORMS)
def test_forms(form, shape, dtype, hq, hkv, d):
    fix = C.batch(*shape, hq, hkv, d, dtype, seed=len(form))
    both(fix, form, **K.options_of(form, fix))


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
@pytest.mark.parametrize("form", ["scale", "window 500", "cap bias"])
def test_long_and_split(form, dtype, d):
    fix = C.batch([5000, 3, 4111], [2, 1, 9], 4, 1, d, dtype, seed=3)
    both(fix, form, **K.options_of(form, fix))
    fix = C.batch([2100, 40, 1], [60, 2, 0], 4, 1, d, dtype, seed=3)
    both(fix, form, **K.options_of(form, fix))


def test_sharp_scores():
    fix = C.batch([400, 300], [70, 1], 8, 2, 128, F16, seed=9, spread=12.0)
    both(fix)
    both(fix, cap=20.0)


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128)])
def test_rows_of_every_size(dtype, d):
    """Blocks whose powers differ by 2^40, and outliers inside them."""
    fix = C.batch([150, 40], [40, 1], 4, 2, d, dtype, seed=4)
    for x in ("k", "v"):
        keep = fix[x].isnan()
        g = torch.Generator().manual_seed(6)
        size = torch.exp2(torch.randint(-24, 2, (*fix[x].shape[:3], d // 32, 1), generator=g).float())
        fix[x] = (torch.randn(fix[x].shape, generator=g) * size.expand(*size.shape[:-1], 32).flatten(-2)).to(dtype)
        fix[x][..., 7] *= 30
        fix[x][keep] = float("nan")
    both(fix)


def test_pages_outside_the_pool_are_not_seen():
    fix = C.batch([200, 90], [70, 1], 8, 2, 128, F16, seed=4)
    fix["pages"][0, 3] = -1
    fix["pages"][0, 7] = 2**31 - 1
    fix["pages"][1, 0] = fix["k"].shape[0]
    both(fix)


@pytest.mark.parametrize("lengths,counts", [([200, 90], [70, 1]), ([3000, 90], [9, 1])])
def test_what_a_row_does_not_see_may_hold_anything(lengths, counts):
    """NaN in tokens behind a row, in tokens of other windows: seen by none of the
    rows, or by some of them, which then are NaN."""
    fix = C.batch(lengths, counts, 4, 2, 64, BF16, seed=8)
    ids = fix["pages"][0].long()
    bad = lengths[0] - 3  # the last three rows' and nobody else's
    for x in ("k", "v"):
        fix[x][ids[bad // 16], bad % 16, 1, 5] = float("nan")
    got = both_with_nan(fix, bad, lengths, counts)
    assert bool(got[:counts[0] - 3].isfinite().all()) and bool(got[counts[0]:].isfinite().all())


def both_with_nan(fix, bad, lengths, counts):
    pool, same = F.pools(fix)
    got = attend(fix, pool).cpu()
    clean = {n: x.clone() if isinstance(x, torch.Tensor) else x for n, x in same.items()}
    ids = fix["pages"][0].long()
    for x in ("k", "v"):
        clean[x][ids[bad // 16], bad % 16, 1, 5] = 0
    want, tol = C.reference(**clean)
    sees = torch.zeros(got.shape[0], got.shape[1], dtype=torch.bool)
    sees[counts[0] - 3:counts[0], 2:] = True  # KV head 1's query heads
    C.check(torch.where(sees[..., None], 0, got.double()), torch.where(sees[..., None], 0, want), tol)
    assert bool(got[sees].isnan().any(-1).all())
    return torch.where(sees[..., None], 0, got)
