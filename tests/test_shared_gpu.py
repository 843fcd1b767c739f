"""shared_chunk_attention against the definition of the attention in 64 bits over
each request's own table, at the group and prefix sizes where it can go wrong.
Slots of the pool that hold no token are NaN throughout."""

import pytest
import torch

import chunk_helpers as C
import fp8_helpers as F
import test_chunk_gpu as K

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16


def attend(fix, groups, shared, **options):
    import branchcraft_torch as bt
    dev = C.on_gpu(fix)
    options = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in options.items()}
    out = bt.shared_chunk_attention(dev["q"], dev["k"], dev["v"], dev["pages"], dev["lengths"], dev["starts"],
                                    groups.cuda(), shared.cuda(), **options)
    torch.cuda.synchronize()
    assert out.dtype == fix["q"].dtype and out.is_contiguous()
    return out


def both(fix, groups, shared, what="", **options):
    """A row's two parts are joined in 32 bits: exponentials and sums of a few
    roundings more, of which C.reference's bound counts 16 per score.  Without a
    window every case is one that reads shared pages once."""
    assert F.pays(fix) or not len(shared)
    want, tol = C.reference(**fix, **options)
    got = attend(fix, groups, shared, **options)
    C.check(got, want, tol, what)
    return got


# (shared tokens, [(own tokens, new tokens), ...]) of each group.
GROUPS = [
    [(16, [(1, 1), (1, 1)])],
    [(160, [(1, 1)] * 8)],
    [(2048, [(5, 1), (64, 1), (1, 1), (17, 1)])],
    [(1000, [(30, 2), (40, 3)]), (64, [(3, 1), (80, 40)]), (0, [(20, 1), (30, 1)])],
    [(130, [(9, 9), (200, 90), (5, 0), (31, 5)]), (333, [(40, 1)] + [(7, 1)] * 5)],
    [(48, [(11, 11)] * 40)],
    [(700, [(3, 1)] * 70), (32, [(8, 3)] * 3)],
    [(17, [(2, 1), (2, 2), (1, 0)]), (15, [(1, 1), (600, 1)])],
]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (7, 1, 64), (4, 4, 64)])
@pytest.mark.parametrize("case", range(len(GROUPS)))
def test_causal(case, hq, hkv, d, dtype):
    both(*F.forks(GROUPS[case], hq, hkv, d, dtype, seed=case))


@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 8, 2, 128), (BF16, 6, 2, 64)])
@pytest.mark.parametrize("case", [3, 4])
@pytest.mark.parametrize("form", K.FORMS)
def test_forms(form, case, dtype, hq, hkv, d):
    fix, groups, shared = F.forks(GROUPS[case], hq, hkv, d, dtype, seed=len(form))
    both(fix, groups, shared, form, **K.options_of(form, fix))


@pytest.mark.parametrize("form", ["scale", "window 50", "window 500", "cap bias", "first"])
@pytest.mark.parametrize("members,new", [(3, 1), (20, 2)])
def test_long_prefixes(form, members, new):
    """Split over workgroups, with few rows and with more than a tile's."""
    fix, groups, shared = F.forks([(3000, [(new + i, new) for i in range(members)]), (1500, [(600, 2), (9, 1)])],
                                  8, 2, 128, BF16, seed=3)
    both(fix, groups, shared, form, **K.options_of(form, fix))


@pytest.mark.parametrize("form", ["window", "window bias", "window full", "cap window", "window first"])
def test_windows(form):
    """With enough requests and heads that a window's tokens pay for it."""
    fix, groups, shared = F.forks([(500, [(1 + i, 1) for i in range(40)]), (300, [(200 + 9 * i, 2) for i in range(24)])],
                                  32, 32, 128, F16, seed=7)
    options = dict(window=400)
    assert F.pays(fix, 400)
    if form == "window bias":
        options["slopes"] = torch.rand(32, generator=torch.Generator().manual_seed(3)) - 0.25
    if form == "window full":
        options["causal"] = False
    if form == "cap window":
        options["cap"] = 5.0
    if form == "window first":
        options.update(K.options_of("first", fix))
    both(fix, groups, shared, form, **options)


@pytest.mark.parametrize("new", [1, 3])
def test_small_batches_read_their_own_pages(new):
    fix, groups, shared = F.forks([(64, [(new, new)] * 3)], 4, 2, 64, F16, seed=5)
    fix["pages"] = fix["pages"][:, :6].contiguous()
    assert not F.pays(fix)
    want, tol = C.reference(**fix)
    C.check(attend(fix, groups, shared), want, tol)


def test_requests_outside_the_groups():
    fix, groups, shared = F.forks([(0, [(90, 3), (5, 1)]), (200, [(3, 1)] * 5), (100, [(4, 2)] * 3), (0, [(33, 33)])],
                                  4, 2, 64, F16, seed=5, lone_ends=1)
    assert groups.tolist() == [2, 7, 10]
    both(fix, groups, shared)
    none = torch.zeros(0, dtype=torch.int32)
    both(fix, groups[:1], none)
    for bounds in ([2, 3, 7, 10], [2, 7, 7, 10], [3, 6, 7, 10]):  # of one and of no request
        both(fix, torch.tensor(bounds, dtype=torch.int32), torch.tensor([64, 96, 96], dtype=torch.int32))


def test_sharp_scores():
    """The shared part's maximum far above the own part's, and the reverse."""
    fix, groups, shared = F.forks([(400, [(60, 9), (2, 2), (30, 1)])], 8, 2, 128, F16, seed=9, spread=12.0)
    both(fix, groups, shared)
    both(fix, groups, shared, cap=20.0)


def test_prefixes_longer_than_what_a_row_sees():
    """Shared tokens that reach past a request's new ones, and past its length."""
    fix, groups, shared = F.forks([(96, [(4, 30), (4, 4)]), (64, [(16, 10), (16, 16), (16, 1)])], 4, 2, 64, BF16, seed=2)
    both(fix, groups, shared)
    both(fix, groups, shared, causal=False)
    for short in (3, 40, 95):
        both(fix, groups, torch.tensor([short, 10 * short % 64], dtype=torch.int32))


def test_rows_of_no_request_are_zero():
    fix, groups, shared = F.forks([(200, [(5, 2)] * 3)], 4, 2, 64, BF16, seed=2)
    g = torch.Generator().manual_seed(1)
    pad = torch.randn((5, 4, 64), generator=g).to(BF16)
    fix["q"] = torch.cat((pad[:2], fix["q"], pad[2:]))
    fix["starts"] = fix["starts"] + 2
    got = both(fix, groups, shared)
    assert bool((got[:2] == 0).all()) and bool((got[8:] == 0).all())


def test_pages_outside_the_pool_are_not_seen():
    fix, groups, shared = F.forks([(160, [(5, 2), (70, 40), (3, 1)])], 4, 2, 64, F16, seed=4)
    fix["pages"][:, 3] = -1
    fix["pages"][:, 7] = fix["k"].shape[0]
    fix["pages"][1, 11] = 2**31 - 1
    both(fix, groups, shared)


@pytest.mark.parametrize("members", [3, 40])
@pytest.mark.parametrize("bad", [(2.0, float("inf")), (float("nan"), 1.0)])
def test_what_a_row_does_not_see_may_hold_anything(bad, members):
    """A token of the prefix that documents hide from some members and not from
    others."""
    fix, groups, shared = F.forks([(200, [(5, 1), (60, 1), (5, 5)] + [(1, 1)] * (members - 3))], 4, 2, 64, BF16, seed=8)
    assert F.pays(fix)
    page = int(fix["pages"][0, 190 // 16])
    fix["k"][page, 190 % 16, 0, 3], fix["v"][page, 190 % 16, 0, 3] = bad
    rows = fix["q"].shape[0]
    first = torch.zeros(rows, dtype=torch.int32)
    first[1], first[7:] = 191, 195
    got = attend(fix, groups, shared, first=first).cpu()
    fix["k"][page, 190 % 16, 0, 3] = fix["v"][page, 190 % 16, 0, 3] = 0
    want, tol = C.reference(**fix, first=first)
    hidden = [1, *range(7, rows)]
    C.check(got[hidden], want[hidden], tol[hidden])
    C.check(got[:, 2:], want[:, 2:], tol[:, 2:])  # the other KV head's
    assert not bool(got[[0, 2, 3, 4, 5, 6], :2, 3].isfinite().any())
