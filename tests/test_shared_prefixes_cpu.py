"""Which neighbours of a list of requests share how many tokens, and what extend makes
of it: bookkeeping alone, no GPU needed."""

import itertools
import random

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def saved(bounds, tokens):
    """Tokens that are not read again, since members read them together."""
    return sum((b - a - 1) * n for a, b, n in zip(bounds, bounds[1:], tokens))


def most_saved(owner, requests):
    """The largest such number of any cut of the list into neighbours, by trying the
    start of the last group."""
    pages = [owner.pages[x][:owner.lengths[x] // 16] for x in requests]
    best = [0]
    for i in range(1, len(pages) + 1):
        most, of = len(pages[i - 1]), [best[i - 1]]
        for j in range(i - 2, -1, -1):
            same = sum(1 for _ in itertools.takewhile(lambda p: p[0] == p[1], zip(pages[j], pages[i - 1])))
            most = min(most, same)
            of.append(best[j] + (i - 1 - j) * most * 16)
        best.append(max(of))
    return best[-1]


@pytest.mark.parametrize("order", ["first", "last", "between", "two"])
def test_forks_of_a_document_beside_requests_behind_the_same_system_prompt(order):
    """A short prompt before everything costs the forks of a long one nothing."""
    from branchcraft_torch.pages import PageOwner
    owner = PageOwner(3000)
    system = owner.new(32)
    chats = [owner.fork(system) for _ in range(2)]
    for i, x in enumerate(chats):
        owner.plan_commit(x, 3000 + i)
    document = owner.fork(system)
    owner.plan_commit(document, 16000)
    forks = [document] + [owner.fork(document) for _ in range(7)]
    for x in forks:
        owner.plan_commit(x, 3)
    requests = {"first": chats[:1] + forks, "last": forks + chats[:1], "between": forks[:3] + chats[:1] + forks[3:],
                "two": chats + forks}[order]
    want = {"first": ([0, 1, 9], [3032, 16032]), "last": ([0, 8, 9], [16032, 3032]),
            "between": ([0, 3, 4, 9], [16032, 3032, 16032]), "two": ([0, 2, 10], [32, 16032])}[order]
    assert owner.shared_prefixes(requests) == want


def test_prefixes_that_grow_shorter_from_one_to_the_next():
    """Each shares a little over half of what the one before it shares: taken one after
    another, each for less than half, they would leave what the last one has."""
    from branchcraft_torch.pages import PageOwner
    owner = PageOwner(9000)
    requests, n = [], 16 * 800
    trunk = owner.new(n)
    branches = [trunk]
    whole = list(owner.pages[trunk])
    while n > 16 * 20:  # requests whose first n tokens are the trunk's
        for _ in range(4):
            x = owner.new(n)
            owner._drop(owner.pages[x])
            owner.pages[x] = whole[:n // 16]
            owner._hold(owner.pages[x])
            owner.plan_commit(x, 40)
            requests.append(x)
        n = n // 16 * 6 // 10 * 16
    requests = branches + requests
    owner.check_invariants()
    got = owner.shared_prefixes(requests)
    assert saved(*got) == most_saved(owner, requests) and len(got[1]) > 2


@pytest.mark.parametrize("seed", range(60))
def test_no_other_groups_read_fewer_tokens(seed):
    """Trees of forks of forks, as they come, sorted by their pages, and shuffled."""
    from branchcraft_torch.pages import PageOwner
    r = random.Random(seed)
    owner = PageOwner(20000)
    requests = [owner.new(r.randint(0, 400))]
    for _ in range(r.choice((3, 20, 60))):
        kind = r.random()
        if kind < 0.1:
            requests.append(owner.new(r.randint(0, 300)))
        elif kind < 0.6:
            requests.append(owner.fork(r.choice(requests)))
        else:
            owner.plan_commit(r.choice(requests), r.randint(1, 150))
    if seed % 3 == 1:
        r.shuffle(requests)
    if seed % 3 == 2:
        requests.sort(key=lambda x: owner.pages[x])
    bounds, tokens = owner.shared_prefixes(requests)
    for a, b, n in zip(bounds, bounds[1:], tokens):
        first = owner.pages[requests[a]]
        assert b - a == 1 and n == owner.lengths[requests[a]] or n > 0 and n % 16 == 0
        assert all(n <= owner.lengths[x] and owner.pages[x][:n // 16] == first[:n // 16]
                   for x in requests[a:b] if b - a > 1)
    assert saved(bounds, tokens) == most_saved(owner, requests)


def test_prefixes_of_no_request():
    from branchcraft_torch.pages import PageOwner
    assert PageOwner(4).shared_prefixes([]) == ([0], [])


# (Tokens in common, own tokens, members) of families behind one system prompt, the
# window, and the groups and tokens that extend tells the attention of.
BATCHES = {
    "nothing in common": (0, [(0, 700, 1)] * 5, 0, None),
    "a system prompt": (64, [(0, 700, 1)] * 5, 0, None),
    "few tokens of many": (0, [(320, 5000, 2)] * 3, 0, None),
    "little of much": (0, [(2048, 9, 4)] + [(0, 7000, 1)] * 4, 0, None),
    "forks": (0, [(1024, 30, 3)], 0, ([0, 3], [1024])),
    "forks beside others": (32, [(0, 700, 1), (2048, 30, 8), (0, 300, 2)], 0, ([0, 1, 9, 11], [0, 2080, 0])),
    "forks behind a window": (0, [(1024, 900, 6)], 1000, None),
    "forks in a window": (0, [(1024, 300, 6)], 1000, ([0, 6], [1024])),
    "one fork in a window": (0, [(1024, 300, 1), (0, 20, 6)], 1000, None),
}


@pytest.mark.parametrize("batch", BATCHES)
def test_extend_shares_where_that_spares_enough(batch, monkeypatch):
    """Elsewhere it is the plain call."""
    from branchcraft_torch import transaction
    calls = []

    def attention(name, real):
        def call(*args, **options):
            if args[0].shape[0]:  # not the check of the options
                calls.append(name)
            return real(*args, **options)
        return call

    for name in ("chunk_attention", "shared_chunk_attention"):
        monkeypatch.setattr(transaction, name, attention(name, getattr(transaction, name)))
    uploads = []
    upload = transaction.PagedTreeCache._upload
    monkeypatch.setattr(transaction.PagedTreeCache, "_upload",
                        lambda self, *lists: (uploads.append(lists), upload(self, *lists))[1])
    system, families, window, want = BATCHES[batch]
    with FakeTensorMode():
        def fill(n, heads=1):
            return torch.zeros(n, heads, 64, device="cuda", dtype=torch.float16)

        cache = transaction.PagedTreeCache(4000, 1, 64)
        root = cache.new(fill(system), fill(system))
        requests = []
        for common, own, members in families:
            first = cache.fork(root)
            if common:
                cache.owner.plan_commit(first, common)
            family = [first] + [cache.fork(first) for _ in range(members - 1)]
            for x in family:
                cache.owner.plan_commit(x, own - 1)
            requests += family
        n = len(requests)
        cache.extend(requests, [1] * n, fill(n, 2), fill(n), fill(n), share=True, **(dict(window=window) if window else {}))
    assert calls == ["chunk_attention" if want is None else "shared_chunk_attention"]
    assert uploads[-1][5:] == (() if want is None else want)


@pytest.mark.parametrize("same", [0, 1, 2, 5, 8, 9])
def test_common_pages_whatever_is_guessed(same):
    from branchcraft_torch.pages import _same_pages
    x = list(range(9))
    y = x[:same] + [100 + i for i in range(9 - same)]
    for end in range(10):
        for guess in range(12):
            assert _same_pages(x, y, end, guess) == min(same, end)


@pytest.mark.parametrize("counts,shares", [([1, 0, 0, 0], False), ([0, 0, 0, 1], False), ([1, 0, 0, 2], True),
                                           ([0, 3, 1, 0], True), ([0, 0, 0, 0], False)])
def test_requests_without_new_tokens_read_nothing(counts, shares, monkeypatch):
    from branchcraft_torch import transaction
    calls = []
    for name in ("chunk_attention", "shared_chunk_attention"):
        real = getattr(transaction, name)
        monkeypatch.setattr(transaction, name, lambda *a, _real=real, _name=name: (calls.append(_name), _real(*a))[1])
    with FakeTensorMode():
        def fill(n, heads=1):
            return torch.zeros(n, heads, 64, device="cuda", dtype=torch.float16)

        cache = transaction.PagedTreeCache(400, 1, 64)
        a = cache.new(fill(2000), fill(2000))
        n = sum(counts)
        cache.extend([a] + [cache.fork(a) for _ in range(3)], counts, fill(n, 2), fill(n), fill(n), share=True)
    assert calls == ["shared_chunk_attention" if shares else "chunk_attention"]
