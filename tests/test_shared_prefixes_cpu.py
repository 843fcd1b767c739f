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


@pytest.mark.parametrize("forks", [0, 1])
def test_extend_without_common_pages_is_the_plain_call(forks, monkeypatch):
    """Also where pages are shared by requests that the call does not name next to each
    other, and by one request of the call alone."""
    from branchcraft_torch import transaction
    seen = []
    for name in ("chunk_attention", "shared_chunk_attention"):
        real = getattr(transaction, name)
        monkeypatch.setattr(transaction, name, lambda *a, _real=real, _name=name, **k: (seen.append(_name), _real(*a, **k))[1])
    with FakeTensorMode():
        def fill(n, heads=2):
            return torch.zeros(n, heads, 64, device="cuda", dtype=torch.float16)

        cache = transaction.PagedTreeCache(40, 2, 64)
        a, b, c = (cache.new(fill(n), fill(n)) for n in (50, 70, 15))
        d, e = cache.fork(a), cache.fork(c)  # of c no whole page is shared
        requests = [a, d, b, c, e] if forks else [a, b, d, c, e]
        cache.extend(requests, [1] * 5, fill(5, 4), fill(5), fill(5), share=True)
        cache.extend([a], [2], fill(2, 4), fill(2), fill(2), share=True)
    assert seen == ["shared_chunk_attention" if forks else "chunk_attention", "chunk_attention"]
