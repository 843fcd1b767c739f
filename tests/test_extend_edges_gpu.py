"""PagedTreeCache.extend: what it refuses leaves pages, lengths and rows as they
were, and what it takes need not be laid out one way."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def rows(g, n, heads, d=64):
    return torch.randn((n, heads, d), generator=g, device="cuda", dtype=torch.float16)


def caches(n, *, pages=8, tokens=20, seed=1):
    from branchcraft_torch.transaction import PagedTreeCache
    out = []
    for _ in range(n):
        g = torch.Generator("cuda").manual_seed(seed)
        cache = PagedTreeCache(pages, 2, 64)
        a = cache.new(rows(g, tokens, 2), rows(g, tokens, 2))
        out.append((cache, a, cache.fork(a)))
    return out, g


def state(cache):
    return ({x: list(p) for x, p in cache.pages.items()}, dict(cache.lengths), list(cache.free),
            list(cache.refcount))


def test_a_strided_first_is_taken():
    """Every second entry of a list of document starts."""
    both, g = caches(2)
    q, k, v = rows(g, 7, 4), rows(g, 7, 2), rows(g, 7, 2)
    first = torch.tensor([0, 9, 3, 9, 20, 9, 21, 9, 1, 9, 20, 9, 4, 9], device="cuda", dtype=torch.int32)[::2]
    assert not first.is_contiguous()
    outs = [cache.extend([a, b], [4, 3], q, k, v, first=f)
            for (cache, a, b), f in zip(both, (first, first.contiguous()))]
    assert torch.equal(*outs)
    assert state(both[0][0]) == state(both[1][0])


def test_a_tangent_on_the_pool_is_refused_before_anything_changes():
    from torch.autograd import forward_ad
    ((cache, a, b),), g = caches(1)
    q, k, v = rows(g, 7, 4), rows(g, 7, 2), rows(g, 7, 2)
    before = state(cache)
    for name in ("k", "v"):
        with forward_ad.dual_level():
            plain = getattr(cache, name)
            setattr(cache, name, forward_ad.make_dual(plain, torch.ones_like(plain)))
            with pytest.raises(ValueError, match="differentiable"):
                cache.extend([a, b], [4, 3], q, k, v)
            setattr(cache, name, plain)
        assert state(cache) == before


def test_rows_that_are_views_of_a_subclass_pool():
    """As with a plain pool: they are read before the pool is written."""
    class Pool(torch.Tensor):
        pass

    both, g = caches(2)
    q, outs = rows(g, 7, 4), []
    for turn, (cache, a, b) in enumerate(both):
        if turn:
            cache.k, cache.v = cache.k.as_subclass(Pool), cache.v.as_subclass(Pool)
        page = cache.pages[a][0]
        outs.append(cache.extend([a, b], [4, 3], q, cache.k[page, 2:9], cache.v[page, 2:9]).as_subclass(torch.Tensor))
    assert torch.equal(*outs)
    assert all(torch.equal(getattr(both[0][0], x), getattr(both[1][0], x).as_subclass(torch.Tensor)) for x in "kv")
    assert state(both[0][0]) == state(both[1][0])


def test_a_capture_is_refused_before_anything_changes():
    """Pages are planned on the host, once; a graph would replay that plan."""
    ((cache, a, b),), g = caches(1)
    q, k, v = rows(g, 7, 4), rows(g, 7, 2), rows(g, 7, 2)
    before = state(cache)
    out = torch.zeros(1, device="cuda")
    with torch.cuda.graph(torch.cuda.CUDAGraph()):
        out += 1
        with pytest.raises(RuntimeError, match="captured"):
            cache.extend([a, b], [4, 3], q, k, v)
    assert state(cache) == before
    assert cache.extend([a, b], [4, 3], q, k, v).shape == q.shape


def test_inference_mode_moves_the_pools_counters():
    """A pool made outside and rows made inside, the whole step."""
    both, g = caches(2)
    (cache, a, b), (other, _, _) = both
    q, k, v = rows(g, 7, 4), rows(g, 7, 2), rows(g, 7, 2)
    want = other.extend([a, b], [4, 3], q, k, v, cap=9.0)
    versions = cache.k._version, cache.v._version
    with torch.inference_mode():
        got = cache.extend([a, b], [4, 3], q.clone(), k.clone(), v.clone(), cap=9.0)
    assert torch.equal(got, want) and torch.equal(cache.k, other.k) and torch.equal(cache.v, other.v)
    assert cache.k._version > versions[0] and cache.v._version > versions[1]
