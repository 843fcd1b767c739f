"""PagedTreeCache.extend's bookkeeping, on fake tensors: no GPU needed."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode


def state(cache):
    return ({x: list(p) for x, p in cache.pages.items()}, dict(cache.lengths), list(cache.free),
            list(cache.refcount))


@pytest.mark.parametrize("at", ["_upload", "copy_pages_", "build_tables", "append_kv_", "chunk_attention"])
def test_a_call_that_fails_leaves_the_pages_as_they_were(at, monkeypatch):
    """An allocation that fails, say: shared and owned partial pages, a request
    that ends on a page and one that is empty.  The same call then takes the
    same pages as on a cache where nothing failed."""
    from branchcraft_torch import transaction
    with FakeTensorMode():
        def fill(n, heads=2):
            return torch.zeros(n, heads, 64, device="cuda", dtype=torch.float16)

        both = []
        for _ in range(2):
            cache = transaction.PagedTreeCache(20, 2, 64)
            a = cache.new(fill(21), fill(21))
            requests = [a, cache.fork(a), cache.new(fill(32), fill(32)), cache.new(fill(0), fill(0)),
                        cache.new(fill(5), fill(5)), cache.fork(a)]
            cache.checkpoint(requests[4])
            both.append(cache)
        cache, other = both
        counts = [20, 3, 1, 17, 2, 0]
        args = (requests, counts, fill(43, 4), fill(43), fill(43))
        before = state(cache)
        with monkeypatch.context() as m:
            def fail(*_, **__):
                raise torch.OutOfMemoryError("no memory")

            m.setattr(transaction.PagedTreeCache if at == "_upload" else transaction, at, fail)
            with pytest.raises(torch.OutOfMemoryError):
                cache.extend(*args)
        assert state(cache) == before
        cache.owner.check_invariants()
        for x in both:
            x.extend(*args)
        assert state(cache) == state(other) != before
