"""Copy-on-write paged KV transaction driving the HIP ops.

Mirrors ``PagedTreeCache`` of the reference
(python/branchcraft_torch/transaction.py:23-150): an FP16 pool
[physical_pages, 16, kv_heads, head_dim] for K and for V, requests that can
be forked and checkpointed, tree verification against a request's pages and
a commit of an accepted root-to-leaf path.  The bookkeeping lives in
:class:`~branchcraft_torch.pages.PageOwner`; the device work -- the clone of
a shared partial page and the accepted-path copy -- runs as the
``copy_pages_`` and ``commit_path_`` HIP ops on the current stream.
``commit_many`` commits several requests with two launches (every clone, then
every accepted node) and one for their index lists, and leaves the same pages and page tables
as committing them one by one in the same order.  ``extend`` appends ordinary new
tokens to several requests and attends to them: a chunk of a prompt, a turn, a
decode step; with ``share``, pages that forks have in common are read once.

``Fp8Cache`` is the same for ordinary tokens in 8 bits: half the pool, half the bytes
of every step.
"""

from __future__ import annotations

import torch
from torch.autograd.forward_ad import unpack_dual

from . import (append_fp8_kv_, append_kv_, build_tables, chunk_attention, commit_path_,
               commit_paths_, copy_fp8_pages_, copy_pages_, fp8_chunk_attention, int_tensor,
               read_fp8_kv, shared_chunk_attention, tree_verify, write_prefix_)
from .pages import CommitPlan, PageOwner, Snapshot

__all__ = ["PagedTreeCache", "Fp8Cache", "Snapshot", "CommitPlan"]


LEAST_SHARED = 256  # tokens


def _worth_reading_once(bounds: list[int], tokens: list[int], lengths: list[int], counts: list[int],
                        window: int) -> tuple[list[int], list[int]] | tuple[()]:
    """The groups of ``PageOwner.shared_prefixes`` as the attention is told of them:
    those that share few tokens as sharing none, and () where they spare too little of
    what the requests with new tokens read.

    Every group starts with a round trip of its own and every row is joined, whatever is
    shared (attention of single tokens, 32/8 heads, D = 128, shared and plain, us): 64
    requests of 2048 tokens in pairs that share 16 tokens 121 and 66, 64 tokens 88 and
    66, 256 70 and 66, 1024 65 and 66; all 64 together 256 tokens 67 and 62, 1024 48 and
    54.  Over 155 batches of forks at five head layouts the calls that these two rules
    choose took 79 % of the plain ones' time (geometric mean) and 6 % (3 us) more at most."""
    saved, once = 0, []
    for a, b, n in zip(bounds, bounds[1:], tokens):
        # What each member sees of it, within a window that ends with the request.
        seen = [max(n - max(x - window, 0), 0) if window else n
                for x, new in zip(lengths[a:b], counts[a:b]) if new]
        worth = len(seen) > 1 and max(seen) >= LEAST_SHARED
        once.append(n if worth else 0)
        saved += sum(seen) - max(seen) if worth else 0
    read = sum(min(x, window) if window else x for x, new in zip(lengths, counts) if new)
    return (bounds, once) if saved and 4 * saved >= read else ()


class PagedTreeCache:
    def __init__(self, physical_pages: int, kv_heads: int, head_dim: int,
                 device: str = "cuda"):
        if head_dim not in (64, 128) or physical_pages < 1:
            raise ValueError("head_dim must be 64/128; physical_pages must be positive")
        self.owner = PageOwner(physical_pages)
        self.k = torch.zeros((physical_pages, 16, kv_heads, head_dim),
                             device=device, dtype=torch.float16)
        self.v = torch.zeros_like(self.k)

    @property
    def dtype(self) -> torch.dtype:
        """The type of the rows that enter the cache, and of queries and outputs."""
        return self.k.dtype

    # What extend does on the device, by the pool's form.
    def _pools(self) -> tuple[torch.Tensor, ...]:
        return self.k, self.v

    def _clone(self, old: torch.Tensor, fresh: torch.Tensor) -> None:
        copy_pages_(self.k, self.v, old, fresh)

    def _append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        append_kv_(self.k, self.v, k, v, slots)

    def _attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                starts: torch.Tensor, groups: tuple[torch.Tensor, ...], **options) -> torch.Tensor:
        op = shared_chunk_attention if groups else chunk_attention
        return op(q, self.k, self.v, table, lengths, starts, *groups, **options)

    # The reference exposes these as attributes.
    @property
    def pages(self) -> dict[int, list[int]]:
        return self.owner.pages

    @property
    def lengths(self) -> dict[int, int]:
        return self.owner.lengths

    @property
    def refcount(self) -> list[int]:
        return self.owner.refcount

    @property
    def free(self) -> list[int]:
        return self.owner.free

    def new(self, prefix_k: torch.Tensor, prefix_v: torch.Tensor) -> int:
        """Create one request from [tokens, KV heads, head dim] FP16 tensors."""
        if prefix_k.shape != prefix_v.shape or prefix_k.ndim != 3:
            raise ValueError("prefix K/V shapes must match [tokens, heads, dim]")
        if prefix_k.dtype != torch.float16 or prefix_k.device != self.k.device:
            raise ValueError("prefix must be FP16 on the cache device")
        if tuple(prefix_k.shape[1:]) != tuple(self.k.shape[2:]):
            raise ValueError("prefix head shape differs from cache")
        tokens = prefix_k.shape[0]
        request = self.owner.new(tokens)
        self._write_prefix(self.owner.pages[request], prefix_k, prefix_v)
        return request

    def _write_prefix(self, pages: list[int], prefix_k: torch.Tensor,
                      prefix_v: torch.Tensor) -> None:
        """Prompt rows into fresh pages: one launch, the page ids in its
        kernel arguments.  What the op does not take -- a pool that is not on
        the GPU, a subclass, or rows that are views of the pool itself -- is
        copied page by page."""
        rows = [prefix_k, prefix_v]
        if self.k.is_cuda and {*map(type, (self.k, *rows))} <= {torch.Tensor, torch.nn.Parameter}:
            store = [x.untyped_storage().data_ptr() for x in (self.k, self.v)]
            if not any(x.untyped_storage().data_ptr() in store for x in rows):
                # V of another type or device is converted as a copy would.
                if prefix_v.dtype != torch.float16 or prefix_v.device != self.k.device:
                    rows[1] = prefix_v.to(self.k.device, torch.float16)
                rows = [x if x.stride(-1) == 1 else x.contiguous() for x in rows]
                if pages:
                    write_prefix_(self.k, self.v, *rows, pages)
                return
        for i, page in enumerate(pages):
            n = min(16, prefix_k.shape[0] - 16 * i)
            self.k[page, :n].copy_(prefix_k[16 * i:16 * i + n])
            self.v[page, :n].copy_(prefix_v[16 * i:16 * i + n])

    def fork(self, source: int) -> int:
        return self.owner.fork(source)

    def checkpoint(self, request: int) -> Snapshot:
        return self.owner.checkpoint(request)

    def rollback(self, snapshot: Snapshot) -> None:
        self.owner.rollback(snapshot)

    def accept(self, snapshot: Snapshot) -> None:
        self.owner.accept(snapshot)

    def _upload(self, *lists) -> tuple[torch.Tensor, ...]:
        """The lists as int32 tensors on the pool's device, all of them parts
        of one.  The values go in kernel arguments; a pool that is not on the
        GPU or holds no memory at all (fake tensors, also on a machine without
        a GPU), entries that are not plain integers, and a stream under capture,
        where the values would be frozen into the graph and a copy raises
        instead, take a copy from host memory.  A step of eight requests of 2053
        tokens (eight verify calls, one commit_many, rollbacks) takes 335 us,
        611 with a copy per list and page-by-page bookkeeping."""
        values = [x for part in lists for x in part]
        if (self.k.is_cuda and type(self.k) is torch.Tensor
                and set(map(type, values)) == {int} and not torch.cuda.is_current_stream_capturing()):
            flat = int_tensor(self.k, values)
        else:
            flat = torch.tensor(values, dtype=torch.int32).to(self.k.device)
        return flat.split([len(part) for part in lists])

    def verify(self, request: int, q: torch.Tensor, draft_k: torch.Tensor,
               draft_v: torch.Tensor, parent: torch.Tensor) -> torch.Tensor:
        """Verify one request; draft inputs have leading batch dimension 1."""
        pages = self.owner.pages[request] or [0]  # unused when the prefix is empty
        table, length = self._upload(pages, [self.owner.lengths[request]])
        return tree_verify(q, self.k, self.v, table.unsqueeze(0), length, draft_k, draft_v,
                           parent)

    def commit(self, request: int, path: list[int], draft_k: torch.Tensor,
               draft_v: torch.Tensor) -> CommitPlan:
        """Append an accepted root-to-leaf path, preserving shared pages."""
        if not path or len(path) > draft_k.shape[1]:
            raise ValueError("path is empty or longer than draft")
        if draft_k.shape != draft_v.shape or draft_k.shape[0] != 1:
            raise ValueError("draft K/V must match and have batch size 1")
        if any(node < 0 or node >= draft_k.shape[1] for node in path):
            raise ValueError("path node out of range")
        plan = self.owner.plan_commit(request, len(path))
        *pair, nodes, pages, slots = self._upload(*([p] for p in plan.cow or ()), path,
                                                  plan.dest_pages, plan.dest_slots)
        if pair:
            copy_pages_(self.k, self.v, *pair)
        commit_path_(self.k, self.v, draft_k, draft_v, nodes, pages, slots, 0)
        return plan

    def commit_many(self, requests: list[int], paths: list[list[int]],
                    draft_k: torch.Tensor, draft_v: torch.Tensor) -> list[CommitPlan]:
        """Commit ``paths[i]`` of request ``requests[i]`` from ``draft_k[i]``.

        Plans are made in list order, as consecutive ``commit`` calls would
        make them.  All clones run first, then all accepted nodes: a page a
        clone reads is shared, so no commit in the batch writes it, and every
        commit target is either a fresh page or one its request owns alone.
        If the pool runs out part way, the plans made so far are still
        executed before the error is raised."""
        if len(requests) != len(paths) or len(set(requests)) != len(requests):
            raise ValueError("requests must be distinct and match paths")
        if draft_k.shape != draft_v.shape or draft_k.shape[0] != len(requests):
            raise ValueError("draft K/V must match and have one row per request")
        nodes = draft_k.shape[1]
        for path in paths:
            if not path or len(path) > nodes:
                raise ValueError("path is empty or longer than draft")
            if any(node < 0 or node >= nodes for node in path):
                raise ValueError("path node out of range")
        plans: list[CommitPlan] = []
        error = None
        for request, path in zip(requests, paths):
            try:
                plans.append(self.owner.plan_commit(request, len(path)))
            except RuntimeError as exc:  # pool exhausted: run what was planned
                error = exc
                break
        self._run_plans(plans, paths, draft_k, draft_v)
        if error is not None:
            raise error
        return plans

    def extend(self, requests: list[int], counts: list[int], q: torch.Tensor,
               k: torch.Tensor, v: torch.Tensor, *, share: bool = False, **options) -> torch.Tensor:
        """Append ``counts[i]`` new tokens to request ``requests[i]`` and attend.

        ``k`` and ``v`` [tokens, KV heads, dim] hold the new tokens' rows,
        request after request, and ``q`` [tokens, query heads, dim] their
        queries; the result is ``chunk_attention`` of them over the requests'
        pages, the new tokens included (``options`` are its keywords).  Pages
        are planned as consecutive commits would take them: shared partial
        pages are cloned first.  A pool without room for all of it raises
        before anything changes, and so does a stream under capture; a call that
        fails later leaves pages and lengths as before it.  A count may be zero.

        ``share``: pages that requests next to each other in the list begin with in
        common (forks of one prompt) are read once for all of them, where that spares a
        quarter of what is read; the result is the same up to rounding, and elsewhere to
        the bit."""
        if len(requests) != len(counts) or len(set(requests)) != len(requests) or not requests:
            raise ValueError("requests must be distinct and match counts")
        total = sum(counts)
        if any(n < 0 for n in counts) or total >= 1 << 27:
            raise ValueError("counts must not be negative, and below 2**27 in all")
        shape = (total, *self.k.shape[2:])
        if tuple(k.shape) != shape or tuple(v.shape) != shape:
            raise ValueError("k and v must have one row of the cache's heads per new token")
        if (q.ndim != 3 or q.shape[0] != total or q.shape[2] != shape[2] or q.shape[1] < 1
                or q.shape[1] % shape[1] or q.shape[1] > 4096):
            raise ValueError("q must have one row of query heads per new token")
        if any(x.dtype != self.dtype or x.device != self.k.device for x in (q, k, v)):
            raise ValueError("q, k and v must have the cache's type and device")
        if not self.k.is_cuda:
            raise ValueError("extend needs a cache on the GPU")
        if any(x.requires_grad and torch.is_grad_enabled() or unpack_dual(x).tangent is not None
               for x in (*self._pools(), q, k, v)):
            raise ValueError("extend is not differentiable: detach q, k and v, or use no_grad")
        plain = {*map(type, (*self._pools(), q, k, v))} <= {torch.Tensor, torch.nn.Parameter}
        if plain and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("extend cannot be captured: its pages are planned on the host, "
                               "once per call; capture build_tables, append_kv_ and chunk_attention")
        q, k, v = (x if x.stride(-1) == 1 else x.contiguous() for x in (q, k, v))
        # Rows that are views of the pool are read before it is written: of one
        # storage with it, or, where all are plain tensors and have an address, of
        # another one of the same memory.

        def store(x: torch.Tensor) -> int:
            return x.untyped_storage().data_ptr() if plain else x.untyped_storage()._cdata

        pools = [store(x) for x in self._pools()]
        q, k, v = (x.clone() if store(x) in pools else x for x in (q, k, v))
        if options:  # refused here, before any page is taken
            empty, first = options, options.get("first")
            if first is not None:
                if tuple(first.shape) != (total,):
                    raise ValueError("first must have one entry per new token")
                # The tensor of the call below; its empty slice is contiguous in any case.
                options["first"] = first = first.contiguous()
                empty = options | {"first": first[:0]}
            none = self._upload([-1] * len(requests), [0] * len(requests), [0] * (len(requests) + 1))
            self._attend(q[:0], none[0].unsqueeze(1), *none[1:], (), **empty)
        owner = self.owner
        # Requests that share a partial last page: all but the last to write
        # it take a clone.
        holders: dict[int, int] = {}
        needed = 0
        for request, n in zip(requests, counts):
            length, pages = owner.lengths[request], owner.pages[request]
            if not n:
                continue
            needed += -(-(length + n) // 16) - len(pages)
            if length % 16:
                last = pages[-1]
                left = holders.setdefault(last, owner.refcount[last])
                if left > 1:
                    needed += 1
                    holders[last] = left - 1
        if needed > len(owner.free):
            raise RuntimeError("KV page pool exhausted")
        plans = [owner.plan_commit(request, n) for request, n in zip(requests, counts) if n]
        try:
            clones = [plan.cow for plan in plans if plan.cow is not None]
            lists = [owner.pages[request] for request in requests]
            lengths = [owner.lengths[request] for request in requests]
            groups = ()
            if share:
                groups = _worth_reading_once(*owner.shared_prefixes(requests), lengths, counts,
                                             options.get("window", 0))
            old, fresh, ids, length, count, *groups = self._upload(
                [old for old, _ in clones], [fresh for _, fresh in clones],
                [page for pages in lists for page in pages], lengths, counts, *groups)
            if clones:
                self._clone(old, fresh)
            width = max(1, *(len(pages) for pages in lists))
            table, starts, slots, _ = build_tables(ids, length, count, width, total)
            self._append(k, v, slots)
            return self._attend(q, table, length, starts, tuple(groups), **options)
        except BaseException:
            # An allocation that failed, say.  Rows written so far lie behind
            # every holder's length, or in pages that are free again.
            for plan in reversed(plans):
                owner.undo_commit(plan)
            raise

    def _run_plans(self, plans, paths, draft_k, draft_v) -> None:
        if not plans:
            return
        cows = [p.cow for p in plans if p.cow is not None]
        # copy_pages_ runs every pair at once: a destination must be fresh,
        # so distinct and never another pair's source (the page owner only
        # hands out free pages as clone targets).
        dsts = [fresh for _, fresh in cows]
        if len(set(dsts)) != len(dsts) or set(dsts) & {old for old, _ in cows}:
            raise RuntimeError("copy-on-write clones overlap")
        old, fresh, *table = self._upload(
            [old for old, _ in cows], dsts,
            [i for i, path in zip(range(len(plans)), paths) for _ in path],
            [node for _, path in zip(plans, paths) for node in path],
            [page for p in plans for page in p.dest_pages],
            [slot for p in plans for slot in p.dest_slots])
        if cows:
            copy_pages_(self.k, self.v, old, fresh)
        commit_paths_(self.k, self.v, draft_k, draft_v, *table)


class Fp8Cache(PagedTreeCache):
    """Requests of ordinary tokens over a pool of 8 bits (see ``append_fp8_kv_``), with
    rows, queries and outputs of ``dtype``: ``new``, ``fork``, ``checkpoint``,
    ``rollback``, ``accept`` and ``extend`` as above, and ``read``.  Trees of draft
    tokens are verified over a 16-bit pool: ``PagedTreeCache.new`` takes what ``read``
    gives."""

    def __init__(self, physical_pages: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device: str = "cuda"):
        if head_dim not in (64, 128) or physical_pages < 1 or kv_heads < 1:
            raise ValueError("head_dim must be 64/128; physical_pages and kv_heads must be positive")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError("dtype must be FP16 or BF16")
        self.owner = PageOwner(physical_pages)
        self._dtype = dtype

        def zeros(*shape: int, type: torch.dtype) -> torch.Tensor:
            return torch.zeros(shape, device=device, dtype=torch.uint8).view(type)

        self.k, self.v = (zeros(physical_pages, 16, kv_heads, head_dim, type=torch.float8_e4m3fn)
                          for _ in range(2))
        self.scale_k, self.scale_v = (zeros(physical_pages, kv_heads, 16, head_dim // 32,
                                            type=torch.float8_e8m0fnu) for _ in range(2))

    @property
    def dtype(self) -> torch.dtype:
        return self._dtype

    def _pools(self) -> tuple[torch.Tensor, ...]:
        return self.k, self.scale_k, self.v, self.scale_v

    def _clone(self, old: torch.Tensor, fresh: torch.Tensor) -> None:
        copy_fp8_pages_(*self._pools(), old, fresh)

    def _append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        append_fp8_kv_(*self._pools(), k, v, slots)

    def _attend(self, q: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
                starts: torch.Tensor, groups: tuple[torch.Tensor, ...], **options) -> torch.Tensor:
        return fp8_chunk_attention(q, *self._pools(), table, lengths, starts, **options)

    def _slots(self, request: int) -> torch.Tensor:
        """The slots of all of a request's tokens."""
        pages, tokens = self.owner.pages[request], self.owner.lengths[request]
        ids, length = self._upload(pages, [tokens])
        return build_tables(ids, length, length, max(1, len(pages)), tokens)[2]

    def new(self, prefix_k: torch.Tensor, prefix_v: torch.Tensor) -> int:
        """Create one request from [tokens, KV heads, head dim] tensors of the cache's type."""
        if prefix_k.shape != prefix_v.shape or prefix_k.ndim != 3:
            raise ValueError("prefix K/V shapes must match [tokens, heads, dim]")
        if any(x.dtype != self.dtype or x.device != self.k.device for x in (prefix_k, prefix_v)):
            raise ValueError("prefix must have the cache's type and device")
        if tuple(prefix_k.shape[1:]) != tuple(self.k.shape[2:]):
            raise ValueError("prefix head shape differs from cache")
        if any(x.requires_grad and torch.is_grad_enabled() or unpack_dual(x).tangent is not None
               for x in (prefix_k, prefix_v)):
            raise ValueError("the cache is not differentiable: detach the prefix, or use no_grad")
        rows = [x if x.stride(-1) == 1 else x.contiguous() for x in (prefix_k, prefix_v)]
        request = self.owner.new(prefix_k.shape[0])
        try:
            self._append(*rows, self._slots(request))
        except BaseException:  # the pages are free again, in the order they had
            for page in reversed(self.owner.pages.pop(request)):
                self.owner.release(page)
            del self.owner.lengths[request]
            raise
        return request

    def read(self, request: int) -> tuple[torch.Tensor, torch.Tensor]:
        """All of a request's K and V rows in the cache's type, [tokens, KV heads, head dim]."""
        return read_fp8_kv(*self._pools(), self._slots(request), self.dtype)

    def extend(self, requests: list[int], counts: list[int], q: torch.Tensor,
               k: torch.Tensor, v: torch.Tensor, *, share: bool = False, **options) -> torch.Tensor:
        """As ``PagedTreeCache.extend``, but every request reads its own pages."""
        if share:
            raise ValueError("share needs a 16-bit pool")
        return super().extend(requests, counts, q, k, v, **options)

    def verify(self, *_, **__):
        raise NotImplementedError("trees are verified over a 16-bit pool: PagedTreeCache")

    commit = commit_many = verify
