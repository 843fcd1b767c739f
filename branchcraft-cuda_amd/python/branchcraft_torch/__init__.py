"""PyTorch dispatcher ops for Branchcraft's MI355X (gfx950) kernels.

Importing this module loads ``_C.so`` (built in-tree by
``branchcraft-cuda_amd/build.py``) which registers ``torch.ops.branchcraft``
with the reference's schemas (bindings/torch_ops.cpp:144-148 of
Haaziq386/branchcraft-cuda) plus ``paged_decode`` (the reference's C++
``branchcraft::decode``), ``copy_pages_``, ``commit_paths_`` and the chunk ops
(``build_tables``, ``append_kv_``, ``chunk_attention``), an 8-bit cache
(``append_fp8_kv_``, ``copy_fp8_pages_``, ``read_fp8_kv``, ``fp8_chunk_attention``)
and attention for forks (``shared_chunk_attention``).  There is no CPU or Python fallback: a missing
extension raises ImportError, and the ops have only a GPU implementation.

FakeTensor implementations follow python/branchcraft_torch/__init__.py:18-31
of the reference so that ``torch.compile`` can trace the ops.
"""

from pathlib import Path

import torch

_library = Path(__file__).with_name("_C.so")
if not _library.exists():
    raise ImportError(
        "Branchcraft HIP extension is missing; run `python branchcraft-cuda_amd/build.py`")
torch.ops.load_library(str(_library))
LIBRARY_PATH = str(_library)


@torch.library.register_fake("branchcraft::tree_verify")
def _fake_tree_verify(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent):
    return q.new_empty(q.shape, dtype=torch.float32)


@torch.library.register_fake("branchcraft::packed_decode_out")
def _fake_packed_decode_out(q, packed_kv, pages, lengths, output, scale):
    return output


@torch.library.register_fake("branchcraft::paged_decode")
def _fake_paged_decode(q, k, v, pages, lengths, splits=0):
    return q.new_empty(q.shape, dtype=torch.float32)


@torch.library.register_fake("branchcraft::commit_path_")
def _fake_commit_path(cache_k, cache_v, draft_k, draft_v, path_nodes, dest_pages,
                      dest_slots, request):
    return None


@torch.library.register_fake("branchcraft::copy_pages_")
def _fake_copy_pages(cache_k, cache_v, src_pages, dst_pages):
    return None


@torch.library.register_fake("branchcraft::commit_paths_")
def _fake_commit_paths(cache_k, cache_v, draft_k, draft_v, requests, path_nodes,
                       dest_pages, dest_slots):
    return None


@torch.library.register_fake("branchcraft::write_prefix_")
def _fake_write_prefix(cache_k, cache_v, k, v, pages):
    return None


@torch.library.register_fake("branchcraft::int_tensor")
def _fake_int_tensor(like, values):
    return like.new_empty((len(values),), dtype=torch.int32)


@torch.library.register_fake("branchcraft::build_tables")
def _fake_build_tables(page_ids, lengths, counts, max_pages, tokens):
    batch = lengths.shape[0]
    return tuple(lengths.new_empty(shape)
                 for shape in ((batch, max_pages), (batch + 1,), (tokens,), (tokens,)))


@torch.library.register_fake("branchcraft::append_kv_")
def _fake_append_kv(cache_k, cache_v, k, v, slots):
    return None


@torch.library.register_fake("branchcraft::chunk_attention")
def _fake_chunk_attention(q, k, v, pages, lengths, starts, scale=None, causal=True, window=0,
                          cap=0.0, slopes=None, prefix=None, first=None):
    return q.new_empty(q.shape)


@torch.library.register_fake("branchcraft::append_fp8_kv_")
def _fake_append_fp8_kv(cache_k, scale_k, cache_v, scale_v, k, v, slots):
    return None


@torch.library.register_fake("branchcraft::copy_fp8_pages_")
def _fake_copy_fp8_pages(cache_k, scale_k, cache_v, scale_v, src_pages, dst_pages):
    return None


@torch.library.register_fake("branchcraft::read_fp8_kv")
def _fake_read_fp8_kv(cache_k, scale_k, cache_v, scale_v, slots, dtype):
    size = (slots.shape[0], *cache_k.shape[2:])
    return tuple(cache_k.new_empty(size, dtype=dtype) for _ in range(2))


@torch.library.register_fake("branchcraft::fp8_chunk_attention")
def _fake_fp8_chunk_attention(q, k, scale_k, v, scale_v, pages, lengths, starts, scale=None,
                              causal=True, window=0, cap=0.0, slopes=None, prefix=None, first=None):
    return q.new_empty(q.shape)


@torch.library.register_fake("branchcraft::shared_chunk_attention")
def _fake_shared_chunk_attention(q, k, v, pages, lengths, starts, groups, shared, scale=None,
                                 causal=True, window=0, cap=0.0, slopes=None, prefix=None, first=None):
    return q.new_empty(q.shape)


# The ops themselves: through the packet a call costs its host 0.4 us more.
_build_tables = torch.ops.branchcraft.build_tables.default
_append_kv = torch.ops.branchcraft.append_kv_.default
_chunk_attention = torch.ops.branchcraft.chunk_attention.default
_append_fp8_kv = torch.ops.branchcraft.append_fp8_kv_.default
_read_fp8_kv = torch.ops.branchcraft.read_fp8_kv.default
_fp8_chunk_attention = torch.ops.branchcraft.fp8_chunk_attention.default
_shared_chunk_attention = torch.ops.branchcraft.shared_chunk_attention.default


def tree_verify(q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent):
    """FP32 [batch, node, query head, dim] outputs; every node attends to its
    request's paged prefix and its own ancestor chain (itself included)."""
    return torch.ops.branchcraft.tree_verify(
        q, prefix_k, prefix_v, pages, lengths, draft_k, draft_v, parent)


def packed_decode_out(q, packed_kv, pages, lengths, output, scale):
    """Decode into a preallocated FP16 output (safe for HIP graph capture).

    ``packed_kv`` is the logical [pages, kv_heads, 16, 2*dim] view of a vLLM
    cache (any outer strides) or a [pages, 2, 16, kv_heads, dim] tensor."""
    return torch.ops.branchcraft.packed_decode_out(
        q, packed_kv, pages, lengths, output, scale)


def paged_decode(q, k, v, pages, lengths, splits=0):
    """Paged GQA decode (the reference's C++ ``branchcraft::decode``): FP32
    [batch, query head, dim] output over K/V pages [P, 16, kv_heads, dim].
    ``splits=0`` picks the split count from the shape (no host sync)."""
    return torch.ops.branchcraft.paged_decode(q, k, v, pages, lengths, splits)


def commit_path_(cache_k, cache_v, draft_k, draft_v, path_nodes, dest_pages,
                 dest_slots, request):
    """Write accepted draft K/V to preallocated physical destinations."""
    return torch.ops.branchcraft.commit_path_(
        cache_k, cache_v, draft_k, draft_v, path_nodes, dest_pages, dest_slots, request)


def copy_pages_(cache_k, cache_v, src_pages, dst_pages):
    """Clone whole pages (K and V): cache[dst[i]] <- cache[src[i]].  All
    pairs copy at once: destinations must be distinct and none may also be
    a source."""
    return torch.ops.branchcraft.copy_pages_(cache_k, cache_v, src_pages, dst_pages)


def commit_paths_(cache_k, cache_v, draft_k, draft_v, requests, path_nodes, dest_pages,
                  dest_slots):
    """Commit the accepted nodes of several requests in one launch: entry i
    writes draft[requests[i], path_nodes[i]] to (dest_pages[i], dest_slots[i])."""
    return torch.ops.branchcraft.commit_paths_(
        cache_k, cache_v, draft_k, draft_v, requests, path_nodes, dest_pages, dest_slots)


def write_prefix_(cache_k, cache_v, k, v, pages):
    """Fill the pages of a host-side list with a prompt's K and V rows
    ([tokens, KV heads, dim], any strides with a contiguous last dim): token t
    goes to (pages[t // 16], t % 16).  Pages must be distinct."""
    return torch.ops.branchcraft.write_prefix_(cache_k, cache_v, k, v, pages)


def int_tensor(like, values):
    """Host integers as an int32 tensor on ``like``'s device, written in
    stream order: the host waits for nothing."""
    return torch.ops.branchcraft.int_tensor(like, values)


def build_tables(page_ids, lengths, counts, max_pages, tokens):
    """Block table, row offsets, slot map and positions of a step, on the GPU:
    ``(pages [batch, max_pages], starts [batch + 1], slots [tokens], positions
    [tokens])``, all int32.  Request b has ``lengths[b]`` tokens, the last
    ``counts[b]`` of them new, and its ceil(length / 16) page ids follow those of
    the request before it in ``page_ids``.  -1 stands behind a request's pages,
    in rows behind the last request, and for rows without a slot.  ``tokens``
    should hold every new token: of a request that is cut, the first rows are
    placed, and ``chunk_attention``, which takes a request's rows as its last
    tokens, must not be used for it."""
    return _build_tables(page_ids, lengths, counts, max_pages, tokens)


def append_kv_(cache_k, cache_v, k, v, slots):
    """Write new tokens' K and V rows ([tokens, KV heads, dim], FP16 or BF16, any
    strides with a contiguous last dim) to the slots of ``build_tables``; -1 and
    slots outside the pool are skipped.  The pools may be strided views, such
    as the two halves of a packed cache."""
    return _append_kv(cache_k, cache_v, k, v, slots)


def chunk_attention(q, k, v, pages, lengths, starts, *, scale=None, causal=True, window=0,
                    cap=0.0, slopes=None, prefix=None, first=None):
    """Attention of every request's new tokens over its pages: [tokens, query
    heads, dim] in the inputs' type (FP16 or BF16).

    Request b's rows of ``q`` are ``starts[b] .. starts[b+1] - 1``, the last of
    its ``lengths[b]`` tokens, whose K and V the pages already hold.  The row at
    place p sees the tokens up to p (all with ``causal=False``; at least the
    first ``prefix[b]`` with a prefix), from ``p - window + 1`` with a window,
    from ``first[row]`` with documents.  Scores are ``scale * q.k`` (default
    1/sqrt(dim)), then ``cap * tanh(score / cap)``, then minus ``slopes[head] *
    |p - token|``.  Rows that see nothing, and rows of no request, are zero.
    The softmax weights are rounded to the inputs' type for the product with V
    (32-bit for tensors not aligned to 16 bytes, which are much slower).
    Not differentiable: tensors that autograd tracks are refused."""
    return _chunk_attention(q, k, v, pages, lengths, starts, scale, causal, window, cap, slopes,
                            prefix, first)


def append_fp8_kv_(cache_k, scale_k, cache_v, scale_v, k, v, slots):
    """Round new tokens' K and V rows (as ``append_kv_`` takes them) to 8 bits and
    write them to the slots of an 8-bit cache: codes ``float8_e4m3fn`` [pages, 16,
    KV heads, dim] (any strides of whole 16 bytes) and, contiguous, scales
    ``float8_e8m0fnu`` [pages, KV heads, 16, dim / 32].  A value is its code times
    the scale of its 32, the least power of two with which they stay within 448.
    Infinities and NaN become NaN."""
    return _append_fp8_kv(cache_k, scale_k, cache_v, scale_v, k, v, slots)


def copy_fp8_pages_(cache_k, scale_k, cache_v, scale_v, src_pages, dst_pages):
    """Copy whole pages of an 8-bit cache, codes and scales, as ``copy_pages_`` copies
    those of a 16-bit one: every pair at once, so destinations must be distinct and
    none may also be a source."""
    return torch.ops.branchcraft.copy_fp8_pages_(cache_k, scale_k, cache_v, scale_v, src_pages, dst_pages)


def read_fp8_kv(cache_k, scale_k, cache_v, scale_v, slots, dtype):
    """Rows of an 8-bit cache in FP16 or BF16, ``(k, v)``, each [len(slots), KV heads,
    dim]; zeros for slots of -1 and outside the pool.  What was written from a type
    comes back in it as exactly code times scale."""
    return _read_fp8_kv(cache_k, scale_k, cache_v, scale_v, slots, dtype)


def fp8_chunk_attention(q, k, scale_k, v, scale_v, pages, lengths, starts, *, scale=None, causal=True,
                        window=0, cap=0.0, slopes=None, prefix=None, first=None):
    """``chunk_attention`` over an 8-bit cache (see ``append_fp8_kv_``), in q's type,
    to which the cache's values are rounded (exactly, where they were written from
    it)."""
    return _fp8_chunk_attention(q, k, scale_k, v, scale_v, pages, lengths, starts, scale, causal, window,
                                cap, slopes, prefix, first)


def shared_chunk_attention(q, k, v, pages, lengths, starts, groups, shared, *, scale=None, causal=True,
                           window=0, cap=0.0, slopes=None, prefix=None, first=None):
    """``chunk_attention`` for requests that begin alike, such as forks: requests
    ``groups[g] .. groups[g+1] - 1`` have their first ``shared[g]`` tokens in pages
    of the same contents, which are read once for all of them (those of the first
    one) where the sizes of the call say that this pays; elsewhere each request's are.
    ``groups`` (not decreasing) and ``shared`` are int32 tensors on the GPU; requests
    outside all groups share nothing.  The results are ``chunk_attention``'s up to
    rounding.  What is shared is not looked at for that choice: groups of less than some
    256 tokens cost more than they spare (``PagedTreeCache.extend`` leaves them out)."""
    return _shared_chunk_attention(q, k, v, pages, lengths, starts, groups, shared, scale, causal, window,
                                   cap, slopes, prefix, first)


__all__ = ["tree_verify", "packed_decode_out", "paged_decode",
           "commit_path_", "copy_pages_", "commit_paths_", "write_prefix_", "int_tensor",
           "build_tables", "append_kv_", "chunk_attention", "append_fp8_kv_", "copy_fp8_pages_", "read_fp8_kv",
           "fp8_chunk_attention", "shared_chunk_attention",
           "LIBRARY_PATH"]
