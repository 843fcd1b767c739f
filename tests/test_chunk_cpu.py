"""Refusals of the chunk entry points, before any launch, and their fake
implementations: no GPU needed."""

import math

import pytest
import torch

import branchcraft_capi as capi

INVALID = capi.BC_ERROR_INVALID_VALUE
FAKE = 0x1000  # a non-null address; never dereferenced on the rejection path


def _shape(**kw):
    base = dict(batch=2, query_heads=32, kv_heads=8, dim=128, max_pages=4, physical_pages=16)
    return capi.Shape(**(base | kw))


def _chunk(**kw):
    base = dict(q=FAKE, k=FAKE, v=FAKE, pages=FAKE, lengths=FAKE, starts=FAKE, output=FAKE,
                q_strides=capi.RowStrides(4096, 128), k_strides=capi.PoolStrides(16384, 1024, 128),
                v_strides=capi.PoolStrides(16384, 1024, 128), tokens=3, dtype=0, causal=1, scale=0.1)
    return capi.ChunkInputs(**(base | kw))


BAD_SHAPES = [dict(batch=0), dict(query_heads=0), dict(kv_heads=0), dict(query_heads=30), dict(dim=96),
              dict(max_pages=0), dict(physical_pages=0), dict(query_heads=8192, kv_heads=8192),
              dict(max_pages=(1 << 27) - 15)]
BAD_INPUTS = [dict(q=None), dict(k=None), dict(v=None), dict(pages=None), dict(lengths=None),
              dict(starts=None), dict(output=None), dict(tokens=-1), dict(window=-1), dict(dtype=2),
              dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf), dict(cap=-1.0),
              dict(cap=math.nan), dict(cap=math.inf), dict(cap=1e-13), dict(cap=1e13), dict(scale=1e-13), dict(scale=1e13),
              dict(q_strides=capi.RowStrides(-1, 128)),
              dict(k_strides=capi.PoolStrides(1, -1, 1)), dict(v_strides=capi.PoolStrides(1, 1, -1))]


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_chunk_rejects_shapes(bad):
    assert capi.load().bc_chunk_attention(_shape(**bad), _chunk(), None, 0, None) == INVALID
    assert capi.load().bc_chunk_attention_workspace_size(_shape(**bad), 3) == 0


@pytest.mark.parametrize("bad", BAD_INPUTS, ids=str)
def test_chunk_rejects_inputs(bad):
    assert capi.load().bc_chunk_attention(_shape(), _chunk(**bad), None, 0, None) == INVALID


def test_no_rows_are_no_launch():
    lib = capi.load()
    assert lib.bc_chunk_attention(_shape(), _chunk(tokens=0, q=None, output=None), None, 0, None) == 0
    row, pool = capi.RowStrides(1024, 128), capi.PoolStrides(16384, 1024, 128)
    assert lib.bc_append_kv(_shape(), FAKE, FAKE, row, row, FAKE, FAKE, pool, pool, FAKE, 0, None) == 0


def test_append_rejects():
    lib = capi.load()
    row, pool = capi.RowStrides(1024, 128), capi.PoolStrides(16384, 1024, 128)
    good = [_shape(), FAKE, FAKE, row, row, FAKE, FAKE, pool, pool, FAKE, 3, None]
    for at, bad in [(0, _shape(dim=80)), (0, _shape(kv_heads=0)), (0, _shape(kv_heads=4097)),
                    (0, _shape(physical_pages=0)), (1, None),
                    (2, None), (5, None), (6, None), (9, None), (10, -1), (3, capi.RowStrides(-8, 1)),
                    (4, capi.RowStrides(8, -1)), (7, capi.PoolStrides(-1, 1, 1)),
                    (8, capi.PoolStrides(1, 1, -1))]:
        args = list(good)
        args[at] = bad
        assert lib.bc_append_kv(*args) == INVALID, (at, bad)


def test_build_tables_rejects():
    lib = capi.load()
    good = [FAKE, 9, FAKE, FAKE, 2, 4, 3, FAKE, FAKE, FAKE, FAKE, None]
    for at, bad in [(0, None), (1, -1), (2, None), (3, None), (4, 0), (5, 0), (6, -1), (7, None), (8, None),
                    (9, None), (10, None), (5, 2**28), (5, 2**27 - 15), (6, 2**28)]:
        args = list(good)
        args[at] = bad
        assert lib.bc_build_tables(*args) == INVALID, (at, bad)


def test_fake_tensors_and_versions():
    import branchcraft_torch as bt
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        ints = [torch.zeros(n, device="cuda", dtype=torch.int32) for n in (9, 3, 3)]
        pages, starts, slots, positions = bt.build_tables(*ints, 5, 7)
        assert [tuple(x.shape) for x in (pages, starts, slots, positions)] == [(3, 5), (4,), (7,), (7,)]
        pools = [torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        rows = [torch.zeros(7, 2, 64, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        bt.append_kv_(*pools, *rows, slots)
        assert [x._version for x in (*pools, *rows)] == [1, 1, 0, 0]
        q = torch.zeros(7, 4, 64, device="cuda", dtype=torch.bfloat16)
        out = bt.chunk_attention(q, *pools, pages, ints[1], starts, cap=3.0)
        assert out.shape == q.shape and out.dtype == q.dtype


def test_what_autograd_tracks_is_refused():
    import branchcraft_torch as bt
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        pools = [torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
        rows = [torch.zeros(7, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2)]
        slots = torch.zeros(7, device="cuda", dtype=torch.int32)
        for at in range(4):
            args = [*pools, *rows]
            args[at] = args[at].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="not differentiable"):
                bt.append_kv_(*args, slots)
            with torch.no_grad():
                bt.append_kv_(*args, slots)
        q = torch.zeros(7, 4, 64, device="cuda", dtype=torch.float16)
        ints = [torch.zeros(n, device="cuda", dtype=torch.int32) for n in ((1, 4), (1,), (2,))]
        slopes = torch.zeros(4, device="cuda")
        for at in range(4):
            args = [q, *pools, slopes]
            args[at] = args[at].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="not differentiable"):
                bt.chunk_attention(*args[:3], *ints, slopes=args[3])
            with torch.no_grad():
                assert not bt.chunk_attention(*args[:3], *ints, slopes=args[3]).requires_grad


def test_extend_on_fake_tensors():
    """Page tables and shapes without a GPU; no warning about an address."""
    import warnings
    from branchcraft_torch.transaction import PagedTreeCache
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode(), warnings.catch_warnings():
        warnings.simplefilter("error")
        cache = PagedTreeCache(8, 2, 64)
        rows = torch.zeros(20, 2, 64, device="cuda", dtype=torch.float16)
        q = torch.zeros(6, 4, 64, device="cuda", dtype=torch.float16)
        a = cache.new(rows, rows)
        b = cache.fork(a)
        assert cache.extend([a, b], [3, 3], q, rows[:6], rows[:6], cap=3.0).shape == (6, 4, 64)
        assert cache.lengths == {a: 23, b: 23} and cache.pages[a][1] != cache.pages[b][1]


def test_cpu_tensors_have_no_implementation():
    import branchcraft_torch as bt
    ints = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        bt.build_tables(ints, ints, ints, 1, 1)


def test_matrix_results_are_waited_for():
    """Wait states between a matrix instruction of the tile kernels and the
    vector instructions that touch its registers, over branches too: the
    compiler keeps twelve to a read of the result, and ten are the fewest that
    an accumulator's next writer has passed with."""
    import shutil
    import tempfile
    from pathlib import Path

    import asm_hazards as H
    if not (shutil.which("hipcc") or Path("/opt/rocm/bin/hipcc").exists()):
        pytest.skip("hipcc not available")
    with tempfile.TemporaryDirectory() as tmp:
        kernels = H.kernels(H.compile_device_asm(H.CSRC / "chunk.hip", Path(tmp)))
    found = 0
    for name, lines in kernels.items():
        insts, labels = H.parse(lines)
        if not any(op.startswith("v_mfma") for op, _ in insts):
            continue
        found += 1
        best = H.scan(insts, labels, window=12)
        assert best.get("RAW", 12) >= 12 and best.get("WAW", 10) >= 10 and best.get("WARC", 10) >= 10, (name, best)
    assert found == 12
