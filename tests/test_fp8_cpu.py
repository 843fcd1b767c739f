"""Refusals of the 8-bit cache's and the shared-prefix entry points, before any launch,
their fake implementations, and the page owner's groups: no GPU needed."""

import random

import pytest
import torch

import branchcraft_capi as capi
from test_chunk_cpu import BAD_INPUTS, BAD_SHAPES, FAKE, INVALID, _chunk, _shape


def _pool(**kw):
    strides = capi.PoolStrides(16 * 8 * 128, 8 * 128, 128)
    base = dict(k=FAKE, v=FAKE, k_scale=FAKE, v_scale=FAKE, k_strides=strides, v_strides=strides)
    return capi.Fp8Pool(**(base | kw))


BAD_POOLS = [dict(k=None), dict(v=None), dict(k_scale=None), dict(v_scale=None), dict(k=FAKE + 8), dict(v=FAKE + 1),
             dict(k_scale=FAKE + 2), dict(v_scale=FAKE + 1), dict(k_strides=capi.PoolStrides(2048, 136, 128)),
             dict(v_strides=capi.PoolStrides(2056, 128, 64)), dict(k_strides=capi.PoolStrides(-16, 128, 16)),
             dict(v_strides=capi.PoolStrides(2048, 128, -16))]
BAD_POOL_SHAPES = [dict(dim=96), dict(kv_heads=0), dict(kv_heads=4097), dict(physical_pages=0)]


def test_rows_are_refused():
    lib = capi.load()
    row = capi.RowStrides(1024, 128)
    good = [_shape(), FAKE, FAKE, row, row, 0, _pool(), FAKE, 3, None]
    bad = [(0, _shape(**x)) for x in BAD_POOL_SHAPES] + [(6, _pool(**x)) for x in BAD_POOLS]
    bad += [(1, None), (2, None), (3, capi.RowStrides(-8, 8)), (4, capi.RowStrides(8, -8)), (5, 2), (5, -1),
            (7, None), (8, -1)]
    for at, x in bad:
        args = list(good)
        args[at] = x
        assert lib.bc_append_fp8_kv(*args) == INVALID, (at, x)
    good[8] = 0
    assert lib.bc_append_fp8_kv(*good) == 0
    good = [_shape(), _pool(), FAKE, 3, 1, FAKE, FAKE, None]
    bad = [(0, _shape(**x)) for x in BAD_POOL_SHAPES] + [(1, _pool(**x)) for x in BAD_POOLS]
    bad += [(2, None), (3, -1), (4, 2), (5, None), (6, None), (5, FAKE + 8), (6, FAKE + 2)]
    for at, x in bad:
        args = list(good)
        args[at] = x
        assert lib.bc_read_fp8_kv(*args) == INVALID, (at, x)
    good[3] = 0
    assert lib.bc_read_fp8_kv(*good) == 0
    good = [_shape(), _pool(), FAKE, FAKE, 3, None]
    bad = [(0, _shape(**x)) for x in BAD_POOL_SHAPES] + [(1, _pool(**x)) for x in BAD_POOLS]
    for at, x in bad + [(2, None), (3, None), (4, -1)]:
        args = list(good)
        args[at] = x
        assert lib.bc_copy_fp8_pages(*args) == INVALID, (at, x)
    assert lib.bc_copy_fp8_pages(*good[:2], None, None, 0, None) == 0


@pytest.mark.parametrize("bad", BAD_SHAPES, ids=str)
def test_shapes_are_refused(bad):
    lib = capi.load()
    assert lib.bc_fp8_chunk_attention(_shape(**bad), _chunk(), FAKE, FAKE, None, 0, None) == INVALID
    assert lib.bc_fp8_chunk_attention_workspace_size(_shape(**bad), 3) == 0
    assert lib.bc_shared_chunk_attention(_shape(**bad), _chunk(), FAKE, FAKE, 1, None, 0, None) == INVALID
    assert lib.bc_shared_chunk_attention_workspace_size(_shape(**bad), 3, 1) == 0


@pytest.mark.parametrize("bad", BAD_INPUTS, ids=str)
def test_inputs_are_refused(bad):
    lib = capi.load()
    assert lib.bc_fp8_chunk_attention(_shape(), _chunk(**bad), FAKE, FAKE, None, 0, None) == INVALID
    assert lib.bc_shared_chunk_attention(_shape(), _chunk(**bad), FAKE, FAKE, 1, None, 0, None) == INVALID


def test_scales_groups_and_alignment_are_refused():
    lib = capi.load()
    for scales in ((None, FAKE), (FAKE, None), (FAKE + 2, FAKE), (FAKE, FAKE + 1)):
        assert lib.bc_fp8_chunk_attention(_shape(), _chunk(), *scales, None, 0, None) == INVALID
    for bad in (dict(k=FAKE + 8), dict(v=FAKE + 4), dict(k_strides=capi.PoolStrides(2048, 136, 128)),
                dict(v_strides=capi.PoolStrides(2048, 128, 8))):
        assert lib.bc_fp8_chunk_attention(_shape(), _chunk(**bad), FAKE, FAKE, None, 0, None) == INVALID
    for groups in ((None, FAKE, 1), (FAKE, None, 1), (FAKE, FAKE, -1), (FAKE, FAKE, 3)):
        assert lib.bc_shared_chunk_attention(_shape(), _chunk(), *groups, None, 0, None) == INVALID
    none = dict(tokens=0, q=None, output=None)
    assert lib.bc_fp8_chunk_attention(_shape(), _chunk(**none), FAKE, FAKE, None, 0, None) == 0
    assert lib.bc_shared_chunk_attention(_shape(), _chunk(**none), FAKE, None, 0, None, 0, None) == 0


def test_workspaces():
    """Sized by shapes alone: nothing where a call never cuts, for shared pages what
    either way of running takes."""
    lib = capi.load()
    long, short = _shape(batch=64, max_pages=2112), _shape(batch=64, max_pages=8)
    assert lib.bc_fp8_chunk_attention_workspace_size(short, 64) == 0
    assert 0 < lib.bc_fp8_chunk_attention_workspace_size(long, 64) < 256 << 20
    assert lib.bc_shared_chunk_attention_workspace_size(short, 64, 1) == 0
    plain = lib.bc_chunk_attention_workspace_size(long, 64)
    assert lib.bc_shared_chunk_attention_workspace_size(long, 64, 0) == plain
    assert plain <= lib.bc_shared_chunk_attention_workspace_size(long, 64, 3) < 256 << 20
    assert lib.bc_shared_chunk_attention_workspace_size(long, 64, 65) == 0


def _fakes(dtype=torch.bfloat16):
    codes = [torch.zeros(4, 16, 2, 64, device="cuda", dtype=torch.uint8).view(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.zeros(4, 2, 16, 2, device="cuda", dtype=torch.uint8).view(torch.float8_e8m0fnu) for _ in range(2)]
    pool = [codes[0], scales[0], codes[1], scales[1]]
    rows = [torch.zeros(7, 2, 64, device="cuda", dtype=dtype) for _ in range(2)]
    ints = [torch.zeros(n, device="cuda", dtype=torch.int32) for n in ((3, 5), (3,), (4,))]
    return pool, rows, torch.zeros(7, device="cuda", dtype=torch.int32), torch.zeros(7, 4, 64, device="cuda", dtype=dtype), ints


def test_fake_tensors_and_versions():
    import branchcraft_torch as bt
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        pool, rows, slots, q, ints = _fakes()
        before = [x._version for x in pool]
        bt.append_fp8_kv_(*pool, *rows, slots)
        assert [x._version - b for x, b in zip(pool, before)] == [1] * 4 and rows[0]._version == 0
        bt.copy_fp8_pages_(*pool, slots, slots)
        assert [x._version - b for x, b in zip(pool, before)] == [2] * 4
        for x in bt.read_fp8_kv(*pool, slots, torch.float16):
            assert x.shape == (7, 2, 64) and x.dtype == torch.float16
        out = bt.fp8_chunk_attention(q, *pool, *ints, cap=3.0, window=4)
        assert out.shape == q.shape and out.dtype == q.dtype
        kv = [torch.zeros(4, 16, 2, 64, device="cuda", dtype=q.dtype) for _ in range(2)]
        groups = [torch.zeros(n, device="cuda", dtype=torch.int32) for n in (2, 1)]
        out = bt.shared_chunk_attention(q, *kv, *ints, *groups, cap=3.0)
        assert out.shape == q.shape and out.dtype == q.dtype


def test_what_autograd_tracks_is_refused():
    import branchcraft_torch as bt
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        pool, rows, slots, q, ints = _fakes()
        slopes = torch.zeros(4, device="cuda")
        kv = [torch.zeros(4, 16, 2, 64, device="cuda", dtype=q.dtype) for _ in range(2)]
        groups = [torch.zeros(n, device="cuda", dtype=torch.int32) for n in (2, 1)]
        for at in range(2):
            args = list(rows)
            args[at] = args[at].clone().requires_grad_()
            with pytest.raises(RuntimeError, match="not differentiable"):
                bt.append_fp8_kv_(*pool, *args, slots)
            with torch.no_grad():
                bt.append_fp8_kv_(*pool, *args, slots)
        for at in range(2):
            a, s = q, slopes
            if at:
                s = s.clone().requires_grad_()
            else:
                a = a.clone().requires_grad_()
            for call in (lambda: bt.fp8_chunk_attention(a, *pool, *ints, slopes=s),
                         lambda: bt.shared_chunk_attention(a, *kv, *ints, *groups, slopes=s)):
                with pytest.raises(RuntimeError, match="not differentiable"):
                    call()
                with torch.no_grad():
                    assert not call().requires_grad


def test_cpu_tensors_have_no_implementation():
    import branchcraft_torch as bt
    ints = torch.zeros(2, dtype=torch.int32)
    codes = torch.zeros(1, 16, 1, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    scales = torch.zeros(1, 1, 16, 2, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    with pytest.raises(NotImplementedError):
        bt.read_fp8_kv(codes, scales, codes, scales, ints, torch.float16)


def test_extend_on_fake_tensors():
    from branchcraft_torch.transaction import Fp8Cache, PagedTreeCache
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        for cache, options in ((Fp8Cache(8, 2, 64, torch.float16), {}), (PagedTreeCache(8, 2, 64), dict(share=True))):
            rows = torch.zeros(20, 2, 64, device="cuda", dtype=torch.float16)
            q = torch.zeros(6, 4, 64, device="cuda", dtype=torch.float16)
            a = cache.new(rows, rows)
            b = cache.fork(a)
            out = cache.extend([a, b], [3, 3], q, rows[:6], rows[:6], cap=3.0, **options)
            assert out.shape == (6, 4, 64) and out.dtype == q.dtype
            assert cache.lengths == {a: 23, b: 23} and cache.pages[a][1] != cache.pages[b][1]


def test_the_8_bit_cache_refuses():
    from branchcraft_torch.transaction import Fp8Cache
    for bad in (dict(physical_pages=0), dict(kv_heads=0), dict(head_dim=96), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            Fp8Cache(**(dict(physical_pages=4, kv_heads=1, head_dim=64, device="cpu") | bad))
    cache = Fp8Cache(4, 1, 64, device="cpu")
    rows = torch.zeros(20, 1, 64, dtype=torch.bfloat16)
    for bad in ((rows, rows[:3]), (rows.half(), rows.half()), (rows[0], rows[0]), (rows[:, :, :32], rows[:, :, :32]),
                (rows.clone().requires_grad_(), rows)):
        with pytest.raises(ValueError):
            cache.new(*bad)
    free = list(cache.free)
    with pytest.raises(NotImplementedError):  # a CPU pool has no implementation: the pages are given back
        cache.new(rows, rows)
    assert cache.free == free and cache.lengths == {} and cache.pages == {}
    cache.owner.check_invariants()
    for call in (lambda: cache.verify(0, rows), lambda: cache.commit(0, [0], rows, rows),
                 lambda: cache.commit_many([0], [[0]], rows, rows)):
        with pytest.raises(NotImplementedError):
            call()
    with pytest.raises(ValueError, match="share"):
        cache.extend([0], [1], rows, rows, rows, share=True)


@pytest.mark.parametrize("seed", range(20))
def test_groups_of_requests_that_share_pages(seed):
    """Whatever was forked, extended and rolled back: the tokens of a group lie in the
    same pages for all of its members, whole ones, and inside their lengths."""
    from branchcraft_torch.pages import PageOwner
    r = random.Random(seed)
    owner = PageOwner(4000)
    requests = [owner.new(r.randint(0, 300))]
    for _ in range(30):
        kind = r.random()
        if kind < 0.2:
            requests.append(owner.new(r.randint(0, 200)))
        elif kind < 0.7:
            requests.append(owner.fork(r.choice(requests)))
        else:
            owner.plan_commit(r.choice(requests), r.randint(1, 50))
    if r.random() < 0.5:
        r.shuffle(requests)
    bounds, tokens = owner.shared_prefixes(requests)
    assert bounds[0] == 0 and bounds[-1] == len(requests) and bounds == sorted(set(bounds))
    assert len(tokens) == len(bounds) - 1
    for a, b, n in zip(bounds, bounds[1:], tokens):
        first = owner.pages[requests[a]]
        for x in requests[a:b]:
            assert n <= owner.lengths[x]
            if b - a > 1:
                assert n > 0 and n % 16 == 0 and owner.pages[x][:n // 16] == first[:n // 16]


def test_all_forks_of_a_prompt_are_one_group():
    from branchcraft_torch.pages import PageOwner
    owner = PageOwner(200)
    a = owner.new(100)
    forks = [a] + [owner.fork(a) for _ in range(5)]
    other = owner.new(33)
    for x in forks:
        owner.plan_commit(x, 3)
    assert owner.shared_prefixes(forks + [other]) == ([0, 6, 7], [96, 33])


@pytest.mark.parametrize("source,count", [("fp8.hip", 12), ("shared.hip", 12)])
def test_matrix_results_and_scalar_bases_are_waited_for(source, count, tmp_path):
    """As tests of the chunk kernels hold: wait states between a matrix instruction
    and what touches its registers, and between a scalar base's write and its use."""
    import shutil
    from pathlib import Path

    import asm_hazards as H
    import test_sgpr_waits_cpu as S
    if not (shutil.which("hipcc") or Path("/opt/rocm/bin/hipcc").exists()):
        pytest.skip("hipcc not available")
    kernels = H.kernels(H.compile_device_asm(H.CSRC / source, tmp_path))
    S.check(kernels)
    found = 0
    for name, lines in kernels.items():
        insts, labels = H.parse(lines)
        if not any(op.startswith("v_mfma") for op, _ in insts):
            continue
        found += 1
        best = H.scan(insts, labels, window=12)
        assert best.get("RAW", 12) >= 12 and best.get("WAW", 10) >= 10 and best.get("WARC", 10) >= 10, (name, best)
    assert found == count
