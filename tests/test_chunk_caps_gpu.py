"""Capped scores where the cap matters, under a bound that an uncapped kernel
does not meet, in every form of the work."""

import pytest
import torch

import chunk_cap_helpers as K
import chunk_helpers as C

pytestmark = pytest.mark.gpu

F16, BF16 = torch.float16, torch.bfloat16
SHAPES = {
    "tiles and ranges": ([333, 1, 90, 64], [130, 1, 17, 40]),
    "one token": ([700], [1]),
    "split": ([1500, 1300, 40], [45, 2, 33]),
}


@pytest.mark.parametrize("dtype,hq,hkv,d", [(F16, 8, 2, 128), (BF16, 6, 2, 64), (F16, 4, 2, 64), (BF16, 4, 1, 128)])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", K.CASES)
def test_caps(name, shape, dtype, hq, hkv, d):
    import branchcraft_torch as bt
    fix, options = K.case(name, *SHAPES[shape], hq, hkv, d, dtype, seed=len(name))
    want, tol = K.reference(**fix, **options)
    dev = C.on_gpu(fix)
    opts = {n: x.cuda() if isinstance(x, torch.Tensor) else x for n, x in options.items()}
    meta = [dev[n] for n in ("pages", "lengths", "starts")]
    C.check(bt.chunk_attention(dev["q"], dev["k"], dev["v"], *meta, **opts), want, tol, name)
    # One element off alignment: row by row.
    q = torch.empty(dev["q"].numel() + 1, device="cuda", dtype=dtype)[1:].view(dev["q"].shape).copy_(dev["q"])
    C.check(bt.chunk_attention(q, dev["k"], dev["v"], *meta, **opts), want, tol, name + ", row by row")
