"""The capped cases tell a capped score from an uncapped one, a bias from none
and an output from zeros: none of these lies within the bound."""

import pytest
import torch

import chunk_cap_helpers as K


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("name", K.CASES)
def test_the_bound_is_finer_than_what_the_cap_does(name, dtype):
    fix, options = K.case(name, [40, 90], [2, 9], 2, 1, 64, dtype)
    want, tol = K.reference(**fix, **options)

    def rows_outside(other):
        return ((other - want).abs() > tol).any(-1).all(-1)

    assert rows_outside(torch.zeros_like(want)).all()
    cap, slopes = options["cap"], options.get("slopes")
    plain, _ = K.reference(**fix, **dict(options, cap=0.0))
    if cap < 1e5:  # rows that reach the cap, and all of them where scores are not tiny
        assert rows_outside(plain)[2::3].all()
        assert rows_outside(plain).all() or cap < 30
    if slopes is not None:
        assert rows_outside(K.reference(**fix, **dict(options, slopes=None))[0]).any()
