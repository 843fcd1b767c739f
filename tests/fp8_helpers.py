"""The 8-bit cache's rounding on the CPU, and fixtures of requests that begin alike."""

from __future__ import annotations

import torch

import chunk_helpers as C

BLOCK = 32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def to_fp8(x):
    """Rows [..., D] of FP16 or BF16 as codes [..., D] and scales [..., D / 32]."""
    y = x.double()
    finite = torch.isfinite(y)
    top = 1.875 * 2.0 ** (15 if x.dtype == torch.float16 else 127)  # rounded up, none of the type
    y = torch.where(finite, y.clamp(-top, top), y)
    y = y.unflatten(-1, (-1, BLOCK))
    finite = finite.unflatten(-1, (-1, BLOCK))
    top = torch.where(finite, y.abs(), 0.0).amax(-1)
    # The least power with top <= 448 * 2^e: that of top's own power of two, or the next.
    e = torch.frexp(top.clamp(min=2.0 ** -140))[1] - 9
    e = torch.where(top <= 448 * torch.exp2(e.double()), e, e + 1).clamp(min=-126)
    codes = torch.where(finite, y * torch.exp2(-e.double())[..., None], float("nan")).float().to(E4M3)
    return codes.flatten(-2), (e + 127).to(torch.uint8).view(E8M0)


def values(codes, scale):
    """Codes [..., D] and scales [..., D / 32] as 64-bit values."""
    power = torch.exp2(scale.view(torch.uint8).double() - 127)
    return codes.double() * power.repeat_interleave(BLOCK, -1)


def pools(fix):
    """A 16-bit fixture's pools in 8 bits: (codes, scales) of K and V, and the fixture
    with their values, in its type, in place of the rows (exact: asserted)."""
    out, same = [], dict(fix)
    for name in ("k", "v"):
        codes, scale = to_fp8(fix[name])
        exact = values(codes, scale)
        same[name] = exact.to(fix[name].dtype)
        assert torch.equal(same[name].double().nan_to_num(1e9), exact.nan_to_num(1e9))
        scale = scale.view(torch.uint8).transpose(1, 2).contiguous().view(E8M0)
        out += [codes, scale]
    return out, same


def forks(groups, hq, hkv, d, dtype, *, seed=0, spread=1.0, lone_ends=0):
    """A batch of groups [(shared tokens, [(own tokens, new tokens), ...]), ...] whose
    members hold the same rows, and the same pages where those are whole, for what
    they share; a partial page is each member's own copy.  `lone_ends`: requests at
    either end that no group holds (the first and last groups' members)."""
    lengths = [s + own for s, members in groups for own, _ in members]
    counts = [n for _, members in groups for _, n in members]
    fix = C.batch(lengths, counts, hq, hkv, d, dtype, seed=seed, spread=spread)
    at = 0
    for s, members in groups:
        lead, whole, rest = fix["pages"][at].clone(), s // C.PAGE, s % C.PAGE
        for i in range(1, len(members)):
            row = fix["pages"][at + i]
            for x in (fix["k"], fix["v"]):
                if rest:
                    x[row[whole], :rest] = x[lead[whole], :rest]
            row[:whole] = lead[:whole]
        at += len(members)
    bounds = torch.tensor([0] + [len(m) for _, m in groups]).cumsum(0).to(torch.int32)
    shared = torch.tensor([s for s, _ in groups], dtype=torch.int32)
    if lone_ends:
        bounds, shared = bounds[1:-1], shared[1:-1]
    return widen(fix), bounds, shared


def pays(fix, window=0):
    """Whether the op reads shared pages once: by what the requests may see, each its
    own, in a table of this width, and by their rows."""
    batch, table = fix["pages"].shape[0], fix["pages"].shape[1] * C.PAGE
    rows = fix["q"].shape[0] * (fix["q"].shape[1] // fix["k"].shape[2])
    seen = min(window or table, table)
    size = batch * seen * fix["k"].shape[2] * fix["k"].shape[3] * 4 / 1e6
    return (batch > 1 and table > 1024 and rows <= 80 * batch and size >= (400 if seen < table else 100)
            and size >= 1.2 * batch)


def widen(fix):
    """The same batch in a table wide enough for that, with or without a window
    (windows have no more tokens than the table then): columns of no page."""
    batch, old = fix["pages"].shape
    each = max(110e6 / batch, 1.3e6)  # bytes of K and V per request
    width = int(each / (C.PAGE * fix["k"].shape[2] * fix["k"].shape[3] * 4)) + 65
    fix["pages"] = torch.cat((fix["pages"], torch.full((batch, max(width - old, 0)), -1, dtype=torch.int32)), 1)
    return fix
