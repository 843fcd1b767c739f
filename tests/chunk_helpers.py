"""Fixtures and the definition, in 64 bits on the CPU, of the chunk ops."""

from __future__ import annotations

import math

import torch

PAGE = 16


def pages_of(n):
    return -(-n // PAGE)


def batch(lengths, counts, hq, hkv, d, dtype, *, seed=0, spare=3, extra_cols=1, spread=1.0):
    """A batch on the CPU: shuffled pages, every slot that holds no token NaN."""
    g = torch.Generator().manual_seed(seed)
    used = sum(pages_of(max(n, 0)) for n in lengths)
    pool = used + spare
    width = max([pages_of(max(n, 0)) for n in lengths] + [1]) + extra_cols
    ids = torch.randperm(pool, generator=g)[:used].to(torch.int32)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    k = torch.full((pool, PAGE, hkv, d), float("nan")).to(dtype)
    v = k.clone()
    at = 0
    for b, n in enumerate(lengths):
        c = pages_of(max(n, 0))
        table[b, :c] = ids[at:at + c]
        for x in (k, v):
            rows = torch.randn((max(n, 0), hkv, d), generator=g).to(dtype)
            for i in range(c):
                part = rows[PAGE * i:PAGE * (i + 1)]
                x[ids[at + i], :part.shape[0]] = part
        at += c
    total = sum(counts)
    q = (spread * torch.randn((total, hq, d), generator=g)).to(dtype)
    starts = torch.tensor([0] + list(torch.tensor(counts).cumsum(0)), dtype=torch.int32)
    return dict(q=q, k=k, v=v, pages=table, lengths=torch.tensor(lengths, dtype=torch.int32),
                starts=starts)


def reference(q, k, v, pages, lengths, starts, *, scale=None, causal=True, window=0, cap=0.0,
              slopes=None, prefix=None, first=None):
    """Outputs in 64 bits, and how far a kernel's may be off, element by element.

    With u half a step of the type: the output's rounding, u |o|; the weights'
    rounding before the product with V, u A with A the softmax-weighted mean
    of |v|; an error of e in every score moves the output by at most 2 e A.
    e: D products and sums in FP32 (2^-24 of sum |q k| each), and 16 further
    roundings of the score, its cap and bias and its exponential, each 2^-22
    of their size at most (the hardware's exp2, reciprocal and log2 e times
    the score are off by one step).  FP16 weights below the normal range:
    2^-32 of the largest weight, for every token."""
    t, hq, d = q.shape
    hkv = k.shape[2]
    g = hq // hkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    out = torch.zeros((t, hq, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(len(lengths)):
        lo_row, hi_row = int(starts[b]), min(int(starts[b + 1]), t)
        full = int(lengths[b])
        n_len = max(0, min(full, pages.shape[1] * PAGE))
        ids = pages[b, :pages_of(n_len)].long()
        in_pool = ((ids >= 0) & (ids < k.shape[0])).repeat_interleave(PAGE)[:n_len]
        safe = ids.clamp(0, k.shape[0] - 1)
        kk = k[safe].reshape(-1, hkv, d)[:n_len].double()
        vv = v[safe].reshape(-1, hkv, d)[:n_len].double()
        for row in range(lo_row, hi_row):
            p = full - (hi_row - row) if starts[b + 1] <= t else full - (t - row)
            if p < 0:
                continue
            lo, hi = 0, n_len - 1
            if causal:
                hi = min(hi, p if prefix is None else max(p, int(prefix[b]) - 1))
            if window:
                lo = max(lo, p - window + 1)
            if first is not None:
                lo = max(lo, int(first[row]))
            seen = torch.arange(n_len)
            seen = seen[(seen >= lo) & (seen <= hi) & in_pool]
            if not seen.numel():
                continue
            ks, vs = kk[seen], vv[seen]
            for h in range(hq):
                qh = q[row, h].double()
                s = scale * (ks[:, h // g] @ qh)
                size = scale * (ks[:, h // g].abs() @ qh.abs()).max()
                if cap:
                    s = cap * torch.tanh(s / cap)
                if slopes is not None:
                    bias = float(slopes[h]) * (p - seen).abs().double()
                    s = s - bias
                    size = size + bias.abs().max()
                w = torch.softmax(s, 0)
                out[row, h] = w @ vs[:, h // g]
                mean = w @ vs[:, h // g].abs()
                e = 2.0 ** -24 * (d + 4 * 16) * max(1.0, float(size), cap)
                tol[row, h] = u * out[row, h].abs() + (u + 2 * e) * mean \
                    + seen.numel() * 2.0 ** -32 * vs.abs().max() + 2.0 ** -24
    return out, tol


def on_gpu(fix):
    return {name: x.cuda() if isinstance(x, torch.Tensor) else x for name, x in fix.items()}


def check(got, want, tol, what=""):
    got = got.double().cpu()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (
        f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}, "
        f"worst {float(((got - want).abs() / tol.clamp(min=1e-12)).nan_to_num(1e9).max()):.2f} of the bound")
