"""Capped scores: cases whose outputs differ from uncapped ones by far more than
a kernel may be off, and that bound, token by token.

With u half a step of the type, w the softmax weights and o the output, an error
of e_j in the score of token j moves the output by at most the sum of
w_j e_j (|v_j| + |o|) (to first order; 5 % are added for the rest, all e being
below 0.02).  e_j is made of
 - the product's rounding, 2^-24 D scale sum |q k|, times the slope of the cap
   at the score, 1 - tanh^2 (raised by what the score's own error makes of it);
 - roundings of the argument: four of 2^-24 of it, times the same slope, so at
   most 2^-22 min(|score|, 0.45 cap);
 - the tanh: up to a cap of 256 as -2 cap / (e^2x + 1), whose exponential, sum
   and reciprocal are off by one, one half and one step of 2^-23, 5 cap 2^-23 at
   most, and whose product with 2 cap log2 e, rounded twice, adds two 2^-24 of
   2 cap: cap 2^-20 in all covers them;
   above it as tanh, off by 12 * 2^-23 of itself at most (from 0.3 on its
   exponential form is off by 3.5 * 2^-23, below it the series by two steps):
   2^-19 of the capped score;
 - a bias: four roundings of 2^-24 of it, and of the sum: 2^-21 of it;
 - the exponential: its argument of up to 32, rounded, and itself: 2^-18.
To that come the weights' rounding to the type, u (mean |v| + |o|), the output's,
u |o|, sums of n terms in 32 bits, n 2^-24 mean |v|, and FP16 weights below the
normal range, 2^-32 of the largest for every token."""

from __future__ import annotations

import math

import torch

import chunk_helpers as C

# cap, options, and the middle of the rows' scores in units of the cap: below 0.3
# (the tanh's series), where it bends, and where it has all but reached 1.
CASES = {
    "3": (3.0, {}, (0.2, 0.8, 3.0)),
    "3 negative": (3.0, {}, (-0.2, -0.8, -3.0)),
    "30 window": (30.0, dict(window=70), (0.2, 0.8, 3.0)),
    "1e-3": (1e-3, {}, (0.2, 4.0, 3e4)),
    "50 full": (50.0, dict(causal=False), (0.2, 0.8, 4.0)),
    "256": (256.0, {}, (0.2, 0.8, 4.0)),
    "256 negative": (256.0, {}, (-0.25, -0.8, -4.0)),
    "300": (300.0, {}, (0.2, 0.8, 4.0)),
    "300 negative": (300.0, {}, (-0.25, -0.8, -4.0)),
    "5 bias": (5.0, dict(slopes=True), (0.2, 0.8, 3.0)),
    "300 bias": (300.0, dict(slopes=True), (0.2, 0.8, 4.0)),
    "1e6 bias": (1e6, dict(slopes=True), (2e-6, 5e-6, 1e-5)),
}


def case(name, lengths, counts, hq, hkv, d, dtype, seed=0):
    """A batch whose keys lie around one direction: a row's scores around
    `middle` caps, spread by an eighth of that, or by less where that would leave
    one token with all the weight."""
    cap, options, middles = CASES[name]
    fix = C.batch(lengths, counts, hq, hkv, d, dtype, seed=seed)
    g = torch.Generator().manual_seed(seed + 1)
    along = torch.randn(d, generator=g)
    along /= along.norm()
    near = 8 if cap < 100 else 32
    fix["k"] = (fix["k"].float() + near * along).to(dtype)
    rows = fix["q"].shape[0]
    middle = torch.tensor(middles)[torch.arange(rows) % len(middles)]
    scale = abs(middles[-1]) * cap / (8 * near)  # q of the last middle has length 8
    fix["q"] = ((8 * middle / abs(middles[-1]))[:, None, None] * along.expand(rows, hq, d)).to(dtype)
    options = dict(options, cap=cap, scale=scale)
    if "slopes" in options:
        options["slopes"] = 0.02 * torch.rand(hq, generator=g)
    return fix, options


def reference(q, k, v, pages, lengths, starts, *, cap, scale, causal=True, window=0, slopes=None):
    t, hq, d = q.shape
    g, u = hq // k.shape[2], torch.finfo(q.dtype).eps / 2
    out = torch.zeros((t, hq, d), dtype=torch.float64)
    tol = torch.zeros_like(out)
    for b in range(len(lengths)):
        n, end = int(lengths[b]), int(starts[b + 1])
        ids = pages[b, :C.pages_of(n)].long()
        kk, vv = (x[ids].flatten(0, 1)[:n].double() for x in (k, v))
        for row in range(int(starts[b]), end):
            p = n - (end - row)
            lo = max(0, p - window + 1) if window else 0
            seen = torch.arange(lo, p + 1 if causal else n)
            for h in range(hq):
                ks, vs, qh = kk[seen, h // g], vv[seen, h // g], q[row, h].double()
                raw = scale * (ks @ qh)
                bent = torch.tanh(raw / cap) if cap else raw
                s = cap * bent if cap else raw
                e = 2.0 ** -24 * d * scale * (ks.abs() @ qh.abs())
                if cap:
                    e = e * (1 - torch.tanh((raw.abs() - e).clamp(min=0) / cap) ** 2) \
                        + 2.0 ** -22 * raw.abs().clamp(max=0.45 * cap)
                    e = e + (cap * 2.0 ** -20 if cap <= 256 else 2.0 ** -19 * s.abs())
                if slopes is not None:
                    bias = float(slopes[h]) * (p - seen).abs().double()
                    s, e = s - bias, e + 2.0 ** -21 * bias
                e = e + 2.0 ** -18
                w = torch.softmax(s, 0)
                o, mean = w @ vs, w @ vs.abs()
                assert not cap or float((w * e).sum()) < 0.02, float((w * e).sum())
                out[row, h] = o
                tol[row, h] = 1.05 * ((w * e) @ vs.abs() + (w @ e) * o.abs()) + u * (mean + 2 * o.abs()) \
                    + len(seen) * (2.0 ** -24 * mean + 2.0 ** -32 * vs.abs().max()) + 2.0 ** -24
    return out, tol
