"""The chunk operators as measurable cases: new tokens of a batch of requests
enter the paged cache and attend to it.

A case is one call through the public Python API (``branchcraft_torch``):
``build_tables`` makes the block table, the row offsets and the slot map of a
step from the requests' lengths, ``append_kv_`` writes the new tokens' K and V
rows by that map, and ``chunk_attention`` lets them attend to their request's
pages.  Each also has its plain form in elementary torch operations.

Sizes are the framework's own: the head layouts of the random-shape tests, the
batches and contexts of the decode and tree sweeps, and chunks between one
token and a whole prompt.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

PAGE = 16
# Query heads, KV heads: GQA groups 1, 2, 4, 7 and 8, and few or many KV heads.
HEADS = ((32, 8), (32, 32), (28, 4), (16, 2), (8, 1), (64, 8), (32, 4), (16, 16), (8, 8), (24, 8))
# No drawn case costs more than the largest listed one of its operator.
MOST_PAIRS = 2048 * 32 * (32768 - 1024)  # visible (row, token) pairs, over the query heads
MOST_TOKENS = 140000  # rows of a slot map
MOST_ROWS = 8192      # rows appended


def listed():
    return [
        # A decode step's tables: one new token for each of 64 chats.
        dict(name="tables 64x1", op="tables", batch=64, lo=128, hi=4096, new="one", mix=1),
        # A batch of whole prompts is admitted: every token is new.
        dict(name="tables 64x128-4096 new", op="tables", batch=64, lo=128, hi=4096, new="all", mix=2),
        # A decode step's K and V rows enter the pool.
        dict(name="append 64", op="append", rows=64, hq=32, hkv=8, d=128, dtype="bf16", fused=False, mix=3),
        # A large prefill step's rows, as slices of the fused projection.
        dict(name="append 8192 fused", op="append", rows=8192, hq=32, hkv=8, d=128, dtype="fp16", fused=True,
             mix=4),
        # One chat, one token, short context: launches and latency.
        dict(name="chunk 1x1 of 512", op="chunk", batch=1, lo=512, hi=512, new="one", hq=32, hkv=8, d=128,
             dtype="fp16", form="causal", mix=5),
        # The single-token form over an ordinary serving batch.
        dict(name="chunk 64x1 of 128-4096", op="chunk", batch=64, lo=128, hi=4096, new="one", hq=32, hkv=8,
             d=128, dtype="bf16", form="causal", mix=6),
        # A whole prompt at once.
        dict(name="chunk 4096 of 4096", op="chunk", batch=1, lo=4096, hi=4096, new="all", hq=32, hkv=8, d=128,
             dtype="fp16", form="causal", mix=7),
        # One chunk of a long document's prefill.
        dict(name="chunk 2048 of 32768", op="chunk", batch=1, lo=32768, hi=32768, new="2048", hq=32, hkv=8,
             d=128, dtype="bf16", form="causal", mix=8),
        # A mixed step: most requests decode, every fourth prefills a chunk.
        dict(name="chunk 32 mixed", op="chunk", batch=32, lo=300, hi=4096, new="mixed", hq=32, hkv=8, d=128,
             dtype="bf16", form="causal", mix=9),
        # Capped scores in a sliding window, as alternating layers have them.
        dict(name="chunk 4x1024 cap window", op="chunk", batch=4, lo=2048, hi=8192, new="1024", hq=24, hkv=8,
             d=128, dtype="bf16", form="cap window", mix=10),
        # A bias that falls with distance, every head its own K and V, ragged.
        dict(name="chunk 16 ragged bias d64", op="chunk", batch=16, lo=300, hi=3000, new="ragged", hq=32,
             hkv=32, d=64, dtype="fp16", form="bias", mix=11),
        # Packed documents in one sequence: a row sees its own document only.
        dict(name="chunk 6001 documents d64", op="chunk", batch=1, lo=6001, hi=6001, new="all", hq=28, hkv=4,
             d=64, dtype="bf16", form="documents", mix=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    while True:
        op = rng.choice(("tables", "append", "chunk", "chunk", "chunk", "chunk"))
        c = dict(op=op, mix=rng.randrange(1 << 20))
        if op == "append":
            hq, hkv = rng.choice(HEADS)
            c.update(rows=_log_int(rng, 1, MOST_ROWS), hq=hq, hkv=hkv, d=rng.choice((64, 128)),
                     dtype=rng.choice(("fp16", "bf16")), fused=rng.random() < 0.5)
            if c["rows"] * hkv * c["d"] <= MOST_ROWS * 8 * 128:
                return c
            continue
        c["batch"] = _log_int(rng, 1, 256 if op == "tables" else 128)
        c["hi"] = _log_int(rng, 17, 8192 if op == "tables" else 32768)
        c["lo"] = c["hi"] if rng.random() < 0.3 else max(1, c["hi"] // rng.choice((2, 8, 32)))
        c["new"] = rng.choice(("one", "all", "ragged", "mixed", str(_log_int(rng, 2, 2048))))
        if op == "tables":
            if sum(_counts(c)) <= MOST_TOKENS:
                return c
            continue
        hq, hkv = rng.choice(HEADS)
        c.update(hq=hq, hkv=hkv, d=rng.choice((64, 128)), dtype=rng.choice(("fp16", "bf16")),
                 form=rng.choice(("causal", "causal", "full", "cap window", "window", "bias", "cap bias",
                                  "prefix", "documents")))
        if hkv * c["d"] * sum(_lengths(c)) <= 1 << 28 and hq * sum(
                n * x for n, x in zip(_counts(c), _lengths(c))) <= MOST_PAIRS:
            return c


# ---------------------------------------------------------------------------
# shapes


def _lengths(c):
    """Tokens of each request, its new ones included."""
    if c["lo"] == c["hi"]:
        return [c["hi"]] * c["batch"]
    r = random.Random(c["mix"])
    return [r.randint(c["lo"], c["hi"]) for _ in range(c["batch"])]


def _counts(c):
    """New tokens of each request."""
    r, kind, out = random.Random(c["mix"] + 1), c["new"], []
    for i, n in enumerate(_lengths(c)):
        if kind == "one":
            out.append(1)
        elif kind == "all":
            out.append(n)
        elif kind == "ragged":
            out.append(r.randint(1, max(1, min(n, 700))))
        elif kind == "mixed":
            out.append(min(n, 512 - i) if i % 4 == 0 else 1)
        else:
            out.append(min(n, int(kind)))
    return out


def _pages(n):
    return -(-n // PAGE)


def _window(c):
    return 1024 if "window" in c["form"] else 0


def _cap(c):
    return 50.0 if "cap" in c["form"] else 0.0


def _prefix(c):
    """With a prefix mask: the tokens of each request that all its rows see."""
    return [max(1, n // 3) for n in _lengths(c)]


def _first(c):
    """With documents: the first token of each row's own one."""
    r, out = random.Random(c["mix"] + 2), []
    for n, new in zip(_lengths(c), _counts(c)):
        begin, at = [], 0
        while at < n:
            size = r.randint(1, max(2, n // 5))
            begin += [at] * min(size, n - at)
            at += size
        out += begin[n - new:]
    return out


def _ranges(c):
    """For each request the first and the last token that each new one sees."""
    out, at, first = [], 0, _first(c) if c["form"] == "documents" else None
    for b, (n, new) in enumerate(zip(_lengths(c), _counts(c))):
        pos = np.arange(n - new, n)
        lo, hi = np.zeros_like(pos), pos
        if c["form"] == "full":
            hi = np.full_like(pos, n - 1)
        elif c["form"] == "prefix":
            hi = np.maximum(pos, _prefix(c)[b] - 1)
        if _window(c):
            lo = np.maximum(lo, pos - _window(c) + 1)
        if first is not None:
            lo = np.asarray(first[at:at + new])
        at += new
        out.append((lo, hi))
    return out


def work(case):
    c = case
    if c["op"] == "append":
        return {"bytes": c["rows"] * (2 * 2 * c["hkv"] * c["d"] * 2 + 4), "flops": 0.0}
    lengths, total = _lengths(c), sum(_counts(c))
    used, width = sum(map(_pages, lengths)), _pages(c["hi"])
    if c["op"] == "tables":
        return {"bytes": 4 * (used + 2 * c["batch"] + c["batch"] * width + c["batch"] + 1 + 2 * total),
                "flops": 0.0}
    pairs = tokens = 0
    for lo, hi in _ranges(c):
        pairs += int((hi - lo + 1).sum())
        tokens += int(hi.max() - lo.min() + 1)
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    return {"bytes": 2 * tokens * hkv * d * 2 + 2 * total * hq * d * 2 + 4 * used + 8 * c["batch"],
            "flops": 4.0 * d * hq * pairs}


# ---------------------------------------------------------------------------
# inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _type(c):
    return torch.float16 if c["dtype"] == "fp16" else torch.bfloat16


def prepare(case, seed):
    c, g = case, _gen(seed)
    rng = np.random.default_rng(seed)
    if c["op"] == "append":
        n, hkv, d, t = c["rows"], c["hkv"], c["d"], _type(c)
        pool = _pages(n) * 2 + 64
        s = {"op": "append", "k_pool": torch.zeros((pool, PAGE, hkv, d), device="cuda", dtype=t),
             "v_pool": torch.zeros((pool, PAGE, hkv, d), device="cuda", dtype=t)}
        if c["fused"]:
            rows = torch.randn((n, c["hq"] + 2 * hkv, d), generator=g, device="cuda", dtype=t)
            s["k"], s["v"] = rows[:, c["hq"]:c["hq"] + hkv], rows[:, c["hq"] + hkv:]
        else:
            s["k"], s["v"] = (torch.randn((n, hkv, d), generator=g, device="cuda", dtype=t) for _ in range(2))
        if n > 256:  # a prompt's rows: whole pages, in order
            pages = rng.permutation(pool)[:_pages(n)]
            slots = (pages[:, None] * PAGE + np.arange(PAGE)).reshape(-1)[:n]
        else:        # single rows of many requests
            slots = rng.permutation(pool * PAGE)[:n]
        s["slots"] = torch.from_numpy(slots.astype(np.int32)).cuda()
        return s
    lengths, counts = _lengths(c), _counts(c)
    used, width = sum(map(_pages, lengths)), _pages(c["hi"])
    pool = used + used // 8 + 7
    ids = rng.permutation(pool)[:used].astype(np.int32)
    s = {"op": c["op"], "lengths": _int(lengths), "total": sum(counts), "width": width}
    if c["op"] == "tables":
        return s | {"ids": torch.from_numpy(ids).cuda(), "counts": _int(counts)}
    table = np.full((c["batch"], width), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(lengths):
        table[b, :_pages(n)] = ids[at:at + _pages(n)]
        at += _pages(n)
    hq, hkv, d, t = c["hq"], c["hkv"], c["d"], _type(c)
    s["pages"] = torch.from_numpy(table).cuda()
    s["starts"] = _int(np.concatenate(([0], np.cumsum(counts))).tolist())
    s["q"] = (2 * torch.randn((sum(counts), hq, d), generator=g, device="cuda")).to(t)
    s["k"], s["v"] = (torch.randn((pool, PAGE, hkv, d), generator=g, device="cuda", dtype=t) for _ in range(2))
    s["options"] = {"window": _window(c), "cap": _cap(c), "causal": c["form"] != "full"}
    if "bias" in c["form"]:
        s["options"]["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda") / hq)
    if c["form"] == "prefix":
        s["options"]["prefix"] = _int(_prefix(c))
    if c["form"] == "documents":
        s["options"]["first"] = _int(_first(c))
    # The requests by their number of new tokens, as the host knows them.
    groups = {}
    for b, n in enumerate(counts):
        groups.setdefault(n, []).append(b)
    s["groups"] = [(n, torch.tensor(who).cuda(), _pages(max(lengths[b] for b in who)))
                   for n, who in sorted(groups.items())]
    return s


# ---------------------------------------------------------------------------
# the plain forms


def _plain_tables(s):
    lengths, counts, ids = s["lengths"].long(), s["counts"].long(), s["ids"]
    held = (lengths + PAGE - 1) // PAGE
    column = torch.arange(s["width"], device=ids.device)
    at = (held.cumsum(0) - held)[:, None] + column
    pages = torch.where(column < held[:, None], ids[at.clamp(max=ids.numel() - 1)], -1)
    ends = counts.cumsum(0)
    token = torch.arange(s["total"], device=ids.device)
    who = torch.searchsorted(ends, token, right=True)
    positions = lengths[who] - ends[who] + token
    slots = pages[who, positions // PAGE] * PAGE + positions % PAGE
    return (pages, torch.cat((ends.new_zeros(1), ends)).int(), slots.int(), positions.int())


def _plain_append(s):
    for pool, rows in ((s["k_pool"], s["k"]), (s["v_pool"], s["v"])):
        pool.view(-1, *pool.shape[2:]).index_copy_(0, s["slots"].long(), rows)
    return s["k_pool"], s["v_pool"]


def _plain_attend(q, k, v, lengths, rows, options):
    """q [R, n, Hq, D] of R requests with n new tokens each, k and v [R, L, Hkv,
    D] their pages' tokens, rows [R, n] the rows' numbers."""
    r, n, hq, d = q.shape
    length, hkv = k.shape[1], k.shape[2]
    q = q.float().view(r, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(r * hkv, -1, d)
    k = k.float().permute(0, 2, 3, 1).reshape(r * hkv, d, length)
    v = v.float().permute(0, 2, 1, 3).reshape(r * hkv, length, d)
    scores = torch.bmm(q, k).mul_(1.0 / math.sqrt(d)).view(r, hq, n, length)
    pos = (lengths[:, None] - n + torch.arange(n, device=q.device))[:, :, None]
    token = torch.arange(length, device=q.device)
    seen = token < lengths[:, None, None]
    if options["causal"]:
        last = pos if "prefix" not in options else torch.maximum(pos, options["prefix"][:, None, None] - 1)
        seen = seen & (token <= last)
    if options["window"]:
        seen = seen & (token > pos - options["window"])
    if "first" in options:
        seen = seen & (token >= options["first"][rows][:, :, None])
    if options["cap"]:
        scores = scores.div_(options["cap"]).tanh_().mul_(options["cap"])
    if "slopes" in options:
        scores = scores - options["slopes"][:, None, None] * (pos - token).abs()[:, None].float()
    scores = scores.masked_fill_(~seen[:, None], -math.inf)
    weights = scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = weights.sum(-1, keepdim=True).view(r * hkv, -1, 1)
    out = torch.bmm(weights.view(r * hkv, -1, length), v) / total.clamp(min=1e-30)
    return out.view(r, hkv, hq // hkv, n, d).permute(0, 3, 1, 2, 4).reshape(r, n, hq, d)


def _plain_chunk(s):
    q, out = s["q"], torch.zeros_like(s["q"])
    for n, who, width in s["groups"]:  # one pass for the requests of equal counts
        ids = s["pages"][who, :width].long().clamp(min=0)
        rows = s["starts"].long()[who][:, None] + torch.arange(n, device=q.device)
        options = dict(s["options"])
        if "prefix" in options:
            options["prefix"] = options["prefix"][who]
        k, v = (x[ids].flatten(1, 2) for x in (s["k"], s["v"]))
        out[rows] = _plain_attend(q[rows], k, v, s["lengths"].long()[who], rows, options).to(q.dtype)
    return out


# ---------------------------------------------------------------------------
# the calls


_bt = None


def _api():
    global _bt
    if _bt is None:
        sys.path.insert(0, str(Path.cwd() / "branchcraft-cuda_amd" / "python"))
        import branchcraft_torch
        _bt = branchcraft_torch
    return _bt


def run(s):
    if not own:
        return {"tables": _plain_tables, "append": _plain_append, "chunk": _plain_chunk}[s["op"]](s)
    bt = _api()
    if s["op"] == "tables":
        return bt.build_tables(s["ids"], s["lengths"], s["counts"], s["width"], s["total"])
    if s["op"] == "append":
        bt.append_kv_(s["k_pool"], s["v_pool"], s["k"], s["v"], s["slots"])
        return s["k_pool"], s["v_pool"]
    return bt.chunk_attention(s["q"], s["k"], s["v"], s["pages"], s["lengths"], s["starts"], **s["options"])


# ---------------------------------------------------------------------------
# the definition, in 64 bits


def exact(case, seed):
    c = case
    if c["op"] != "chunk":
        return None
    s, d, group, at = prepare(c, seed), c["d"], c["hq"] // c["hkv"], 0
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    slopes = [2.0 ** (-8.0 * (h + 1) / c["hq"]) for h in range(c["hq"])]
    for b, (length, new, (lo, hi)) in enumerate(zip(_lengths(c), _counts(c), _ranges(c))):
        ids = s["pages"][b, :_pages(length)].long()
        j = torch.arange(length, device="cuda")
        lo, hi = torch.from_numpy(lo).cuda()[:, None], torch.from_numpy(hi).cuda()[:, None]
        hidden = (j < lo) | (j > hi)
        distance = (torch.arange(length - new, length, device="cuda")[:, None] - j).abs().double()
        for h in range(c["hq"]):
            k, v = (x[ids, :, h // group].reshape(-1, d)[:length].double() for x in (s["k"], s["v"]))
            y = s["q"][at:at + new, h].double() @ k.t().contiguous() / math.sqrt(d)
            if _cap(c):
                y = _cap(c) * torch.tanh(y / _cap(c))
            if "bias" in c["form"]:
                y = y - slopes[h] * distance
            out[at:at + new, h] = torch.softmax(y.masked_fill(hidden, -math.inf), dim=-1) @ v
        at += new
    return out
