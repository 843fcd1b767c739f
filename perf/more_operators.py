"""Long caches at half the bytes, or read once for many, as measurable cases.

A case is one call (or the pair that belongs together) through the public Python
API (``branchcraft_torch``): ``append_fp8_kv_`` rounds new tokens' K and V rows to
8 bits as they enter the paged cache and ``read_fp8_kv`` hands rows of it back in
16, ``fp8_chunk_attention`` attends over such a cache, and
``shared_chunk_attention`` over 16-bit pages whose requests, forks of one another,
begin with the same ones.  Each also has its plain form in elementary torch
operations.

A row of 8 bits: every 32 values of one head have one power of two, the least
with which they stay within 448, and each value is rounded to e4m3 of that.

Sizes are the framework's own: the head layouts of the random-shape tests, the
batches and contexts of the decode and tree sweeps, chunks between one token and
two thousand.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

PAGE, BLOCK = 16, 32
# Query heads, KV heads: GQA groups 1, 2, 4, 7 and 8, and few or many KV heads.
HEADS = ((32, 8), (32, 32), (28, 4), (16, 2), (8, 1), (64, 8), (32, 4), (16, 16), (8, 8), (24, 8))
# No drawn case costs more than the largest listed one of its operator.
MOST_ROWS = 8192                              # rows written, of 8 heads of 128
MOST_READ = 32768                             # rows read back
MOST_PAIRS = 2048 * 32 * (32768 - 1024)       # visible (row, token) pairs of a chunk, over the query heads
MOST_SHARED = 64 * 32 * 34000                 # the same of requests that share a prefix


def listed():
    return [
        # A decode step of 64 chats: its rows enter the cache, and come back for a check of the step.
        dict(name="store 64", op="store", rows=64, hq=32, hkv=8, d=128, dtype="bf16", fused=False, mix=1),
        # A large prefill step's rows, as slices of the fused projection.
        dict(name="store 8192 fused", op="store", rows=8192, hq=32, hkv=8, d=128, dtype="fp16", fused=True,
             mix=2),
        # A short chat's rows go back to 16-bit pages.
        dict(name="read 500", op="read", rows=500, hkv=8, d=64, dtype="fp16", mix=3),
        # A long document's rows do.
        dict(name="read 32768", op="read", rows=32768, hkv=8, d=128, dtype="bf16", mix=4),
        # One chat, one token, short context: launches and latency.
        dict(name="fp8 1x1 of 512", op="fp8", batch=1, lo=512, hi=512, new="one", hq=32, hkv=8, d=128,
             dtype="fp16", form="causal", mix=5),
        # The single-token form over an ordinary serving batch.
        dict(name="fp8 64x1 of 128-4096", op="fp8", batch=64, lo=128, hi=4096, new="one", hq=32, hkv=8, d=128,
             dtype="bf16", form="causal", mix=6),
        # One chunk of a long document's prefill.
        dict(name="fp8 2048 of 32768", op="fp8", batch=1, lo=32768, hi=32768, new="2048", hq=32, hkv=8,
             d=128, dtype="bf16", form="causal", mix=7),
        # A mixed step in a sliding window with capped scores, every head its own K and V.
        dict(name="fp8 24 mixed cap window d64", op="fp8", batch=24, lo=300, hi=4096, new="mixed", hq=32,
             hkv=32, d=64, dtype="fp16", form="cap window", mix=8),
        # Eight samples of one prompt, a few tokens in.
        dict(name="shared 8x1 of 2048", op="shared", groups=1, members=8, plen=2048, lo=1, hi=64, new="one",
             hq=32, hkv=8, d=128, dtype="fp16", form="causal", mix=9),
        # A serving batch behind one long document.
        dict(name="shared 64x1 of 32768", op="shared", groups=1, members=64, plen=32768, lo=16, hi=1024,
             new="one", hq=32, hkv=8, d=128, dtype="bf16", form="causal", mix=10),
        # Short turns behind a few system prompts, members of each as they come.
        dict(name="shared 5 prompts turns d64", op="shared", groups=5, members=24, plen=4096, lo=20, hi=700,
             new="few", hq=28, hkv=4, d=64, dtype="fp16", form="causal", mix=11),
        # Drafted tokens of a batch in a window that reaches into the prompt, with a distance bias.
        dict(name="shared 32x8 window bias", op="shared", groups=2, members=16, plen=6000, lo=8, hi=2000,
             new="8", hq=24, hkv=8, d=128, dtype="bf16", form="window bias", mix=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    while True:
        op = rng.choice(("store", "read", "fp8", "fp8", "shared", "shared"))
        hq, hkv = rng.choice(HEADS)
        c = dict(op=op, mix=rng.randrange(1 << 20), hkv=hkv, d=rng.choice((64, 128)),
                 dtype=rng.choice(("fp16", "bf16")))
        if op in ("store", "read"):
            c["rows"] = _log_int(rng, 1, MOST_ROWS if op == "store" else MOST_READ)
            if op == "store":
                c.update(hq=hq, fused=rng.random() < 0.5)
            if c["rows"] * hkv * c["d"] <= (MOST_ROWS if op == "store" else MOST_READ) * 8 * 128:
                return c
            continue
        c["hq"] = hq
        if op == "fp8":
            c.update(batch=_log_int(rng, 1, 128), hi=_log_int(rng, 17, 32768),
                     new=rng.choice(("one", "one", "all", "ragged", "mixed", str(_log_int(rng, 2, 2048)))),
                     form=rng.choice(("causal", "causal", "full", "cap window", "window", "bias", "cap bias",
                                      "prefix", "documents")))
        else:
            c.update(groups=_log_int(rng, 1, 12), members=_log_int(rng, 1, 128),
                     plen=_log_int(rng, 32, 32768), hi=_log_int(rng, 17, 2048),
                     new=rng.choice(("one", "one", "few", str(_log_int(rng, 2, 32)))),
                     form=rng.choice(("causal", "causal", "full", "cap", "window", "bias", "window bias")))
        c["lo"] = c["hi"] if rng.random() < 0.3 else max(1, c["hi"] // rng.choice((2, 8, 32)))
        pairs = hq * sum(n * (p + x) for n, p, x in zip(_counts(c), _prompts(c), _lengths(c)))
        held = sum(_lengths(c)) + sum({g: p for g, p in zip(_group_of(c), _prompts(c))}.values())
        if hkv * c["d"] * held <= 1 << 28 and pairs <= (MOST_PAIRS if op == "fp8" else MOST_SHARED):
            return c


# ---------------------------------------------------------------------------
# shapes


def _group_of(c):
    """The group of each request that shares a prompt; every group has as many members, or fewer."""
    if c["op"] != "shared":
        return [0] * c["batch"]
    r = random.Random(c["mix"] + 3)
    few = c["groups"] > 2
    return [g for g in range(c["groups"])
            for _ in range(r.randint(max(1, c["members"] // 4), c["members"]) if few else c["members"])]


def _prompts(c):
    """For each request the tokens that it shares with its group: whole pages."""
    if c["op"] != "shared":
        return [0] * c["batch"]
    r = random.Random(c["mix"] + 4)
    few = c["groups"] > 2
    each = [r.randint(c["plen"] // 2, c["plen"]) if few else c["plen"] for _ in range(c["groups"])]
    return [each[g] // PAGE * PAGE for g in _group_of(c)]


def _lengths(c):
    """Tokens of each request behind what it shares, its new ones included."""
    r = random.Random(c["mix"])
    return [r.randint(c["lo"], c["hi"]) for _ in _group_of(c)]


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
        elif kind == "few":
            out.append(r.randint(1, max(1, min(n, 16))))
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
    for b, (own_n, p, new) in enumerate(zip(_lengths(c), _prompts(c), _counts(c))):
        n = p + own_n
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


def _row_bytes(c):
    """One token's K or V in 8 bits, its powers of two included."""
    return c["hkv"] * (c["d"] + c["d"] // BLOCK)


def work(case):
    c = case
    if c["op"] == "store":  # rows read, written in 8 bits, and written in 16
        return {"bytes": c["rows"] * (2 * (4 * c["hkv"] * c["d"] + _row_bytes(c)) + 4), "flops": 0.0}
    if c["op"] == "read":
        return {"bytes": c["rows"] * (2 * (2 * c["hkv"] * c["d"] + _row_bytes(c)) + 4), "flops": 0.0}
    pairs = tokens = 0
    least = {}  # of what a group shares: the first token that any member sees
    for g, p, (lo, hi) in zip(_group_of(c), _prompts(c), _ranges(c)):
        pairs += int((hi - lo + 1).sum())
        tokens += int(hi.max() - max(lo.min(), p) + 1)
        if p:
            least[g] = (min(least.get(g, (p, p))[0], int(lo.min())), p)
    tokens += sum(p - at for at, p in least.values())
    hq, hkv, d, total = c["hq"], c["hkv"], c["d"], sum(_counts(c))
    row = _row_bytes(c) if c["op"] == "fp8" else 2 * hkv * d
    return {"bytes": 2 * tokens * row + 2 * total * hq * d * 2 + 4 * _pages(tokens) + 8 * len(_lengths(c)),
            "flops": 4.0 * d * hq * pairs}


# ---------------------------------------------------------------------------
# inputs


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _int(values):
    return torch.tensor(values, dtype=torch.int32).cuda()


def _type(c):
    return torch.float16 if c["dtype"] == "fp16" else torch.bfloat16


def _rows(g, shape, t):
    """K or V rows: some channels of every head are several times the others."""
    d = shape[-1]
    size = torch.where(torch.arange(d, device="cuda") % 29 == 3, 6.0, 1.0)
    return (torch.randn(shape, generator=g, device="cuda") * size).to(t)


def _to_8bit(x):
    """The codes of rows [..., D] and the powers of two [..., D / 32] of their blocks."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(x.abs().amax(-1))  # the largest is m * 2^e, m in [1/2, 1)
    e = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126)
    codes = (x * _power(-e)[..., None]).to(torch.float8_e4m3fn)
    return codes.flatten(-2), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _power(e):
    return ((e + 127) << 23).view(torch.float32)


def _pool(pages, c, g):
    """An 8-bit pool as a program that has run for a while holds it."""
    codes, scale = _to_8bit(_rows(g, (pages, PAGE, c["hkv"], c["d"]), _type(c)))
    return codes, scale.view(torch.uint8).transpose(1, 2).contiguous().view(torch.float8_e8m0fnu)


def prepare(case, seed):
    c, g = case, _gen(seed)
    rng = np.random.default_rng(seed)
    if c["op"] in ("store", "read"):
        n, hkv, d, t = c["rows"], c["hkv"], c["d"], _type(c)
        pool = _pages(n) * 2 + 64
        if n > 256:  # a prompt's rows: whole pages, in order
            pages = rng.permutation(pool)[:_pages(n)]
            slots = (pages[:, None] * PAGE + np.arange(PAGE)).reshape(-1)[:n]
        else:        # single rows of many requests
            slots = rng.permutation(pool * PAGE)[:n]
        s = {"op": c["op"], "slots": torch.from_numpy(slots.astype(np.int32)).cuda(), "type": t}
        for x in "kv":
            s[x + "_pool"], s[x + "_scale"] = _pool(pool, c, g)
        if c["op"] == "store":
            if c["fused"]:
                rows = _rows(g, (n, c["hq"] + 2 * hkv, d), t)
                s["k"], s["v"] = rows[:, c["hq"]:c["hq"] + hkv], rows[:, c["hq"] + hkv:]
            else:
                s["k"], s["v"] = (_rows(g, (n, hkv, d), t) for _ in range(2))
        return s
    counts, prompts, group_of = _counts(c), _prompts(c), _group_of(c)
    lengths = [p + n for p, n in zip(prompts, _lengths(c))]
    batch, width = len(lengths), _pages(max(lengths))
    used = sum(_pages(n) - p // PAGE for n, p in zip(lengths, prompts)) + sum(
        p // PAGE for p in {g: p for g, p in zip(group_of, prompts)}.values())
    pool = used + used // 8 + 7
    ids = rng.permutation(pool)[:used].astype(np.int32)
    table = np.full((batch, width), -1, dtype=np.int32)
    at, of_group = 0, {}
    for b, n in enumerate(lengths):
        held = prompts[b] // PAGE
        if held:  # the group's pages, then its own
            if group_of[b] not in of_group:
                of_group[group_of[b]] = ids[at:at + held]
                at += held
            table[b, :held] = of_group[group_of[b]]
        table[b, held:_pages(n)] = ids[at:at + _pages(n) - held]
        at += _pages(n) - held
    hq, hkv, d, t = c["hq"], c["hkv"], c["d"], _type(c)
    s = {"op": c["op"], "lengths": _int(lengths), "pages": torch.from_numpy(table).cuda(),
         "starts": _int(np.concatenate(([0], np.cumsum(counts))).tolist()),
         "q": (2 * torch.randn((sum(counts), hq, d), generator=g, device="cuda")).to(t)}
    if c["op"] == "fp8":
        for x in "kv":
            s[x], s[x + "_scale"] = _pool(pool, c, g)
    else:
        s["k"], s["v"] = (torch.randn((pool, PAGE, hkv, d), generator=g, device="cuda", dtype=t)
                          for _ in range(2))
        bounds = [0] + [b for b in range(1, batch) if group_of[b] != group_of[b - 1]]
        s["groups"], s["shared"] = _int(bounds + [batch]), _int([prompts[b] for b in bounds])
        s["members"] = list(zip(bounds, bounds[1:] + [batch], [prompts[b] for b in bounds]))
    s["options"] = {"window": _window(c), "cap": _cap(c), "causal": c["form"] != "full"}
    if "bias" in c["form"]:
        s["options"]["slopes"] = torch.exp2(-8.0 * torch.arange(1, hq + 1, device="cuda") / hq)
    if c["form"] == "prefix":
        s["options"]["prefix"] = _int(_prefix(c))
    if c["form"] == "documents":
        s["options"]["first"] = _int(_first(c))
    # What the host knows of the requests: those of equal counts, and each group's longest.
    equal = {}
    for b, n in enumerate(counts):
        equal.setdefault(n, []).append(b)
    s["equal"] = [(n, torch.tensor(who).cuda(), _pages(max(lengths[b] for b in who)))
                  for n, who in sorted(equal.items())]
    s["most"] = [(max(counts[i:j]), _pages(max(lengths[i:j]))) for i, j, _ in s.get("members", ())]
    return s


# ---------------------------------------------------------------------------
# the plain forms


def _bytes_of(x):
    return x.view(torch.uint8)


def _plain_store(s):
    slots = s["slots"].long()
    page, at = slots // PAGE, slots % PAGE
    for x in "kv":
        codes, scale = _to_8bit(s[x])
        pool = _bytes_of(s[x + "_pool"])
        pool.view(-1, *pool.shape[2:]).index_copy_(0, slots, _bytes_of(codes))
        _bytes_of(s[x + "_scale"])[page, :, at] = _bytes_of(scale)
    return _plain_read(s)


def _values(codes, scale):
    """Codes [..., D] with the bytes of their blocks' powers [..., D / 32]."""
    x = codes.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, BLOCK))
    return (x * _power(scale.int() - 127)[..., None]).flatten(-2)


def _plain_read(s):
    slots = s["slots"].long()
    page, at = slots // PAGE, slots % PAGE
    return tuple(_values(_bytes_of(s[x + "_pool"])[page, at], _bytes_of(s[x + "_scale"])[page, :, at]).to(s["type"])
                 for x in "kv")


def _weights(scores, pos, token, length, rows, options):
    """exp of the masked scores [R, Hq, n, tokens], less each row's maximum; rows at pos [R, n], tokens [tokens]."""
    pos = pos[:, :, None]
    seen = token < length[:, None, None]
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
    return scores.sub_(scores.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()


def _heads_first(q, hkv):
    r, n, hq, d = q.shape
    return q.float().view(r, n, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4)  # [R, Hkv, group, n, D]


def _plain_fp8(s):
    q, out, hkv, d = s["q"], torch.zeros_like(s["q"]), s["k"].shape[2], s["q"].shape[2]
    hq = q.shape[1]
    for n, who, width in s["equal"]:  # one pass for the requests of equal counts
        ids = s["pages"][who, :width].long().clamp(min=0)
        rows = s["starts"].long()[who][:, None] + torch.arange(n, device=q.device)
        options = dict(s["options"])
        if "prefix" in options:
            options["prefix"] = options["prefix"][who]
        k, v = (_values(_bytes_of(s[x])[ids], _bytes_of(s[x + "_scale"])[ids].transpose(2, 3)).flatten(1, 2)
                for x in "kv")  # [R, tokens, Hkv, D]
        r, length = k.shape[:2]
        k = k.permute(0, 2, 3, 1).reshape(r * hkv, d, length)
        scores = torch.bmm(_heads_first(q[rows], hkv).reshape(r * hkv, -1, d), k).mul_(1.0 / math.sqrt(d))
        lengths = s["lengths"].long()[who]
        pos = lengths[:, None] - n + torch.arange(n, device=q.device)
        weights = _weights(scores.view(r, hq, n, length), pos, torch.arange(length, device=q.device), lengths,
                           rows, options)
        y = torch.bmm(weights.view(r * hkv, -1, length), v.permute(0, 2, 1, 3).reshape(r * hkv, length, d))
        y = y / weights.sum(-1).view(r * hkv, -1, 1).clamp(min=1e-30)
        out[rows] = y.view(r, hkv, hq // hkv, n, d).permute(0, 3, 1, 2, 4).reshape(r, n, hq, d).to(q.dtype)
    return out


def _plain_shared(s):
    q, out, hkv, d = s["q"], torch.zeros_like(s["q"]), s["k"].shape[2], s["q"].shape[2]
    hq = q.shape[1]
    for (i, j, p), (n, width) in zip(s["members"], s["most"]):  # one pass for a group
        starts, r = s["starts"].long()[i:j + 1], j - i
        lengths, counts = s["lengths"].long()[i:j], starts[1:] - starts[:-1]
        nth = torch.arange(n, device=q.device)
        real = nth < counts[:, None]
        rows = (starts[:-1, None] + nth).clamp(max=q.shape[0] - 1)
        pos = lengths[:, None] - counts[:, None] + nth
        held = s["pages"][i, :p // PAGE].long()
        ids = s["pages"][i:j, p // PAGE:width].long().clamp(min=0)
        x = _heads_first(q[rows], hkv)
        # What the group shares, once for all rows, then each member's own tokens.
        ks, vs = (s[y][held].flatten(0, 1).float().transpose(0, 1) for y in "kv")   # [Hkv, tokens, D]
        ko, vo = (s[y][ids].flatten(1, 2).float().transpose(1, 2) for y in "kv")    # [R, Hkv, tokens, D]
        every = x.transpose(0, 1).reshape(hkv, -1, d)
        a = torch.bmm(every, ks.transpose(1, 2).contiguous()).view(hkv, r, -1, n, p).transpose(0, 1)
        b = torch.bmm(x.reshape(r * hkv, -1, d), ko.transpose(2, 3).reshape(r * hkv, d, -1))
        scores = torch.cat((a.reshape(r, hq, n, p), b.view(r, hq, n, -1)), -1).mul_(1.0 / math.sqrt(d))
        weights = _weights(scores, pos, torch.arange(scores.shape[-1], device=q.device), lengths, rows,
                           s["options"])
        a = weights[..., :p].reshape(r, hkv, -1, p).transpose(0, 1).reshape(hkv, -1, p)
        b = weights[..., p:].reshape(r * hkv, hq // hkv * n, -1)
        y = torch.bmm(a, vs).view(hkv, r, -1, d).transpose(0, 1) + torch.bmm(
            b, vo.reshape(r * hkv, -1, d)).view(r, hkv, -1, d)
        y = y / weights.sum(-1).view(r, hkv, -1, 1).clamp(min=1e-30)
        out[rows[real]] = y.reshape(r, hq, n, d).transpose(1, 2)[real].to(q.dtype)
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
        return {"store": _plain_store, "read": _plain_read, "fp8": _plain_fp8, "shared": _plain_shared}[s["op"]](s)
    bt = _api()
    if s["op"] in ("store", "read"):
        pools = s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"]
        if s["op"] == "store":
            bt.append_fp8_kv_(*pools, s["k"], s["v"], s["slots"])
        return bt.read_fp8_kv(*pools, s["slots"], s["type"])
    if s["op"] == "fp8":
        return bt.fp8_chunk_attention(s["q"], s["k"], s["k_scale"], s["v"], s["v_scale"], s["pages"],
                                      s["lengths"], s["starts"], **s["options"])
    return bt.shared_chunk_attention(s["q"], s["k"], s["v"], s["pages"], s["lengths"], s["starts"], s["groups"],
                                     s["shared"], **s["options"])


# ---------------------------------------------------------------------------
# the definition, in 64 bits


def _rounded(x):
    """The e4m3 values nearest to x (|x| <= 448), ties to even: steps of 2^-3 of the power of two below."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _stored(x):
    """What rows [..., D] become in the cache."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    top = x.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100)
    unit = torch.exp2(torch.ceil(torch.log2(top / 448)))
    return (_rounded(x / unit) * unit).flatten(-2)


def _held(codes, scale):
    """The values of a pool [P, 16, Hkv, D]."""
    powers = scale.view(torch.uint8).transpose(1, 2).double() - 127
    return codes.double() * torch.exp2(powers).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    if c["op"] == "store":
        return tuple(_stored(s[x]) for x in "kv")
    if c["op"] == "read":
        slots = s["slots"].long()
        return tuple(_held(s[x + "_pool"], s[x + "_scale"]).flatten(0, 1)[slots] for x in "kv")
    d, group, at = c["d"], c["hq"] // c["hkv"], 0
    out = torch.empty(s["q"].shape, device="cuda", dtype=torch.float64)
    slopes = [2.0 ** (-8.0 * (h + 1) / c["hq"]) for h in range(c["hq"])]
    pools = [_held(s[x], s[x + "_scale"]) if c["op"] == "fp8" else s[x] for x in "kv"]
    for b, (new, (lo, hi)) in enumerate(zip(_counts(c), _ranges(c))):
        length = _prompts(c)[b] + _lengths(c)[b]
        ids = s["pages"][b, :_pages(length)].long()
        j = torch.arange(length, device="cuda")
        lo, hi = torch.from_numpy(lo).cuda()[:, None], torch.from_numpy(hi).cuda()[:, None]
        hidden = (j < lo) | (j > hi)
        distance = (torch.arange(length - new, length, device="cuda")[:, None] - j).abs().double()
        kv = [x[ids].flatten(0, 1)[:length].double() for x in pools]
        for h in range(c["hq"]):
            k, v = (x[:, h // group].contiguous() for x in kv)
            y = s["q"][at:at + new, h].double() @ k.t().contiguous() / math.sqrt(d)
            if _cap(c):
                y = _cap(c) * torch.tanh(y / _cap(c))
            if "bias" in c["form"]:
                y = y - slopes[h] * distance
            out[at:at + new, h] = torch.softmax(y.masked_fill(hidden, -math.inf), dim=-1) @ v
        at += new
    return out
