"""The operators of a paged key-value cache as measurable cases.

A case is one call that a host makes per layer around its attention: new keys
and values put into the cache (as they are or in 8-bit floats, quantised as they
are written), a part of the cache read back as BF16, or the attention of one new
token per sequence over the cache. Sizes are those of the layers that the
benchmark and the tests use (16 heads of 128, every one with its own keys) and
generic ones with shared key heads, other head sizes and lengths.

A cache holds pages of ``page`` tokens, [pages, kv_heads, page, dim]; row b of a
page table names the pages of sequence b in order, each page wherever it was
free. In 8 bits a token's keys (values) of one head share a scale: d =
max|v| / 448, at least 2^-126, 1 for zeros; code = e4m3(v / d).
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda:0"
FP8_MAX = 448.0
TINY = 2.0 ** -126


def listed():
    return [
        # One user, the first tokens of an answer: latency counts.
        {"name": "attend_b1_short", "op": "attend", "batch": 1, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16,
         "fp8": True, "low": 77, "high": 77, "window": 0},
        # The benchmark's batch of 32 sequences, of every age.
        {"name": "attend_b32", "op": "attend", "batch": 32, "heads": 16, "kv_heads": 16, "dim": 128, "page": 64,
         "fp8": False, "low": 1, "high": 2047, "window": 0},
        # A window over sequences of which one is empty, seven query heads to a
        # key head, heads of 80.
        {"name": "attend_b13_window", "op": "attend", "batch": 13, "heads": 28, "kv_heads": 4, "dim": 80, "page": 32,
         "fp8": True, "low": 0, "high": 1999, "window": 1000},
        # One long document with shared key heads: a few rows, all of the length.
        {"name": "attend_b1_long", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "dim": 128, "page": 128,
         "fp8": False, "low": 131071, "high": 131071, "window": 0},
        # A full server: 64 long conversations in 8 bits.
        {"name": "attend_b64_fp8", "op": "attend", "batch": 64, "heads": 16, "kv_heads": 16, "dim": 128, "page": 16,
         "fp8": True, "low": 4001, "high": 8191, "window": 0},
        # Decode of one sequence: its new token joins the cache.
        {"name": "append_b1", "op": "append", "batch": 1, "kv_heads": 16, "dim": 128, "page": 16, "fp8": True,
         "fewest": 1, "tokens": 1, "past": 77},
        # Decode of the benchmark's 32 sequences, kept in BF16.
        {"name": "append_b32", "op": "append", "batch": 32, "kv_heads": 16, "dim": 128, "page": 64, "fp8": False,
         "fewest": 1, "tokens": 1, "past": 2046},
        # Next turns of five conversations, padded to the longest.
        {"name": "append_b5_ragged", "op": "append", "batch": 5, "kv_heads": 4, "dim": 80, "page": 32, "fp8": True,
         "fewest": 41, "tokens": 333, "past": 1500},
        # Eight long prompts prefilled together.
        {"name": "append_b8_t4095", "op": "append", "batch": 8, "kv_heads": 16, "dim": 128, "page": 16, "fp8": True,
         "fewest": 2500, "tokens": 4095, "past": 0},
        # A conversation's next turn attends to what the cache holds of it.
        {"name": "read_b1", "op": "read", "batch": 1, "kv_heads": 16, "dim": 128, "page": 16, "fp8": True,
         "low": 777, "high": 777},
        # Three documents of different length, in BF16.
        {"name": "read_b3_long", "op": "read", "batch": 3, "kv_heads": 8, "dim": 128, "page": 128, "fp8": False,
         "low": 5000, "high": 32767},
        # The same of eight sequences in 8 bits.
        {"name": "read_b8_fp8", "op": "read", "batch": 8, "kv_heads": 16, "dim": 128, "page": 64, "fp8": True,
         "low": 1001, "high": 8191},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, evenly over their logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    # (heads, key heads): every head its own, shared by 2 to 16, all one
    heads, kv_heads = rng.choice([(16, 16), (16, 16), (12, 6), (32, 8), (28, 4), (40, 5), (32, 2), (8, 1)])
    dim = rng.choice([128, 128, 128, 64, 80, 96, 192, 256])
    base = {"kv_heads": kv_heads, "dim": dim, "page": rng.choice([16, 16, 32, 64, 128, 256]), "fp8": rng.random() < 0.5}
    op = rng.choice(["attend", "attend", "append", "read"])
    most = max(work(c)["bytes"] for c in listed() if c["op"] == op)
    while True:
        case = {"op": op, "batch": _spread(rng, 1, 64), **base}
        if op == "append":
            case["tokens"] = 1 if rng.random() < 0.3 else _spread(rng, 1, 4095)
            case["fewest"] = rng.randint(0, case["tokens"])
            case["past"] = rng.randint(0, 2000)
        else:
            case["high"] = _spread(rng, 1, 131071 if op == "attend" else 32767)
            case["low"] = rng.randint(0, case["high"])
            if op == "attend":
                case["heads"] = heads
                case["window"] = rng.choice([0, 0, _spread(rng, 1, case["high"])])
        # (the widest sequence is what a dense form holds for all of them)
        widest = dict(case, low=case.get("high", 0), window=0, fewest=case.get("tokens", 0))
        if work(widest)["bytes"] <= most:
            return case


def _between(low, high, n):
    """n whole numbers from low to high, evenly; high alone for n = 1."""
    return [high] if n == 1 else [low + (high - low) * i // (n - 1) for i in range(n)]


def work(case):
    token = 4 * case["dim"]  # keys and values of one head in BF16
    held = 2 * case["dim"] + 8 if case["fp8"] else token
    batch, kv_heads = case["batch"], case["kv_heads"]
    if case["op"] == "append":
        tokens = sum(_between(case["fewest"], case["tokens"], batch))
        return {"bytes": tokens * kv_heads * (token + held) + 12 * batch, "flops": 6 * tokens * kv_heads * case["dim"]}
    lengths = _between(case["low"], case["high"], batch)
    if case["op"] == "read":
        return {"bytes": kv_heads * (sum(lengths) * held + batch * case["high"] * token)
                + 4 * sum(-(-n // case["page"]) for n in lengths),
                "flops": 2 * sum(lengths) * kv_heads * case["dim"]}
    seen = sum(min(n, case["window"] or n) for n in lengths)
    pages = sum(min(-(-n // case["page"]), (case["window"] or n) // case["page"] + 1) for n in lengths)
    return {"bytes": seen * kv_heads * held + 4 * batch * case["heads"] * case["dim"] + 4 * pages + 4 * batch,
            "flops": 4 * seen * case["heads"] * case["dim"]}


# ------------------------------------------------------------- plain form --
def _quantized(v):
    """Codes and scales of v [..., dim] (float), a scale for each row."""
    most = v.abs().amax(-1)
    d = torch.where(most == 0, torch.ones_like(most), (most / FP8_MAX).clamp_min(TINY))
    return (v / d[..., None]).to(torch.float8_e4m3fn), d


def _gathered(pages, scales, table, length):
    """[batch, kv_heads, length, dim] in 32 bits: what the table's pages hold."""
    batch, width = table.shape
    used = _bytes(pages)[table.clamp_min(0).long()].view(pages.dtype).float()  # [batch, width, kv_heads, page, dim]
    if scales is not None:
        used = used * scales[table.clamp_min(0).long()][..., None]
    return used.transpose(1, 2).reshape(batch, pages.shape[1], width * pages.shape[2], -1)[:, :, :length]


def _visible(lengths, longest, window):
    """[batch, longest]: the positions that the next token of a sequence sees."""
    at = torch.arange(longest, device=lengths.device)
    seen = at < lengths[:, None]
    return seen & (at >= lengths[:, None] - window) if window else seen


def _bytes(t):
    """The tensor's elements as a type that every indexing operation takes."""
    return t.view(torch.uint8) if t.dtype is torch.float8_e4m3fn else t


# ----------------------------------------------------------------- inputs --
def prepare(case, seed):
    """What a host holds before the call: the layer's cache, in use (whatever
    finished sequences left in its other places), the page table, lengths and
    the new token's queries, or new keys and values as a projection gives them."""
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    batch, kv_heads, dim, page = case["batch"], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device=DEVICE) * std

    def mixed(values):
        order = torch.randperm(batch, generator=g, device=DEVICE)
        return torch.tensor(values, dtype=torch.int32, device=DEVICE)[order]

    state = dict(case)
    if case["op"] == "append":
        state["starts"] = mixed(_between(0, case["past"], batch) if batch > 1 else [case["past"]])
        state["counts"] = mixed(_between(case["fewest"], case["tokens"], batch))
        longest, ends = case["past"] + case["tokens"], state["starts"] + state["counts"]
    else:
        state["lengths"] = mixed(_between(case["low"], case["high"], batch))
        longest, ends = case["high"], state["lengths"]
    width = max(1, -(-longest // page))
    used = (ends + page - 1) // page
    here = torch.arange(width, device=DEVICE) < used[:, None]
    count = int(used.sum()) + 3
    free = torch.randperm(count, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=DEVICE)
    table[here] = free[:int(used.sum())]
    state["table"] = table

    channel = torch.exp(0.5 * normal(kv_heads, 1, dim))  # some channels of the keys are larger throughout
    for name, scale in (("k", channel), ("v", 1.0)):
        pages = torch.empty(count, kv_heads, page, dim, device=DEVICE,
                            dtype=torch.float8_e4m3fn if case["fp8"] else torch.bfloat16)
        scales = torch.empty(count, kv_heads, page, device=DEVICE) if case["fp8"] else None
        step = max(1, (1 << 28) // (kv_heads * page * dim))
        for i in range(0, count, step):  # (a full server's cache in 32 bits would be four times the state)
            v = (normal(min(step, count - i), kv_heads, page, dim) * scale).to(torch.bfloat16)
            if case["fp8"]:
                codes, scales[i:i + step] = _quantized(v.float())
                _bytes(pages)[i:i + step] = _bytes(codes)
            else:
                pages[i:i + step] = v
        state[name + "_pages"], state[name + "_scales"] = pages, scales
        if case["op"] == "append":
            # a projection gives [batch, tokens, heads * dim]; heads come first by a view
            new = normal(batch, case["tokens"], kv_heads, dim).to(torch.bfloat16).transpose(1, 2)
            state[name] = (new * scale).to(torch.bfloat16) if name == "k" else new
    if case["op"] == "attend":
        state["q"] = (1.5 * normal(batch, case["heads"], dim)).to(torch.bfloat16)
    return state


# ------------------------------------------------------------------- runs --
@functools.lru_cache(maxsize=None)
def _extension():
    """The library's operators and its cache type, as a host loads them once."""
    package = str(Path.cwd() / "uma-qmoe_amd")
    if package not in sys.path:
        sys.path.insert(0, package)
    from uma_qmoe_amd.native_backend import KVCache, load_native_extension

    return load_native_extension()[1], KVCache


def _held(s):
    """The cache after an append, whole."""
    out = {"k": s["k_pages"], "v": s["v_pages"]}
    if s["fp8"]:
        out["k_scales"], out["v_scales"] = s["k_scales"], s["v_scales"]
    return out


def _run_own(s):
    ext, cache = _extension()
    kv = cache(s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"])
    if s["op"] == "append":
        ext.kv_append(kv, s["k"], s["v"], s["table"], s["starts"], s["counts"])
        return _held(s)
    if s["op"] == "read":
        return ext.kv_read(kv, s["table"], s["lengths"], s["high"])
    return ext.paged_attention(s["q"], kv, s["table"], s["lengths"], window=s["window"] or None)


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "append":
        at = torch.arange(s["tokens"], device=s["k"].device)
        b, j = (at < s["counts"][:, None]).nonzero(as_tuple=True)
        position = s["starts"][b].long() + j
        page, slot = s["table"][b, position // s["page"]].long(), position % s["page"]
        for name in "kv":
            new = s[name].transpose(1, 2)[b, j]  # [tokens, kv_heads, dim]
            if s["fp8"]:
                new, s[name + "_scales"][page, :, slot] = _quantized(new.float())
            _bytes(s[name + "_pages"])[page, :, slot] = _bytes(new)
        return _held(s)
    if s["op"] == "read":
        seen = _visible(s["lengths"], s["high"], 0)[:, None, :, None]
        return tuple(torch.where(seen, _gathered(s[n + "_pages"], s[n + "_scales"], s["table"], s["high"]), 0.0)
                     .to(torch.bfloat16) for n in "kv")
    batch, heads, dim = s["q"].shape
    seen = _visible(s["lengths"], s["high"], s["window"])[:, None, :, None]
    q = s["q"].float().view(batch, s["kv_heads"], -1, dim).transpose(2, 3).contiguous() / math.sqrt(dim)
    keys = _gathered(s["k_pages"], s["k_scales"], s["table"], s["high"])
    scores = (keys @ q).masked_fill(~seen, -math.inf)  # [batch, kv_heads, length, queries of a key head]
    del keys
    most = scores.amax(2, keepdim=True)
    p = torch.exp(scores - torch.where(most == -math.inf, 0.0, most))
    values = _gathered(s["v_pages"], s["v_scales"], s["table"], s["high"])
    total = p.sum(2).unsqueeze(-1)
    out = p.transpose(2, 3).contiguous() @ torch.where(seen, values, 0.0)
    return torch.where(total > 0, out / total, 0.0).reshape(batch, heads, dim).to(torch.bfloat16)


# ------------------------------------------------------- 64-bit definition --
def _exact_rows(s, name, b, first, last):
    """Positions first .. last - 1 of sequence b, [kv_heads, last - first, dim]."""
    at = torch.arange(first, last, device=DEVICE)
    page, slot = s["table"][b, at // s["page"]].long(), at % s["page"]
    rows = _bytes(s[name + "_pages"])[page, :, slot].view(s[name + "_pages"].dtype).double()
    if s["fp8"]:
        rows *= s[name + "_scales"][page, :, slot].double()[..., None]
    return rows.transpose(0, 1)


def exact(case, seed):
    s = prepare(case, seed)
    batch, kv_heads, dim = case["batch"], case["kv_heads"], case["dim"]
    if case["op"] == "append":
        out = {n: t.double() for n, t in _held(s).items()}
        starts, counts = s["starts"].tolist(), s["counts"].tolist()
        for b in range(batch):
            at = torch.arange(starts[b], starts[b] + counts[b], device=DEVICE)
            page, slot = s["table"][b, at // case["page"]].long(), at % case["page"]
            for n in "kv":
                rows = s[n][b, :, :counts[b]].double()
                if case["fp8"]:
                    d = rows.abs().max(2).values / FP8_MAX
                    d[d == 0] = 1.0
                    d = d.clamp(min=TINY)
                    rows = rows / d[..., None]
                    out[n + "_scales"][page, :, slot] = d.t()
                out[n][page, :, slot] = rows.transpose(0, 1)
        return out
    lengths = s["lengths"].tolist()
    if case["op"] == "read":
        out = [torch.zeros(batch, kv_heads, case["high"], dim, dtype=torch.float64, device=DEVICE) for _ in "kv"]
        for b, n in enumerate(lengths):
            for t, name in zip(out, "kv"):
                t[b, :, :n] = _exact_rows(s, name, b, 0, n)
        return tuple(out)
    out = torch.zeros(batch, case["heads"], dim, dtype=torch.float64, device=DEVICE)
    group = case["heads"] // kv_heads
    for b, n in enumerate(lengths):
        if n == 0:
            continue
        first = max(0, n - case["window"]) if case["window"] else 0
        keys, values = _exact_rows(s, "k", b, first, n), _exact_rows(s, "v", b, first, n)
        for r in range(group):
            q = s["q"][b, r::group].double()
            scores = (keys * q[:, None]).sum(2) / dim ** 0.5
            out[b, r::group] = (torch.softmax(scores, 1)[..., None] * values).sum(1)
    return out
