"""The operators of long contexts over the paged KV cache, as cases that can be timed and checked.

Five ways a serving program uses them, each through the library's public entry points:

* append: the norm of every query and key head, its rotation and the store of the new
  keys and values into the cache's pages, for one token, for a batch of sequences and
  for a whole prompt;
* bounds: the smallest and the largest key of each page, dimension by dimension, which
  the selection reads (of a prompt's pages);
* sparse: one decode step of attention over the pages that a cheap score selects: the
  newest page's bounds, the selection, the attention over the pages it lists;
* weights: one decode step of attention that also adds each position's softmax weight
  to what it has gathered so far;
* evict: the slots with the least weight leave a cache that holds too many.

Queries and keys have the size that a per-head norm gives them, with a drift from page
to page, as the keys of real text have; weights are spread over several powers of ten,
with exact zeros (slots just filled). Block tables are shuffled.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

ROOT = Path(__file__).resolve().parent.parent
PACKAGE = ROOT / "local-ai-gpu-acceleration_amd"
if str(PACKAGE) not in sys.path:
    sys.path.insert(0, str(PACKAGE))

own = False

DEV = "cuda:0"
THETA = 500000.0
EPS = 1e-6
NONE = 0xFFFFFFFF  # the position of a padded row
H_MAX = 65504.0    # the largest fp16 value


# ---- the cases ----------------------------------------------------------------


def listed() -> list[dict]:
    return [
        # One new token of one sequence at the 8B shape: latency.
        dict(name="append_1", kind="append", heads=32, kv=8, dim=128, rotary=128, pairing="halves", page=64, ctx=4000,
             count=1, pad=0, prompt=False, slots=False),
        # Six sequences in a batch of eight, small heads, partial rotation of adjacent
        # pairs, a cache that eviction keeps short: slot and position differ.
        dict(name="append_8", kind="append", heads=20, kv=4, dim=64, rotary=32, pairing="adjacent", page=16, ctx=1500,
             count=8, pad=2, prompt=False, slots=True),
        # A prompt of 4001 tokens at once: throughput.
        dict(name="append_prompt", kind="append", heads=32, kv=8, dim=128, rotary=128, pairing="halves", page=64,
             ctx=4001, count=4001, pad=0, prompt=True, slots=False),
        # The bounds of three short prompts' pages.
        dict(name="bounds_short", kind="bounds", heads=32, kv=8, dim=128, page=32, ctx=1999, count=3),
        # The bounds of a long prompt's pages.
        dict(name="bounds_long", kind="bounds", heads=32, kv=8, dim=128, page=64, ctx=65536, count=1),
        # One sequence of 16 thousand positions that attends 16 pages of 64.
        dict(name="sparse_1", kind="sparse", heads=32, kv=8, dim=128, page=64, ctx=16000, count=1, pad=0, select=16,
             first=1, last=2),
        # Eight users with contexts up to 65 thousand, 64 pages each.
        dict(name="sparse_8", kind="sparse", heads=32, kv=8, dim=128, page=64, ctx=65500, count=8, pad=0, select=64,
             first=1, last=2),
        # Wide heads, five to a key head, small pages, a padded batch.
        dict(name="sparse_wide", kind="sparse", heads=10, kv=2, dim=256, page=24, ctx=9001, count=4, pad=1, select=40,
             first=2, last=4),
        # One sequence with a budget of a few thousand positions.
        dict(name="weights_1", kind="weights", heads=32, kv=8, dim=128, page=64, ctx=4001, count=1, pad=0),
        # Eight sequences of up to 16 thousand.
        dict(name="weights_8", kind="weights", heads=32, kv=8, dim=128, page=64, ctx=16384, count=8, pad=0),
        # Eight sequences give up 64 positions each over a budget of 2048.
        dict(name="evict_step", kind="evict", heads=32, kv=8, dim=128, page=64, ctx=2112, count=8, keep=2048, first=4,
             recent=256, ragged=False),
        # Two prompts shrink to a budget of 4096.
        dict(name="evict_prompt", kind="evict", heads=32, kv=8, dim=128, page=64, ctx=32768, count=2, keep=4096,
             first=4, recent=512, ragged=True),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _heads(rng) -> dict:
    kv = rng.choice([1, 2, 4, 8])
    return dict(heads=kv * rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 12, 16]), kv=kv, dim=rng.choice([64, 128, 128, 256]),
                page=rng.choice([8, 16, 24, 32, 48, 64, 64, 128, 256]))


def draw(rng) -> dict:
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), work(c)["bytes"])
    kind = rng.choice(["append", "append", "bounds", "sparse", "sparse", "weights", "weights", "evict"])
    while True:
        c = dict(kind=kind, **_heads(rng))
        if kind == "append":
            prompt = rng.random() < 0.4
            c.update(rotary=rng.choice([8, c["dim"] // 4, c["dim"] // 2, c["dim"], c["dim"]]),
                     pairing=rng.choice(["halves", "adjacent"]), prompt=prompt, slots=rng.random() < 0.4)
            if prompt:
                n = _log(rng, 2, 8192)
                c.update(ctx=n + _log(rng, 1, 4096), count=n, pad=0)
            else:
                n = rng.randint(1, 12)
                c.update(ctx=_log(rng, 1, 16384), count=n, pad=rng.randint(0, n - 1) if rng.random() < 0.3 else 0)
        elif kind == "bounds":
            c.update(ctx=_log(rng, 1, 65536), count=rng.randint(1, 8))
        elif kind == "sparse":
            n, first, last = rng.randint(1, 8), rng.randint(0, 4), rng.randint(1, 4)
            c.update(ctx=_log(rng, 1, 65536), count=n, pad=rng.randint(0, n - 1) if rng.random() < 0.3 else 0,
                     select=max(first + last, _log(rng, 1, 128)), first=first, last=last)
        elif kind == "weights":
            n = rng.randint(1, 8)
            c.update(ctx=_log(rng, 1, 32768), count=n, pad=rng.randint(0, n - 1) if rng.random() < 0.3 else 0)
        else:
            ctx = _log(rng, 2, 32768)
            keep = rng.randint(1, ctx - 1) if rng.random() < 0.5 else max(1, ctx - _log(rng, 1, 128))
            first = rng.randint(0, min(8, keep))
            c.update(ctx=ctx, count=rng.randint(1, 8), keep=keep, first=first, recent=rng.randint(0, keep - first),
                     ragged=rng.random() < 0.4)
        if work(c)["bytes"] <= most[kind]:
            return c


def _lengths(case) -> list[int]:
    """Filled positions of each sequence: the first has ctx, the others less and less
    (0: a padded row)."""
    n, ctx = case["count"], case["ctx"]
    if case["kind"] == "append" and case["prompt"]:
        return [ctx]
    live = n - case.get("pad", 0)
    if not case.get("ragged", True):
        return [ctx] * n
    return [max(1, ctx * (live - i) // live) for i in range(live)] + [0] * (n - live)


def work(case) -> dict:
    heads, kv, dim, page = case["heads"], case["kv"], case["dim"], case["page"]
    lens, group = _lengths(case), heads // kv
    row = 2 * dim  # bytes of a cached key or value of one head
    if case["kind"] == "append":
        rows = case["count"] - case["pad"]
        moved = 4 * (2 * heads + 2 * kv) * dim + 2 * kv * row + (8 * kv if case["slots"] else 0) + 4
        return dict(bytes=rows * moved + 8 * dim, flops=rows * (heads + kv) * (4 * dim + 3 * case["rotary"]))
    if case["kind"] == "bounds":
        keys, pages = sum(lens) * kv, sum(-(-n // page) for n in lens) * kv
        return dict(bytes=keys * row + pages * (2 * row + 4), flops=2 * keys * dim)
    live = sum(n > 0 for n in lens)
    queries = live * heads * dim * 8  # the query and the result, fp32
    if case["kind"] == "sparse":
        pages = sum(-(-n // page) for n in lens) * kv
        seen = kv * sum(min(n, case["select"] * page) for n in lens)
        fresh = kv * sum((n - 1) % page + 1 for n in lens if n)
        listed_bytes = 4 * sum(min(-(-n // page), case["select"]) for n in lens) * kv
        return dict(bytes=pages * (2 * row + 4) + seen * 2 * row + fresh * row + listed_bytes + queries,
                    flops=4 * dim * group * (pages + seen) + 2 * fresh * dim)
    if case["kind"] == "weights":
        seen = kv * sum(lens)
        return dict(bytes=seen * (2 * row + 8) + queries + 4 * sum(-(-n // page) for n in lens),
                    flops=(4 * dim + 2) * group * seen)
    keep = case["keep"]
    stay = sum(min(n, keep) for n in lens)
    moves = sum((n - keep) * keep // n for n in lens if n > keep)  # kept slots behind the budget, spread evenly
    return dict(bytes=kv * (8 * sum(lens) + 8 * stay + moves * 4 * row), flops=kv * sum(lens))


# ---- inputs -------------------------------------------------------------------


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape) -> torch.Tensor:
    return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32)


def _ints(values) -> torch.Tensor:
    """uint32 values, held as int32 (torch's own unsigned type lacks most operations)."""
    return torch.tensor([v - (1 << 32) if v >= 1 << 31 else v for v in values], dtype=torch.int32, device=DEV)


def _inputs(case, seed) -> dict:
    g = _gen(seed)
    kind, heads, kv, dim, page = case["kind"], case["heads"], case["kv"], case["dim"], case["page"]
    lens = _lengths(case)
    entries = -(-max(lens) // page)
    n_pages = entries * len(lens)
    s = dict(case=case, lens=lens, entries=entries, capacity=entries * page)
    k = torch.empty(n_pages, kv, page, dim, dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    for i in range(0, n_pages, 512):
        part = k[i:i + 512]
        part.copy_(0.9 * _randn(g, *part.shape) + 0.45 * _randn(g, part.shape[0], kv, 1, dim))
        v[i:i + 512].copy_(_randn(g, *part.shape))
    table = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32).reshape(len(lens), entries).contiguous()
    s.update(k=k, v=v, table=table)
    rows = case["count"]
    if kind == "append":
        if case["prompt"]:
            last = range(case["ctx"] - rows, case["ctx"])
        else:
            last = [n - 1 if n else NONE for n in lens]
        s["slot"] = _ints(last)
        # after an eviction the positions run ahead of the slots
        s["pos"] = _ints([p if p == NONE or not case["slots"] else p + 20011 for p in last])
        # the three parts of one stacked projection's output
        stacked = _randn(g, rows, (heads + 2 * kv) * dim) * (0.2 + 3.0 * torch.rand(rows, 1, generator=g, device=DEV))
        q, kk, vv = stacked.split([heads * dim, kv * dim, kv * dim], dim=1)
        s.update(q=q.unflatten(1, (heads, dim)), knew=kk.unflatten(1, (kv, dim)), vnew=vv.unflatten(1, (kv, dim)),
                 qw=1.0 + 0.1 * _randn(g, dim), kw=1.0 + 0.1 * _randn(g, dim),
                 q_out=torch.zeros(rows, heads, dim, device=DEV))
        if case["slots"]:
            s["slot_pos"] = torch.zeros(len(lens), kv, s["capacity"], dtype=torch.int32, device=DEV)
            s["weight"] = torch.rand(len(lens), kv, s["capacity"], generator=g, device=DEV)
        return s
    if kind == "evict":
        cap = s["capacity"]
        s["weight"] = torch.exp(2.0 * _randn(g, rows, kv, cap)) * (torch.rand(rows, kv, cap, generator=g, device=DEV) < 0.9)
        # every slot holds another position, in order but for what earlier evictions moved
        order = torch.arange(cap, device=DEV) + 40.0 * (torch.rand(rows, kv, cap, generator=g, device=DEV) < 0.1)
        for r, n in enumerate(lens):
            order[r, :, n:] = 1e9  # (not filled)
        s["slot_pos"] = (3 * order.argsort(dim=-1, stable=True).argsort(dim=-1)).to(torch.int32).contiguous()
        s["pos"] = _ints([3 * (n - 1) for n in lens])
        s["length"] = _ints(lens)
        s.update(weight_out=torch.zeros_like(s["weight"]), slot_pos_out=torch.zeros_like(s["slot_pos"]),
                 length_out=torch.zeros_like(s["length"]))
        return s
    s["pos"] = _ints([n - 1 if n else NONE for n in lens])
    if kind != "bounds":
        s["q"] = _randn(g, rows, heads, dim)
        s["out"] = torch.zeros(rows, heads, dim, device=DEV)
    if kind == "weights":
        s["weight"] = torch.exp(2.0 * _randn(g, rows, kv, s["capacity"]))
        s["weight_out"] = torch.zeros_like(s["weight"])
    else:
        s["bounds"] = torch.zeros(n_pages, kv, 2, dim, dtype=torch.float16, device=DEV)
    if kind == "sparse":
        # the bounds of the earlier steps' pages
        for i in range(0, n_pages, 512):
            s["bounds"][i:i + 512, :, 0] = k[i:i + 512].amax(2)
            s["bounds"][i:i + 512, :, 1] = k[i:i + 512].amin(2)
        s["pages"] = torch.full((rows, kv, case["select"]), -1, dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed) -> dict:
    s = _inputs(case, seed)
    if not own:
        return s
    from rtxllm_amd import paged

    table = s["table"][0] if case["kind"] == "append" and case["prompt"] else s["table"]
    cache = s["cache"] = paged.PagedKV(s["k"], s["v"], table)
    rows, kind = case["count"], case["kind"]
    if kind == "sparse":
        s["work"] = paged.select_workspace(cache, rows)
        s["work2"] = paged.attn_pages_workspace(cache, case["heads"], case["select"], rows)
    elif kind == "weights":
        s["work"] = paged.attn_weights_workspace(cache, case["heads"], rows)
    elif kind == "evict":
        s["work"] = paged.evict_workspace(cache, case["keep"], rows)
    if kind in ("sparse", "weights", "evict"):
        # Several small launches: captured once and replayed, as this library's decode step is.
        _own(s)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                s["answer"] = _own(s)
        torch.cuda.current_stream().wait_stream(side)
        s["graph"] = graph
    return s


# ---- the library's operators ---------------------------------------------------


def _own(s):
    from rtxllm_amd import paged

    case, cache = s["case"], s["cache"]
    kind = case["kind"]
    if kind == "append":
        paged.qk_norm_rope_append(cache, s["q"], s["knew"], s["vnew"], s["qw"], s["kw"], s["pos"], theta=THETA, eps=EPS,
                                  rotary_dim=case["rotary"], pairing=case["pairing"], slot=s["slot"], q_out=s["q_out"],
                                  slot_pos=s.get("slot_pos"), slot_weight=s.get("weight"))
        return [s["q_out"], s["k"], s["v"]] + ([s["slot_pos"], s["weight"]] if case["slots"] else [])
    if kind == "bounds":
        paged.page_bounds(cache, s["pos"], s["bounds"], first=torch.zeros_like(s["pos"]), span=s["entries"])
        return s["bounds"]
    if kind == "sparse":
        paged.page_bounds(cache, s["pos"], s["bounds"])
        paged.select_pages(cache, s["bounds"], s["q"], s["pos"], case["select"], n_first=case["first"],
                           n_last=case["last"], pages=s["pages"], workspace=s["work"])
        paged.attn_pages(cache, s["q"], s["pages"], s["pos"], out=s["out"], workspace=s["work2"])
        return [s["bounds"], s["pages"], s["out"]]
    if kind == "weights":
        paged.attn_weights(cache, s["q"], s["pos"], s["weight"], weight_out=s["weight_out"], out=s["out"],
                           workspace=s["work"])
        return [s["out"], s["weight_out"]]
    paged.evict(cache, s["length"], s["pos"], case["keep"], s["weight"], s["slot_pos"], n_first=case["first"],
                n_recent=case["recent"], weight_out=s["weight_out"], slot_pos_out=s["slot_pos_out"],
                length_out=s["length_out"], workspace=s["work"])
    return [s["k"], s["v"], s["weight_out"], s["slot_pos_out"], s["length_out"]]


def run(s):
    if not own:
        return _PLAIN[s["case"]["kind"]](s)
    if "graph" in s:
        s["graph"].replay()
        return s["answer"]
    return _own(s)


# ---- the plain forms -----------------------------------------------------------


def _rotate(x, pos, rotary, pairing):
    """x [rows][heads][dim] at the 64-bit angles pos * theta^(-2i / rotary)."""
    i = torch.arange(rotary // 2, device=DEV, dtype=torch.float64)
    angle = pos.double()[:, None] * THETA ** (-2.0 * i / rotary)
    c, sn = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = rotary // 2
    a, b = (slice(0, half), slice(half, rotary)) if pairing == "halves" else (slice(0, rotary, 2), slice(1, rotary, 2))
    out = x.clone()
    out[..., a] = x[..., a] * c - x[..., b] * sn
    out[..., b] = x[..., a] * sn + x[..., b] * c
    return out


def _plain_append(s):
    case = s["case"]
    page, kv = case["page"], case["kv"]
    rows = case["count"] - case["pad"]
    pos, slot = s["pos"][:rows].long(), s["slot"][:rows].long()
    seq = torch.zeros_like(slot) if case["prompt"] else torch.arange(rows, device=DEV)

    def normed(x, w):
        x = x[:rows]
        return _rotate(x * (1.0 / ((x * x).mean(-1, keepdim=True) + EPS).sqrt()) * w, pos, case["rotary"], case["pairing"])

    q_out = torch.zeros_like(s["q_out"])
    q_out[:rows] = normed(s["q"], s["qw"])
    at = s["table"][seq, slot // page].long()
    s["k"][at, :, slot % page] = normed(s["knew"], s["kw"]).to(torch.float16)
    s["v"][at, :, slot % page] = s["vnew"][:rows].to(torch.float16)
    if not case["slots"]:
        return [q_out, s["k"], s["v"]]
    s["slot_pos"][seq, :, slot] = pos.to(torch.int32)[:, None].expand(rows, kv)
    s["weight"][seq, :, slot] = 0.0
    return [q_out, s["k"], s["v"], s["slot_pos"], s["weight"]]


def _bounds_of(s, bounds, row, first, n):
    """The bounds of logical pages first.. of a sequence with n filled positions."""
    page = s["case"]["page"]
    at = s["table"][row, first:-(-n // page)].long()
    keys = s["k"][at].float()  # [pages][kv][page][dim]
    there = (torch.arange(keys.shape[0] * page, device=DEV) + first * page < n).reshape(-1, 1, page, 1)
    there = there & ~keys.isnan()
    bounds[at, :, 0] = keys.masked_fill(~there, -H_MAX).amax(2).clamp(-H_MAX, H_MAX).to(torch.float16)
    bounds[at, :, 1] = keys.masked_fill(~there, H_MAX).amin(2).clamp(-H_MAX, H_MAX).to(torch.float16)


def _plain_bounds(s):
    for r, n in enumerate(s["lens"]):
        _bounds_of(s, s["bounds"], r, 0, n)
    return s["bounds"]


def _attend(s, r, at):
    """Plain attention of row r over logical positions at [kv][n] (ascending, all filled):
    the result [kv][group][dim] and the softmax weights [kv][group][n]."""
    case = s["case"]
    kv, page = case["kv"], case["page"]
    phys, off = s["table"][r][at // page].long(), at % page
    head = torch.arange(kv, device=DEV)[:, None]
    keys, values = s["k"][phys, head, off].float(), s["v"][phys, head, off].float()
    q = s["q"][r].reshape(kv, -1, case["dim"]) * (1.0 / math.sqrt(case["dim"]))
    score = torch.matmul(q, keys.transpose(1, 2).contiguous())
    e = (score - score.amax(-1, keepdim=True)).exp()
    p = e / e.sum(-1, keepdim=True)
    return torch.matmul(p, values), p


def _plain_sparse(s):
    case = s["case"]
    kv, dim, page, select = case["kv"], case["dim"], case["page"], case["select"]
    out, pages = torch.zeros_like(s["out"]), torch.full_like(s["pages"], -1)
    for r, n in enumerate(s["lens"]):
        if n == 0:
            continue
        used = -(-n // page)
        _bounds_of(s, s["bounds"], r, used - 1, n)
        # the selection is decided in 64 bits: scores may lie close to one another
        b = s["bounds"][s["table"][r, :used].long()].double()  # [used][kv][2][dim]
        q = s["q"][r].double().reshape(kv, -1, dim)
        score = torch.full((kv, used), -math.inf, dtype=torch.float64, device=DEV)
        for h in range(q.shape[1]):
            best = torch.maximum(q[:, h] * b[:, :, 0], q[:, h] * b[:, :, 1]).sum(-1)
            score = torch.maximum(score, best.T)
        score[:, :case["first"]] = math.inf
        score[:, max(0, used - case["last"]):] = math.inf
        take = min(used, select)
        chosen = score.sort(dim=-1, descending=True, stable=True).indices[:, :take].sort(-1).values
        pages[r, :, :take] = chosen.to(torch.int32)
        at = (chosen[:, :, None] * page + torch.arange(page, device=DEV)).reshape(kv, -1)
        if bool(case["last"]):  # the newest page is the last one listed: it alone may end early
            at = at[:, :(take - 1) * page + (n - 1) % page + 1]
        out[r] = _attend(s, r, at)[0].reshape(-1, dim)
    return [s["bounds"], pages, out]


def _plain_weights(s):
    out, weight = torch.zeros_like(s["out"]), torch.zeros_like(s["weight"])
    for r, n in enumerate(s["lens"]):
        if n == 0:
            continue
        at = torch.arange(n, device=DEV).expand(s["case"]["kv"], n)
        o, p = _attend(s, r, at)
        out[r] = o.reshape(-1, s["case"]["dim"])
        weight[r, :, :n] = s["weight"][r, :, :n] + p.sum(1)
    return [out, weight]


def _plain_evict(s):
    case = s["case"]
    keep, page = case["keep"], case["page"]
    weight, slot_pos = torch.zeros_like(s["weight"]), torch.zeros_like(s["slot_pos"])
    for r, n in enumerate(s["lens"]):
        w, p = s["weight"][r, :, :n], s["slot_pos"][r, :, :n]
        if n <= keep:
            weight[r, :, :n], slot_pos[r, :, :n] = w, p
            continue
        stays = (p < case["first"]) | (p.long() + case["recent"] > s["pos"][r].long())
        order = w.masked_fill(stays, math.inf).sort(dim=-1, descending=True, stable=True).indices[:, :keep]
        kept = torch.zeros_like(stays).scatter_(1, order, True)
        head, hole = (~kept[:, :keep]).nonzero(as_tuple=True)
        source = kept[:, keep:].nonzero(as_tuple=True)[1] + keep  # the i-th kept slot behind goes into the i-th hole
        weight[r, :, :keep], slot_pos[r, :, :keep] = w[:, :keep], p[:, :keep]
        weight[r, head, hole], slot_pos[r, head, hole] = w[head, source], p[head, source]
        to, of = s["table"][r][hole // page].long(), s["table"][r][source // page].long()
        for c in (s["k"], s["v"]):
            c[to, head, hole % page] = c[of, head, source % page]
    return [s["k"], s["v"], weight, slot_pos, s["length"].clamp(max=keep)]


_PLAIN = dict(append=_plain_append, bounds=_plain_bounds, sparse=_plain_sparse, weights=_plain_weights,
              evict=_plain_evict)


# ---- the definitions in 64 bits --------------------------------------------------


def _slots(s, r, head, slots):
    """Flat row numbers of a sequence's slots in the [page][kv][slot] order of the cache."""
    page, kv = s["case"]["page"], s["case"]["kv"]
    return (s["table"][r].long()[slots // page] * kv + head) * page + slots % page


def _softmax_rows(s, r, head, query, slots):
    dim = s["case"]["dim"]
    rows = _slots(s, r, head, slots)
    score = s["k"].reshape(-1, dim)[rows].double() @ query.double() / math.sqrt(dim)
    p = torch.exp(score - torch.logsumexp(score, 0))
    return p, p @ s["v"].reshape(-1, dim)[rows].double()


def exact(case, seed):
    s = _inputs(case, seed)
    kind, kv, dim, page = case["kind"], case["kv"], case["dim"], case["page"]
    group = case["heads"] // kv
    if kind == "append":
        return _exact_append(s)
    if kind == "evict":
        return _exact_evict(s)
    if kind == "weights":
        out, weight = s["out"].double(), s["weight_out"].double()
        for r, n in enumerate(s["lens"]):
            for h in range(case["heads"] if n else 0):
                p, o = _softmax_rows(s, r, h // group, s["q"][r, h], torch.arange(n, device=DEV))
                if h % group == 0:
                    weight[r, h // group, :n] = s["weight"][r, h // group, :n].double()
                weight[r, h // group, :n] += p
                out[r, h] = o
        return [out, weight]
    bounds = s["bounds"].double()
    for r, n in enumerate(s["lens"]):
        for t in range(0 if kind == "bounds" else max(0, (n - 1) // page), -(-n // page)):
            keys = s["k"][int(s["table"][r, t]), :, :min(page, n - t * page)].double()
            bounds[int(s["table"][r, t])] = torch.stack([keys.max(1).values, keys.min(1).values], 1)
    if kind == "bounds":
        return bounds
    out, pages = s["out"].double(), s["pages"].clone()
    for r, n in enumerate(s["lens"]):
        used = -(-n // page)
        for g in range(kv if n else 0):
            b = bounds[s["table"][r, :used].long(), g]
            q = s["q"][r, g * group:(g + 1) * group].double()
            top = (q.clamp(min=0.0) @ b[:, 0].T + q.clamp(max=0.0) @ b[:, 1].T).amax(0).cpu().tolist()
            forced = set(range(min(case["first"], used))) | set(range(max(0, used - case["last"]), used))
            ranked = sorted(range(used), key=lambda t: (t not in forced, -top[t], t))
            chosen = sorted(ranked[:case["select"]])
            pages[r, g, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32, device=DEV)
            slots = torch.tensor([p for t in chosen for p in range(t * page, min(n, t * page + page))], device=DEV)
            for h in range(g * group, (g + 1) * group):
                out[r, h] = _softmax_rows(s, r, g, s["q"][r, h], slots)[1]
    return [bounds, pages, out]


def _exact_append(s):
    case = s["case"]
    dim, rotary, half = case["dim"], case["rotary"], case["rotary"] // 2
    rows = case["count"] - case["pad"]
    pos = s["pos"][:rows].double()
    parts = []
    for x, w in ((s["q"], s["qw"]), (s["knew"], s["kw"])):
        x = x[:rows].double()
        x = x / torch.sqrt(x.square().sum(-1, keepdim=True) / dim + EPS) * w.double()
        if case["pairing"] == "halves":
            z = torch.complex(x[..., :half], x[..., half:rotary])
        else:
            z = torch.view_as_complex(x[..., :rotary].unflatten(-1, (half, 2)).contiguous())
        turn = torch.outer(pos, torch.exp(torch.arange(half, device=DEV, dtype=torch.float64) * (-2.0 * math.log(THETA) / rotary)))
        z = z * torch.polar(torch.ones_like(turn), turn)[:, None]
        turned = torch.cat([z.real, z.imag], -1) if case["pairing"] == "halves" else torch.view_as_real(z).flatten(-2)
        parts.append(torch.cat([turned, x[..., rotary:]], -1))
    q_out = s["q_out"].double()
    q_out[:rows] = parts[0]
    k, v = s["k"].double().reshape(-1, dim), s["v"].double().reshape(-1, dim)
    slot = s["slot"][:rows].long()
    for r in range(1 if case["prompt"] else rows):
        of = slice(None) if case["prompt"] else slice(r, r + 1)
        for g in range(case["kv"]):
            at = _slots(s, r, g, slot[of])
            k[at], v[at] = parts[1][of, g], s["vnew"][:rows][of, g].double()
    answer = [q_out, k.reshape(s["k"].shape), v.reshape(s["v"].shape)]
    if case["slots"]:
        slot_pos, weight = s["slot_pos"], s["weight"].double()
        for i in range(rows):
            r = 0 if case["prompt"] else i
            slot_pos[r, :, int(slot[i])], weight[r, :, int(slot[i])] = s["pos"][i], 0.0
        answer += [slot_pos, weight]
    return answer


def _exact_evict(s):
    case = s["case"]
    keep, dim = case["keep"], case["dim"]
    k, v = s["k"].reshape(-1, dim), s["v"].reshape(-1, dim)
    weight, slot_pos = s["weight_out"].double(), s["slot_pos_out"].clone()
    for r, n in enumerate(s["lens"]):
        newest = int(s["pos"][r])
        for g in range(case["kv"]):
            w, p = s["weight"][r, g, :n].cpu().tolist(), s["slot_pos"][r, g, :n].cpu().tolist()
            order = sorted(range(n), key=lambda i: (not (p[i] < case["first"] or p[i] + case["recent"] > newest), -w[i], i))
            kept = set(order[:keep])
            where = list(range(min(n, keep)))
            late = iter(sorted(i for i in kept if i >= keep))
            where = [i if i in kept else next(late) for i in where]
            at = torch.tensor(where, device=DEV)
            weight[r, g, :len(where)] = s["weight"][r, g][at].double()
            slot_pos[r, g, :len(where)] = s["slot_pos"][r, g][at]
            moved = torch.tensor([i for i, j in enumerate(where) if i != j], dtype=torch.long, device=DEV)
            to, of = _slots(s, r, g, moved), _slots(s, r, g, at[moved])
            k[to], v[to] = k[of], v[of]
    return [s["k"].double(), s["v"].double(), weight, slot_pos, s["length"].clamp(max=keep)]
