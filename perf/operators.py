"""What the operators of the 8-bit page cache are measured by.

A server whose context memory is the limit keeps keys and values in 8 bits: page pools ``[num_blocks, kv_heads, 16, head_dim]`` of
e4m3 numbers, and for every page and kv head one power-of-two scale for the keys and one for the values, ``[num_blocks, kv_heads]``
e8m0 numbers between 2^-32 and 2^31.  Four operators make up one pass of such a server:

  map      from request lengths: pages for the new tokens out of a list of free ones, and per new token its sequence, position
           and slot (page * 16 + offset)                                                    ``ops.kv_slot_map``
  append   new keys and values into their slots.  The scale of a page is the smallest power of two for which its largest finite
           number fits; it grows with what is added, the page's earlier numbers are then rounded anew, and begins anew with a
           page's first token                                                               ``ops.kv8_append``
  decode   attention of one new token per sequence over its pages                           ``ops.kv8_attn_decode``
  prompt   causal attention of consecutive tokens of one sequence over its pages            ``ops.kv8_attn_prefill``

Head layouts are those of the built-in models (32, 64 or 16 query heads on 4 or 2 kv heads, head_dim 128 and 64).  Pages lie
shuffled in the pools, table entries behind a sequence's last page are no page, and slots behind its last token hold NaN.
Lengths of a batch are sizes: they come from the case and not from the seed.
"""
from __future__ import annotations

import importlib
import math
import random

import torch

own = False

PAGE = 16
DEV = "cuda"
BF, F8, E8 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
LOW, HIGH, TOP = -32, 31, 448.0  # exponents of a scale, the largest e4m3 number


# ---------------------------------------------------------------------- cases


def listed() -> list[dict]:
    return [
        # the bookkeeping of one decode step of a full batch: 256 sequences, one token each, a page for every sixteenth of them
        dict(name="map-step-256", op="map", rows=256, new_min=1, new_max=1, ctx_min=512, ctx_max=4096, pages=320),
        # a batch of prompts, some behind a cached prefix, padded to a round number of rows
        dict(name="map-prompts-48", op="map", rows=48, new_min=1, new_max=1500, ctx_min=0, ctx_max=2000, pages=256),
        # the new tokens of a decode step, one in each of 256 pages
        dict(name="append-step-256", op="append", rows=256, new_min=1, new_max=1, ctx_min=512, ctx_max=4096, kv_heads=4, head_dim=128, dtype="bf16"),
        # prompts that begin and end inside pages
        dict(name="append-prompts-8", op="append", rows=8, new_min=333, new_max=2048, ctx_min=0, ctx_max=100, kv_heads=4, head_dim=128, dtype="bf16"),
        # a small model in fp32 whose prompts are short
        dict(name="append-fp32-61", op="append", rows=61, new_min=1, new_max=40, ctx_min=0, ctx_max=300, kv_heads=2, head_dim=64, dtype="fp32"),
        # one user: every launch and every dependent load shows
        dict(name="decode-1", op="decode", rows=1, ctx_min=777, ctx_max=777, q_heads=32, kv_heads=4, head_dim=128),
        # one user with a long document
        dict(name="decode-1-long", op="decode", rows=1, ctx_min=131001, ctx_max=131001, q_heads=32, kv_heads=4, head_dim=128),
        # the headline batch of the framework: 256 sequences
        dict(name="decode-256", op="decode", rows=256, ctx_min=512, ctx_max=4096, q_heads=32, kv_heads=4, head_dim=128),
        # a small model, an odd number of chats of all ages, some of them empty rows
        dict(name="decode-d64-33", op="decode", rows=33, ctx_min=0, ctx_max=2900, q_heads=16, kv_heads=2, head_dim=64),
        # a prompt of the benchmark's length
        dict(name="prompt-2048", op="prompt", tokens=2048, cached=0, q_heads=32, kv_heads=4, head_dim=128),
        # a chunk of a long prompt
        dict(name="prompt-1024-deep", op="prompt", tokens=1024, cached=14336, q_heads=32, kv_heads=4, head_dim=128),
        # a short question about a long document, 16 query heads per kv head
        dict(name="prompt-17-deep", op="prompt", tokens=17, cached=14001, q_heads=64, kv_heads=4, head_dim=128),
    ]


HEADS = ((32, 4, 128), (64, 4, 128), (16, 2, 64), (8, 2, 64), (32, 4, 128))


def spread(rng, lo: int, hi: int) -> int:
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(hi + 1))))))


def draw(rng) -> dict:
    op = rng.choice(("map", "append", "decode", "prompt"))
    hq, hkv, d = rng.choice(HEADS)
    if op == "map":
        rows, step = spread(rng, 1, 256), rng.random() < 0.5
        most = 1 if step else min(spread(rng, 2, 2000), 60000 // rows + 1)
        return dict(op=op, rows=rows, new_min=1 if step else 0, new_max=most, ctx_min=rng.choice((0, 500)), ctx_max=spread(rng, 501, 2900), pages=320)
    if op == "append":
        rows, step = spread(rng, 1, 256), rng.random() < 0.4
        most = 1 if step else min(spread(rng, 2, 2000), 9000 // rows + 1)
        return dict(op=op, rows=rows, new_min=1, new_max=most, ctx_min=0, ctx_max=spread(rng, 1, 2000), kv_heads=hkv, head_dim=d, dtype=rng.choice(("bf16", "fp32")))
    if op == "decode":
        rows = spread(rng, 1, 256)
        most = min(spread(rng, 1, 120000), 590000 // rows)
        return dict(op=op, rows=rows, ctx_min=spread(rng, 1, most) if rng.random() < 0.7 else 0, ctx_max=most, q_heads=hq, kv_heads=hkv, head_dim=d)
    tokens = spread(rng, 1, 1500)
    cached = 0 if rng.random() < 0.3 else spread(rng, 1, min(14000, 15000000 // tokens * 32 // hq))
    return dict(op=op, tokens=tokens, cached=cached, q_heads=hq, kv_heads=hkv, head_dim=d)


def lengths(case) -> tuple[list[int], list[int]]:
    """(tokens that every sequence has, new ones), by the case alone."""
    r = random.Random("%d %d %d %s" % (case["rows"], case["ctx_min"], case["ctx_max"], case.get("new_max")))
    ctx = [r.randint(case["ctx_min"], case["ctx_max"]) for _ in range(case["rows"])]
    if case["op"] == "decode" and case["ctx_min"] == 0:
        ctx = [0 if r.random() < 0.1 else c for c in ctx]
        ctx[0] = case["ctx_max"]
    new = [spread(r, case["new_min"], case["new_max"]) for _ in range(case["rows"])] if "new_max" in case else []
    if new and case["op"] == "map" and case["new_min"] == 0:
        new = [0 if r.random() < 0.2 else n for n in new]
    return ctx, new


def up(n: int, to: int = PAGE) -> int:
    return -(-n // to)


def padded(total: int) -> int:
    """Rows of a pass of `total` tokens, as a program with graphs of fixed sizes rounds them up."""
    return up(max(total, 1), 64) * 64


def work(case) -> dict:
    op = case["op"]
    if op in ("map", "append"):
        ctx, new = lengths(case)
        total, B = sum(new), len(ctx)
        fresh = sum(up(c + n) - up(c) for c, n in zip(ctx, new))
        if op == "map":  # lengths, free pages; pages into the table, lengths and first rows, three numbers per row
            return {"bytes": 4.0 * (2 * B + 2 * fresh + 2 * B + 1 + 3 * padded(total)), "flops": 1.0 * padded(total)}
        pages = sum(up(c + n) - c // PAGE for c, n in zip(ctx, new))
        wide = 2 if case["dtype"] == "bf16" else 4
        H, D = case["kv_heads"], case["head_dim"]
        return {"bytes": 2.0 * total * H * D * (wide + 1) + 4.0 * total + 2 * 2 * pages * H, "flops": 4.0 * total * H * D}
    Hq, H, D = case["q_heads"], case["kv_heads"], case["head_dim"]
    if op == "decode":
        ctx, _ = lengths(case)
        return {"bytes": 2.0 * sum(ctx) * H * D + sum(up(c) * (2 * H + 4) for c in ctx) + 4.0 * len(ctx) * Hq * D, "flops": 4.0 * sum(ctx) * Hq * D}
    n, c = case["tokens"], case["cached"]
    return {"bytes": 2.0 * (n + c) * H * D + up(n + c) * (2 * H + 4) + 4.0 * n * Hq * D, "flops": 4.0 * Hq * D * (n * c + n * (n + 1) / 2)}


# --------------------------------------------------------------------- inputs


def rows_like(g, *shape):
    """Keys or values as a model makes them: normal numbers, some channels several times as wide as the others."""
    wide = 1 + 6 * (torch.rand(shape[-2:], device=DEV, generator=g) < 0.06)
    return torch.randn(shape, device=DEV, generator=g) * wide * (0.3 + torch.rand(*shape[:-1], 1, device=DEV, generator=g))


def pools(g, blocks: int, H: int, D: int):
    """A pool of whole pages and its scales."""
    x = rows_like(g, blocks, H, PAGE, D)
    m, e = torch.frexp(x.abs().amax((2, 3)))
    e = (e - 9 + (m > 0.875)).clamp(LOW, HIGH)
    return (x * torch.exp2(-e.float())[:, :, None, None]).to(F8), (e + 127).to(torch.uint8).view(E8)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    op = case["op"]
    if op == "prompt":
        ctx, new = [case["cached"] + case["tokens"]], []
    else:
        ctx, new = lengths(case)
    B = len(ctx)
    have = [up(c) for c in ctx]
    last = [up(c + n) for c, n in zip(ctx, new)] if new else have
    blocks = max(sum(last) + 5, 8)
    width = case.get("pages") or max(max(last), 1) + 3
    ids = torch.randperm(blocks, device=DEV, generator=g).int()
    take = torch.full((B, width), -1, dtype=torch.int64)
    at = 0
    for b, n in enumerate(have):
        take[b, :n] = torch.arange(at, at + n)
        at += n
    take = take.to(DEV)
    table = torch.where(take >= 0, ids[take.clamp(min=0)], -1).int()
    s = dict(case=case, blocks=blocks)
    if op == "map":
        s |= dict(table=table, ctx=ints(ctx), new=ints(new), supply=ids, used=ints([at]), total=padded(sum(new)))
        return s
    H, D = case["kv_heads"], case["head_dim"]
    s["k"], s["ks"] = pools(g, blocks, H, D)
    s["v"], s["vs"] = pools(g, blocks, H, D)
    if op == "append":
        table = table.cpu().tolist()
        free, slots = ids.cpu().tolist(), []
        for b in range(B):
            row = table[b][:have[b]] + free[at:at + last[b] - have[b]]
            at += last[b] - have[b]
            slots += [row[p // PAGE] * PAGE + p % PAGE for p in range(ctx[b], ctx[b] + new[b])]
        n = len(slots)
        s["slots"] = ints(slots + [-1] * (padded(n) - n))
        for x in ("nk", "nv"):
            s[x] = rows_like(g, padded(n), H, D).to(BF if case["dtype"] == "bf16" else torch.float32)
        return s
    n = case["tokens"] if op == "prompt" else B
    s["q"] = (torch.randn(n, case["q_heads"], D, device=DEV, generator=g) * 1.5).to(BF)
    for b in range(B):  # slots behind the last token
        if ctx[b] % PAGE:
            for pool in (s["k"], s["v"]):
                pool.view(torch.uint8)[table[b, have[b] - 1].long(), :, ctx[b] % PAGE:] = 0x7F
    s |= dict(scale=D ** -0.5, table=table, ctx=ints(ctx), most=max(ctx))
    return s


# ----------------------------------------------------------------- plain form


def fit(top):
    """The smallest exponent e with top <= 448 * 2^e, within the scales' range."""
    m, e = torch.frexp(top)
    return torch.where(top > 0, e - 9 + (m > 0.875), LOW).clamp(LOW, HIGH)


def power(e):
    return torch.exp2(e.float())


def exponents(scale):
    return scale.view(torch.uint8).int() - 127


def plain_map(s):
    ctx, new, table = s["ctx"].long(), s["new"].long(), s["table"]
    lens = ctx + new
    have, need = (ctx + PAGE - 1) // PAGE, (lens + PAGE - 1) // PAGE
    first = s["used"] + torch.cumsum(need - have, 0) - (need - have)
    col = torch.arange(table.shape[1], device=DEV)
    fresh = (col >= have[:, None]) & (col < need[:, None])
    page = s["supply"][(first[:, None] + col - have[:, None]).clamp(0, s["supply"].numel() - 1)]
    table.copy_(torch.where(fresh, page, table))
    start = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    row = torch.arange(s["total"], device=DEV)
    real = row < start[-1]
    seq = torch.searchsorted(start[1:], row, right=True).clamp(max=new.numel() - 1)
    pos = ctx[seq] + row - start[seq]
    slot = table[seq, (pos // PAGE).clamp(0, table.shape[1] - 1)].long() * PAGE + pos % PAGE
    return dict(table=table, lens=lens.int(), row_start=start.int(), row_seq=torch.where(real, seq, -1).int(), positions=torch.where(real, pos, 0).int(),
                slots=torch.where(real, slot, -1).int(), used=(s["used"] + (need - have).sum()).int())


def plain_append(rows, slots, pool, scale):
    blocks, H = scale.shape
    real = torch.where(slots >= 0, torch.arange(slots.numel(), device=DEV), 0)  # rows of no slot do again what the first row does
    x, blk, off = rows.float()[real], (slots[real] // PAGE).long(), (slots[real] % PAGE).long()
    x = torch.where(torch.isfinite(x), x, float("nan"))
    top = torch.zeros(blocks, H, device=DEV).index_reduce_(0, blk, x.abs().nan_to_num(0.0).amax(2), "amax")[blk]
    first = torch.full((blocks,), PAGE, device=DEV).scatter_reduce_(0, blk, off, "amin")[blk, None]
    old = exponents(scale)[blk]
    e = torch.where(first > 0, torch.maximum(old, fit(top)), fit(top))
    codes = pool.view(torch.uint8)
    kept = (pool.view(torch.uint8)[blk].view(F8).float() * power(old - e)[:, :, None, None]).to(F8).view(torch.uint8)
    codes[blk] = torch.where((torch.arange(PAGE, device=DEV) < first)[:, None, :, None], kept, codes[blk])
    codes[blk, :, off] = (x * power(-e)[:, :, None]).clamp(-TOP, TOP).to(F8).view(torch.uint8)
    scale.view(torch.uint8)[blk] = (e + 127).to(torch.uint8)
    return pool, scale


def pages_of(pool, scale, table):
    """[..., pages * 16, H, D] fp32 numbers of the pages that a table lists."""
    t = table.clamp(min=0).long()
    x = pool.view(torch.uint8)[t].view(F8).float() * power(exponents(scale)[t])[..., None, None]
    return x.transpose(-3, -2).flatten(-4, -3)


def weighted(scores, v, seen):
    """Softmax over the last axis of scores where `seen`, times v; rows that see nothing are zero."""
    scores = torch.where(seen, scores, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top > float("-inf"), top, 0.0))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, 1.0)


def plain_decode(s):
    q, table, ctx = s["q"].float(), s["table"][:, :max(up(s["most"]), 1)], s["ctx"].long()
    B, Hq, D = q.shape
    H = s["k"].shape[1]
    seen = torch.arange(table.shape[1] * PAGE, device=DEV) < ctx[:, None]
    k, v = (pages_of(s[a], s[b], table).masked_fill(~seen[:, :, None, None], 0.0) for a, b in (("k", "ks"), ("v", "vs")))
    scores = torch.matmul(q.view(B, H, Hq // H, D), k.permute(0, 2, 3, 1)) * s["scale"]
    return weighted(scores, v.permute(0, 2, 1, 3), seen[:, None, None]).reshape(B, Hq, D).to(BF)


def plain_prompt(s):
    q, n, most = s["q"].float(), s["q"].shape[0], s["most"]
    Hq, D = q.shape[1:]
    H = s["k"].shape[1]
    k, v = (pages_of(s[a], s[b], s["table"][0, :up(most)])[:most] for a, b in (("k", "ks"), ("v", "vs")))
    scores = torch.matmul(q.view(n, H, Hq // H, D).permute(1, 2, 0, 3), k.permute(1, 2, 0)[:, None]) * s["scale"]
    at = torch.arange(most, device=DEV)
    return weighted(scores, v.permute(1, 0, 2)[:, None], at <= at[most - n:, None]).permute(2, 0, 1, 3).reshape(n, Hq, D).to(BF)


# ------------------------------------------------------------------------ run


def pkg(sub: str):
    return importlib.import_module("inference-server_b200." + sub)


def own_run(s):
    ops, op = pkg("ops"), s["case"]["op"]
    if op == "map":
        m = ops.kv_slot_map(s["ctx"], s["new"], s["table"], s["supply"], s["used"], s["total"], s["blocks"])
        return dict(table=s["table"], lens=m.lens, row_start=m.row_start, row_seq=m.row_seq, positions=m.positions, slots=m.slots, used=m.supply_used)
    if op == "append":
        ops.kv8_append(s["nk"], s["nv"], s["k"], s["v"], s["ks"], s["vs"], s["slots"])
        return dict(k=s["k"], ks=s["ks"], v=s["v"], vs=s["vs"])
    cache = s["k"], s["v"], s["ks"], s["vs"]
    n, Hq, D = s["q"].shape
    H = s["k"].shape[1]
    if op == "decode":
        if "ws" not in s:  # a program keeps it for all its steps
            s["ws"] = ops.kv8_attn_workspace(n, Hq, H, D, s["table"].shape[1], s["q"].device)
        return ops.kv8_attn_decode(s["q"], *cache, s["table"], s["ctx"], s["scale"], workspace=s["ws"])
    if "ws" not in s:
        s["ws"] = ops.kv8_attn_prefill_workspace(n, s["most"] - n, Hq, H, D, s["q"].device)
    return ops.kv8_attn_prefill(s["q"], *cache, s["table"][0], s["most"] - n, s["scale"], workspace=s["ws"])


def run(s):
    if own:
        return own_run(s)
    op = s["case"]["op"]
    if op == "map":
        return plain_map(s)
    if op == "append":
        k, ks = plain_append(s["nk"], s["slots"], s["k"], s["ks"])
        v, vs = plain_append(s["nv"], s["slots"], s["v"], s["vs"])
        return dict(k=k, ks=ks, v=v, vs=vs)
    return plain_decode(s) if op == "decode" else plain_prompt(s)


# ---------------------------------------------------------------------- exact


def two_to(e):
    """Exact powers of two, which pow() does not promise."""
    return torch.tensor([2.0 ** i for i in range(-99, 100)], dtype=torch.float64, device=DEV)[e.long() + 99]


TINY = 1e-9  # log2 of a power of two may be off by less; the power's neighbours among numbers of 24 bits are 1e-7 away


def in_e4m3(x):
    """x rounded to the nearest e4m3 number, ties to even, as a 64-bit number."""
    a = x.abs()
    step = two_to(torch.floor(torch.log2(a.clamp(min=2.0 ** -6)) + TINY) - 3)
    return torch.sign(x) * (torch.round(a / step) * step).clamp(max=TOP)


def exact_append(rows, slots, pool, scale):
    pool, e = pool.double(), torch.round(torch.log2(scale.double()))
    x = rows.double()
    at = 0
    while at < len(slots) and slots[at] >= 0:
        to = at + 1
        while to < len(slots) and slots[to] == slots[to - 1] + 1 and slots[to] % PAGE:
            to += 1
        page, off = slots[at] // PAGE, slots[at] % PAGE
        new = x[at:to].transpose(0, 1)
        top = torch.ceil(torch.log2(new.abs().amax((1, 2)) / TOP) - TINY).clamp(LOW, HIGH)
        was = e[page].clone()
        if off:
            top = torch.maximum(top, was)
            pool[page, :, :off] = in_e4m3(pool[page, :, :off] * two_to(was - top)[:, None, None])
        e[page] = top
        pool[page, :, off:off + to - at] = in_e4m3(new * two_to(-top)[:, None, None])
        at = to
    return pool, two_to(e)


def exact(case, seed):
    op = case["op"]
    if op == "map":  # whole numbers
        return None
    s = prepare(case, seed)
    if op == "append":
        slots = s["slots"].cpu().tolist()
        k, ks = exact_append(s["nk"], slots, s["k"], s["ks"])
        v, vs = exact_append(s["nv"], slots, s["v"], s["vs"])
        return dict(k=k, ks=ks, v=v, vs=vs)
    q = s["q"].double()
    H, group = case["kv_heads"], case["q_heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    ctx = s["ctx"].tolist()
    for b, L in enumerate(ctx):
        page = s["table"][b, :up(L)].long()
        if not L:
            continue
        k, v = ((s[a].view(torch.uint8)[page].view(F8).double() * s[c].view(torch.uint8)[page].view(E8).double()[:, :, None, None]) for a, c in (("k", "ks"), ("v", "vs")))
        rows = slice(b, b + 1) if op == "decode" else slice(0, q.shape[0])
        for h in range(H):
            kh, vh = k[:, h].reshape(-1, q.shape[2])[:L], v[:, h].reshape(-1, q.shape[2])[:L]
            for j in range(h * group, (h + 1) * group):
                sc = q[rows, j] @ kh.T * s["scale"]
                if op == "prompt":
                    sc += torch.full_like(sc, float("-inf")).triu(case["cached"] + 1)
                out[rows, j] = torch.softmax(sc, 1) @ vh
    return out
