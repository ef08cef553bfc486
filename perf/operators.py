"""Plain forms, cases and exact results of the 4-bit K/V cache operators:

- tables: block tables and slot maps of a paged cache, built on the GPU from request lengths;
- store:  new keys and values into the 4-bit pages, and the stored values read back;
- attend: attention of one or more query tokens per request over the 4-bit pages.

The cache.  A pool is uint8 [pages, kv_heads, page bytes].  A page holds page_size positions
(a multiple of 16) of one request, per K/V head as page_size / 16 tiles of 16 positions.
Every K or V vector of head_dim values is cut into groups of 64 (the last one shorter); a
group is stored as 4-bit codes c with an fp16 scale s and an fp16 bias b and stands for
s c + b, with

    b = fp16(min x),   s = fp16(fp32((max x - min x) / 15)),
    c = how many of the 15 borders b + (k + 1/2) s (k = 0 .. 14) are <= x

(x clamped to +-65504 first; s = 0: c = 0; a group with a NaN reads as NaN).  A tile of nw =
head_dim / 8 code words per vector (dim 8 w + i in bits 4 i .. 4 i + 3 of word w) holds, in
32-bit words,
    K: word w of position r at 64 j + 2 (min(4, nw - 4 j) (r % 8) + w % 4) + r / 8, j = w / 4,
    V: word w of position r at 16 nw + 16 w + 4 ((r % 8) / 2) + 2 (r / 8) + r % 2,
    (s, b) of group n at 32 nw + 32 n + 4 (r % 8) + 2 (V: 1, K: 0) + r / 8.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_HERE = os.path.dirname(os.path.abspath(__file__))
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _kv():
    """The framework's package (only where `own` is true)."""
    path = os.path.join(os.path.dirname(_HERE), "moonshine-mlx_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import moonshine_b200
    return moonshine_b200


# ---------------------------------------------------------------- cases
def listed():
    return [
        # block tables: one decode step of 64 utterances (a token each, pages of 16 positions,
        # up to 195 tokens: 30 s at 6.5 tokens per second) -- launch latency
        {"name": "tables_step", "op": "tables", "rows": 64, "page": 16, "width": 13, "old": 194, "new": 1},
        # 256 utterances of 2 to 30 s get pages for all their memory frames (up to 1500)
        {"name": "tables_frames", "op": "tables", "rows": 256, "page": 64, "width": 24, "old": 0, "new": 1500},
        # a large server: 4096 requests with up to 32K cached tokens append prompt chunks
        {"name": "tables_server", "op": "tables", "rows": 4096, "page": 16, "width": 2112, "old": 32768, "new": 1024},
        # store: one decode step of 64 utterances (8 heads of 64)
        {"name": "store_step", "op": "store", "tokens": 64, "kv_heads": 8, "dim": 64, "page": 16, "type": "bf16"},
        # the cross K/V of one layer for 64 utterances of 250 to 750 frames (8 heads of 40)
        {"name": "store_frames", "op": "store", "tokens": 32001, "kv_heads": 8, "dim": 40, "page": 64, "type": "fp32"},
        # a server's prompts, heads of 128
        {"name": "store_prompts", "op": "store", "tokens": 262144, "kv_heads": 8, "dim": 128, "page": 64,
         "type": "bf16"},
        # attend: cross attention of one utterance of 30 s, exact types -- latency
        {"name": "attend_one", "op": "attend", "rows": 1, "q": 1, "heads": 8, "kv_heads": 8, "dim": 40, "page": 16,
         "context": 1500, "causal": False, "type": "fp32"},
        # cross attention of a decode step of 256 utterances of up to 30 s (10 heads of 64)
        {"name": "attend_frames", "op": "attend", "rows": 256, "q": 1, "heads": 10, "kv_heads": 10, "dim": 64,
         "page": 64, "context": 1500, "causal": False, "type": "bf16"},
        # a decode step of few requests with long contexts, 4 query heads per K/V head
        {"name": "attend_long", "op": "attend", "rows": 4, "q": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "page": 64, "context": 131072, "causal": True, "type": "bf16"},
        # drafted tokens checked in one pass, ragged, odd head count
        {"name": "attend_drafts", "op": "attend", "rows": 33, "q": 5, "heads": 28, "kv_heads": 4, "dim": 128,
         "page": 16, "context": 8000, "causal": True, "type": "fp16"},
        # chunks of prompts over a cache that holds what came before
        {"name": "attend_prompts", "op": "attend", "rows": 8, "q": 512, "heads": 16, "kv_heads": 4, "dim": 64,
         "page": 64, "context": 4096, "causal": True, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tables", "store", "attend", "attend"])
    if op == "tables":
        rows = _log(rng, 1, 4096)
        page = rng.choice([16, 32, 64, 128])
        old, new = rng.choice([0, _log(rng, 1, 32768)]), rng.choice([1, _log(rng, 2, 1024)])
        return {"op": op, "rows": rows, "page": page, "width": -(-(old + new) // page) + rng.randint(0, 3), "old": old,
                "new": new}
    kv_heads, per, dim = rng.choice([(8, 1, 40), (8, 1, 64), (10, 1, 64), (4, 4, 64), (8, 4, 128), (4, 7, 128),
                                     (2, 6, 96), (1, 5, 80), (3, 1, 24), (1, 12, 128)])
    page, kind = rng.choice([16, 32, 64]), rng.choice(["bf16", "fp16", "fp32"])
    if op == "store":
        most = 262144 * 8 * 128 // (kv_heads * dim) // (2 if kind == "fp32" else 1)
        return {"op": op, "tokens": _log(rng, 1, min(most, 400000)), "kv_heads": kv_heads, "dim": dim, "page": page,
                "type": kind}
    q = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 512)])
    rows = _log(rng, 1, 256 if q == 1 else 64 if q <= 8 else 8)
    room = min(131072, 4 * 131072 * 8 * 144 // (rows * kv_heads * (dim + 8 * -(-dim // 64))))  # bytes of attend_long
    if q > 1:  # and the products of attend_prompts
        room = min(room, 8 * 512 * 16 * 4096 * 64 // (rows * q * kv_heads * per * dim))
    context = max(1, _log(rng, 1, max(2, room)) if q == 1 else max(q, _log(rng, 1, max(2, room))))
    return {"op": op, "rows": rows, "q": q, "heads": kv_heads * per, "kv_heads": kv_heads, "dim": dim, "page": page,
            "context": context, "causal": rng.choice([True, True, False]), "type": kind}


def _ragged(case):
    """Context and query lengths of an attend case (by the case alone): one request of the full
    length, the others from an eighth of it up, the odd one empty in larger batches."""
    rng = random.Random("%(rows)d %(q)d %(context)d %(dim)d" % case)
    lens = [rng.randint(max(1, case["context"] // 8), case["context"]) for _ in range(case["rows"])]
    lens[rng.randrange(case["rows"])] = case["context"]
    qs = [case["q"] if case["q"] <= 2 else rng.randint(1 + case["q"] // 2, case["q"]) for _ in lens]
    if case["rows"] > 20:
        lens[0 if lens[0] != case["context"] else 1] = 0
    return lens, qs


def _nbytes(dim):  # bytes of one position's K and V for one head
    return dim + 8 * -(-dim // 64)


def work(case):
    if case["op"] == "tables":
        cap = case["rows"] * case["new"]
        return {"bytes": case["rows"] * (8 + 4 + 4 * case["width"]) + 8 * cap, "flops": 0}
    size = _TYPES[case["type"]].itemsize
    if case["op"] == "store":  # values in, cache out, cache in, values out
        n = case["tokens"] * case["kv_heads"]
        return {"bytes": n * (4 * case["dim"] * size + 2 * _nbytes(case["dim"])) + 16 * case["tokens"], "flops": 0}
    lens, qs = _ragged(case)
    pairs = sum(sum(max(0, n - q + i + 1) for i in range(q)) if case["causal"] else n * q for n, q in zip(lens, qs))
    return {"bytes": sum(lens) * case["kv_heads"] * _nbytes(case["dim"]) + 2 * sum(qs) * case["heads"] * case["dim"] * size
            + 4 * sum(-(-n // case["page"]) + 2 for n in lens),
            "flops": 4 * pairs * case["heads"] * case["dim"]}


# ---------------------------------------------------------------- the cache, plainly
def _places(dim, device):
    """Word indexes inside a tile: K and V [16, nw], (scale, bias) [2, 16, groups]."""
    nw = dim // 8
    r, w = torch.arange(16, device=device)[:, None], torch.arange(nw, device=device)[None, :]
    j = w // 4
    k = 64 * j + 2 * (torch.clamp(nw - 4 * j, max=4) * (r % 8) + w % 4) + r // 8
    v = 16 * nw + 16 * w + 4 * ((r % 8) // 2) + 2 * (r // 8) + r % 2
    n = torch.arange(-(-dim // 64), device=device)
    m = 32 * nw + 32 * n[None, None, :] + 4 * (r % 8)[None] + 2 * torch.arange(2, device=device)[:, None, None] + (r // 8)[None]
    return k, v, m


def _spread(x, dim):
    """[..., groups] to [..., dim]: each group's value for each of its dims."""
    return x.repeat_interleave(64, dim=-1)[..., :dim]


def _encode(x):
    """Codes, scales and biases of x [..., dim]."""
    dim = x.shape[-1]
    x = torch.clamp(x.float(), -65504.0, 65504.0)
    n = -(-dim // 64)
    grouped = torch.nn.functional.pad(x, (0, 64 * n - dim)).unflatten(-1, (n, 64))
    real = (torch.arange(64 * n, device=x.device) < dim).view(n, 64)
    lo = torch.where(real, grouped, torch.inf).amin(-1)
    hi = torch.where(real, grouped, -torch.inf).amax(-1)
    # a scale that rounds the other way moves codes next to a border: the quotient in 64 bits
    s, b = ((hi.double() - lo.double()) / 15.0).float().half(), lo.half()
    s64, b64 = _spread(s, dim).double(), _spread(b, dim).double()
    # next to a border 32 bits do not say on which side a value lies: borders in 64
    c = torch.where(s64 > 0, torch.floor((x.double() - b64) / s64 + 0.5), 0.0).clamp(0, 15)
    c = torch.where((c > 0) & (x.double() < b64 + (c - 0.5) * s64), c - 1, c)
    c = torch.where((c < 15) & (s64 > 0) & (x.double() >= b64 + (c + 0.5) * s64), c + 1, c)
    return c.to(torch.int32), s, b


def _words(codes):
    """[..., dim] codes to [..., dim / 8] int32 words."""
    shift = 4 * torch.arange(8, device=codes.device)
    return (codes.unflatten(-1, (-1, 8)).long() << shift).sum(-1).to(torch.int32)


def _meta(s, b):
    """fp16 scale and bias as one int32 word."""
    return torch.stack([s, b], -1).contiguous().view(torch.int32).squeeze(-1)


def _decode(tiles, where, meta, dim):
    """Tile words [..., words] to the values [..., 16, dim] that they stand for."""
    shift = 4 * torch.arange(8, device=tiles.device, dtype=torch.int32)
    c = ((tiles[..., where][..., None] >> shift) & 15).flatten(-2).float()
    sb = tiles[..., meta].contiguous().view(torch.float16).unflatten(-1, (-1, 2)).float()
    return c * _spread(sb[..., 0], dim) + _spread(sb[..., 1], dim)


def _tiles(pool, dim):
    """The pool's 32-bit words [pages, heads, tiles of a page, words of a tile]."""
    return pool.view(torch.int32).unflatten(-1, (-1, 4 * _nbytes(dim)))


def _store(pool, k, v, slots):
    dim, page = k.shape[-1], pool.shape[-1] // _nbytes(k.shape[-1])
    tiles = _tiles(pool, dim)
    here = slots >= 0
    slot = slots[here]
    p, t, r = slot // page, slot % page // 16, slot % 16
    wk, wv, wm = _places(dim, pool.device)
    heads = torch.arange(k.shape[1], device=pool.device)[None, :, None]
    p, t = p[:, None, None], t[:, None, None]
    c, s, b = _encode(k[here])
    tiles[p, heads, t, wk[r][:, None, :]] = _words(c)
    tiles[p, heads, t, wm[0][r][:, None, :]] = _meta(s, b)
    c, s, b = _encode(v[here])
    tiles[p, heads, t, wv[r][:, None, :]] = _words(c)
    tiles[p, heads, t, wm[1][r][:, None, :]] = _meta(s, b)


def _fetch(pool, slots, dim, dtype):
    page = pool.shape[-1] // _nbytes(dim)
    here = (slots >= 0)[:, None, None]
    slot = torch.clamp(slots, min=0)
    tiles = _tiles(pool, dim)[slot // page, :, slot % page // 16]
    wk, wv, wm = _places(dim, pool.device)
    r = (slot % 16)[:, None, None, None]
    pick = lambda x: torch.where(here, x.gather(2, r.expand(-1, x.shape[1], 1, dim)).squeeze(2), 0.0).to(dtype)  # noqa: E731
    return pick(_decode(tiles, wk, wm[0], dim)), pick(_decode(tiles, wv, wm[1], dim))


def _attend(q, pool, table, lens, cu_q, max_q, causal):
    heads, dim = q.shape[1:]
    pages, kv_heads = pool.shape[:2]
    page, rows, per = pool.shape[-1] // _nbytes(dim), table.shape[0], heads // pool.shape[1]
    tiles = _tiles(pool, dim)[torch.clamp(table, 0, pages - 1).long()]  # [rows, width, kv_heads, tiles, words]
    wk, wv, wm = _places(dim, pool.device)
    flat = lambda x: x.permute(0, 2, 1, 3, 4, 5).reshape(rows, kv_heads, -1, dim)  # noqa: E731
    keys = flat(_decode(tiles, wk, wm[0], dim))
    i = torch.arange(max_q, device=q.device)
    n = (cu_q[1:] - cu_q[:-1])[:, None]
    at = torch.clamp(cu_q[:-1, None] + i, max=q.shape[0] - 1).long()
    x = q[at].float().view(rows, max_q, kv_heads, per, dim).permute(0, 2, 3, 1, 4).reshape(rows, kv_heads, per * max_q, dim)
    score = (x @ keys.transpose(-1, -2)).view(rows, kv_heads, per, max_q, -1) * dim ** -0.5
    del keys
    position = torch.arange(score.shape[-1], device=q.device)
    seen = (position < lens[:, None, None]) & (table >= 0).repeat_interleave(page, 1)[:, None, :]
    if causal:
        seen = seen & (position <= (lens[:, None] - n + i)[:, :, None])
    score = torch.where(seen[:, None, None], score, -torch.inf)
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - torch.where(top == -torch.inf, 0.0, top))
    del score
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p.flatten(2, 3) @ flat(torch.nan_to_num(_decode(tiles, wv, wm[1], dim)))
    out = out.view(rows, kv_heads, per, max_q, dim).permute(0, 3, 1, 2, 4).reshape(rows, max_q, heads, dim)
    return out[(i < n)].to(q.dtype)


def _tables(lengths, new, table, page, cap, free):
    width = table.shape[1]
    have, need = -(-lengths // page), -(-(lengths + new) // page)
    take = need - have
    start = torch.cumsum(take, 0) - take
    cu = torch.cat([torch.zeros(1, dtype=torch.int32, device=table.device), torch.cumsum(new, 0).to(torch.int32)])
    column = torch.arange(width, device=table.device)[None, :]
    index = (start[:, None] + column - have[:, None]).long()
    fresh = torch.where((index >= 0) & (index < len(free)), free[torch.clamp(index, 0, len(free) - 1)], -1)
    table.copy_(torch.where(column < have[:, None], table, torch.where(column < need[:, None], fresh, -1)))
    token = torch.arange(cap, device=table.device)
    row = torch.clamp(torch.searchsorted(cu[1:], token, right=True), max=len(new) - 1)
    position = lengths[row] + token - cu[row]
    block = torch.clamp(position // page, max=width - 1)
    where = table[row, block].long()
    good = (token < cu[-1]) & (position // page < width) & (where >= 0)
    slots = torch.where(good, where * page + position % page, -1)
    return slots, cu, torch.stack([take.sum(), new.sum()]).to(torch.int32)


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    rng = random.Random(seed)
    page = case["page"]
    if case["op"] == "tables":
        rows, width = case["rows"], case["width"]
        old = [rng.randint(case["old"] // 4, case["old"]) for _ in range(rows)]
        new = [case["new"] if case["new"] == 1 else rng.randint(0, case["new"]) for _ in range(rows)]
        have = [-(-n // page) for n in old]
        need = sum(-(-(a + b) // page) - c for a, b, c in zip(old, new, have))
        ids = torch.randperm(sum(have) + need + 8, generator=g, device=dev).to(torch.int32)
        table = torch.full((rows, width), -1, dtype=torch.int32, device=dev)
        mine = torch.arange(width, device=dev)[None, :] < torch.tensor(have, device=dev)[:, None]
        table[mine] = ids[: sum(have)]
        return {"op": "tables", "lengths": torch.tensor(old, dtype=torch.int32, device=dev),
                "new": torch.tensor(new, dtype=torch.int32, device=dev), "table": table, "page": page,
                "cap": rows * case["new"], "free": ids[sum(have):].clone()}
    dtype, dim, kv_heads = _TYPES[case["type"]], case["dim"], case["kv_heads"]
    # keys with a mean and a spread per channel, as projections have them; values without
    mean = torch.randn(kv_heads, dim, generator=g, device=dev)
    spread = torch.exp(0.5 * torch.randn(kv_heads, dim, generator=g, device=dev))
    if case["op"] == "store":
        n = case["tokens"]
        pages = -(-n // page) + 5
        # whole pages in a random order, the last one part full, one token in 50 without a slot
        order = torch.randperm(pages, generator=g, device=dev)
        at = torch.arange(n, device=dev)
        slots = order[at // page] * page + at % page
        slots[torch.rand(n, generator=g, device=dev) < 0.02] = -1
        k = torch.randn(n, kv_heads, dim, generator=g, device=dev).mul_(spread).add_(mean).to(dtype)
        v = torch.randn(n, kv_heads, dim, generator=g, device=dev).to(dtype)
        return {"op": "store", "k": k, "v": v, "slots": slots,
                "pool": torch.zeros(pages, kv_heads, page * _nbytes(dim), dtype=torch.uint8, device=dev)}
    lens, qs = _ragged(case)
    blocks = [-(-n // page) for n in lens]
    pages = sum(blocks) + 3
    pool = torch.zeros(pages, kv_heads, page * _nbytes(dim), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 25) // (page * kv_heads * dim))
    for p in range(0, pages, step):
        n = min(step, pages - p) * page
        slots = p * page + torch.arange(n, device=dev)
        k = torch.randn(n, kv_heads, dim, generator=g, device=dev).mul_(spread).add_(mean).to(dtype)
        v = torch.randn(n, kv_heads, dim, generator=g, device=dev).to(dtype)
        _store(pool, k, v, slots)
    width = -(-case["context"] // page)
    table = torch.full((case["rows"], width), -1, dtype=torch.int32, device=dev)
    mine = torch.arange(width, device=dev)[None, :] < torch.tensor(blocks, device=dev)[:, None]
    table[mine] = torch.randperm(pages, generator=g, device=dev)[: sum(blocks)].to(torch.int32)
    q = torch.randn(sum(qs), case["heads"], dim, generator=g, device=dev).to(dtype)
    return {"op": "attend", "q": q, "pool": pool, "table": table, "causal": case["causal"], "max_q": max(qs),
            "lens": torch.tensor(lens, dtype=torch.int32, device=dev),
            "cu_q": torch.tensor([0] + list(np.cumsum(qs)), dtype=torch.int32, device=dev)}


def run(state):
    s = state
    if own:
        kv = _kv()
        if s["op"] == "tables":
            slots, cu, counts = kv.kv_block_tables(s["lengths"], s["new"], s["table"], s["page"], s["cap"],
                                                   free_pages=s["free"])
            return {"table": s["table"], "slots": slots, "cu_new": cu, "counts": counts}
        if s["op"] == "store":
            kv.kv4_append(s["pool"], s["k"], s["v"], s["slots"])
            k, v = kv.kv4_read(s["pool"], s["slots"], s["k"].shape[-1], s["k"].dtype)
            return {"k": k, "v": v}
        return kv.kv4_attention(s["q"], s["pool"], s["table"], s["lens"], cu_q=s["cu_q"], max_q=s["max_q"],
                                causal=s["causal"])
    if s["op"] == "tables":
        slots, cu, counts = _tables(s["lengths"], s["new"], s["table"], s["page"], s["cap"], s["free"])
        return {"table": s["table"], "slots": slots, "cu_new": cu, "counts": counts}
    if s["op"] == "store":
        _store(s["pool"], s["k"], s["v"], s["slots"])
        k, v = _fetch(s["pool"], s["slots"], s["k"].shape[-1], s["k"].dtype)
        return {"k": k, "v": v}
    return _attend(s["q"], s["pool"], s["table"], s["lens"], s["cu_q"], s["max_q"], s["causal"])


# ---------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "tables":
        lengths, new = s["lengths"].tolist(), s["new"].tolist()
        table, free, page = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy(), s["page"]
        slots, cu, used = np.full(s["cap"], -1, dtype=np.int64), [0], 0
        for b, (n, m) in enumerate(zip(lengths, new)):
            first, last = (n + page - 1) // page, (n + m + page - 1) // page
            table[b, first:] = -1
            got = free[used:used + last - first]
            table[b, first:first + len(got)] = got
            used += last - first
            at = np.arange(n, n + m)
            where = table[b, at // page].astype(np.int64)
            slots[cu[-1]:cu[-1] + m] = np.where(where < 0, -1, where * page + at % page)
            cu.append(cu[-1] + m)
        return {"table": table, "slots": slots, "cu_new": np.array(cu, np.int32),
                "counts": np.array([used, cu[-1]], np.int32)}
    dim = case["dim"]
    if case["op"] == "store":
        def stored(x):
            y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
            for a in range(0, dim, 64):
                z = x[..., a:a + 64].double().clamp(-65504, 65504)
                low, high = z.min(-1, keepdim=True)[0], z.max(-1, keepdim=True)[0]
                scale, bias = ((high - low) / 15).float().half().double(), low.half().double()
                code = torch.zeros_like(z)
                for k in range(15):
                    code += ((z >= bias + (k + 0.5) * scale) & (scale > 0)).double()
                y[..., a:a + 64] = bias + scale * code
            y[s["slots"] < 0] = 0
            return y
        return {"k": stored(s["k"]), "v": stored(s["v"])}
    lens, qs = _ragged(case)
    page, heads, kv_heads = case["page"], case["heads"], case["kv_heads"]
    q, pool, table = s["q"].double(), s["pool"].flatten(), s["table"].long()
    nw, stride = dim // 8, page * _nbytes(dim)
    d = torch.arange(dim, device="cuda")
    w, group = d // 8, d // 64
    outs, first = [], 0
    for b in range(case["rows"]):
        n, m = lens[b], qs[b]
        x = q[first:first + m]
        first += m
        y = torch.zeros(m, heads, dim, dtype=torch.float64, device="cuda")
        outs.append(y)
        if n == 0:
            continue
        at = torch.arange(n, device="cuda")
        r = (at % 16)[:, None]
        past = torch.arange(m, device="cuda")[:, None] + (n - m if case["causal"] else n)
        for h in range(kv_heads):
            base = ((table[b, at // page] * kv_heads + h) * stride + at % page // 16 * 16 * _nbytes(dim))[:, None]
            got = []
            for kind in range(2):
                word = (64 * (w // 4) + 2 * ((nw - w // 4 * 4).clamp(max=4) * (r % 8) + w % 4) + r // 8
                        if kind == 0 else 16 * nw + 16 * w + 4 * (r % 8 // 2) + 2 * (r // 8) + r % 2)
                code = (pool[base + 4 * word + d % 8 // 2].long() >> 4 * (d % 2)) & 15
                meta = base + 4 * (32 * nw + 32 * torch.arange(-(-dim // 64), device="cuda") + 4 * (r % 8) + 2 * kind + r // 8)
                scale, bias = (torch.stack([pool[meta + o], pool[meta + o + 1]], -1).view(torch.float16).squeeze(-1).double()
                               for o in (0, 2))
                got.append(code * scale[:, group] + bias[:, group])
            for e in range(h * heads // kv_heads, (h + 1) * heads // kv_heads):
                z = x[:, e] @ got[0].T / math.sqrt(dim)
                z[at[None, :] > past] = -math.inf
                z = torch.exp(z - z.max(-1, keepdim=True)[0].clamp(min=-1e300))
                y[:, e] = z @ got[1] / z.sum(-1, keepdim=True).clamp(min=1e-300)
    return torch.cat(outs)
