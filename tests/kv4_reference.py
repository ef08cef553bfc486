"""Plain 64-bit restatement of the 4-bit K/V cache operators (include/moonshine_b200.h) for their
tests: quantization, page layout, block tables and attention, written from the definitions."""
import math

import torch

GROUP = 64


def position_bytes(hd):
    return hd + 8 * -(-hd // GROUP)


def quantize(x):
    """(codes int64, scale fp64, bias fp64 [..., groups], values fp64) of x [..., hd]."""
    hd = x.shape[-1]
    x = x.double()
    codes = torch.zeros(x.shape, dtype=torch.int64, device=x.device)
    values = torch.zeros_like(x)
    scales, biases = [], []
    for a in range(0, hd, GROUP):
        z = x[..., a:a + GROUP]
        bad = torch.isnan(z).any(-1, keepdim=True)
        z = torch.nan_to_num(z, nan=0.0, posinf=math.inf, neginf=-math.inf).clamp(-65504, 65504)
        low, high = z.min(-1, keepdim=True)[0], z.max(-1, keepdim=True)[0]
        s = ((high - low) / 15).float().half().double()
        b = low.half().double()
        c = torch.zeros_like(z)
        for k in range(15):
            c += ((z >= b + (k + 0.5) * s) & (s > 0)).double()
        codes[..., a:a + GROUP] = c.long()
        values[..., a:a + GROUP] = torch.where(bad, math.nan, s * c + b)
        scales.append(s)
        biases.append(b)
    return codes, torch.cat(scales, -1), torch.cat(biases, -1), values


def code_byte(hd, w, r, value):
    """Byte offset of code word w of position r inside its tile."""
    nw = hd // 8
    if value:
        return 4 * (16 * nw + 16 * w + 4 * (r % 8 // 2) + 2 * (r // 8) + r % 2)
    j = w // 4
    return 4 * (64 * j + 2 * (min(4, nw - 4 * j) * (r % 8) + w % 4) + r // 8)


def meta_byte(hd, n, r, value):
    return 4 * (32 * (hd // 8) + 32 * n + 4 * (r % 8) + 2 * value + r // 8)


def page_bytes(codes_k, s_k, b_k, codes_v, s_v, b_v):
    """The bytes of one page of one head from [page_size, hd] codes and [page_size, groups] scales."""
    P, hd = codes_k.shape
    each = position_bytes(hd)
    out = bytearray(P * each)
    for p in range(P):
        base, r = p // 16 * 16 * each, p % 16
        for value, (c, s, b) in enumerate(((codes_k, s_k, b_k), (codes_v, s_v, b_v))):
            for w in range(hd // 8):
                at = base + code_byte(hd, w, r, value)
                for i in range(8):
                    out[at + i // 2] |= int(c[p, 8 * w + i]) << (4 * (i % 2))
            for n in range(s.shape[-1]):
                at = base + meta_byte(hd, n, r, value)
                out[at:at + 4] = torch.stack([s[p, n], b[p, n]]).half().numpy().tobytes()
    return bytes(out)


def block_tables(lengths, new, table, page, free, n_slots):
    """Lists in, (table, slots, cu, counts) out."""
    table = [list(row) for row in table]
    slots, cu, used = [], [0], 0
    for b, (n, m) in enumerate(zip(lengths, new)):
        n, m = max(n, 0), max(m, 0)
        width = len(table[b])
        have, need = -(-n // page), -(-(n + m) // page)
        for k in range(have, width):
            i = used + k - have
            table[b][k] = (free[i] if i < len(free) else -1) if k < need else -1
        used += need - have
        for p in range(n, n + m):
            pg = table[b][p // page] if p // page < width else -1
            slots.append(pg * page + p % page if pg >= 0 else -1)
        cu.append(cu[-1] + m)
    slots = (slots + [-1] * n_slots)[:n_slots]
    return table, slots, cu, [used, cu[-1]]


def attention(q, keys, values, lens, cu, causal, scale, present=None):
    """fp64 attention; q [tokens, H, hd], keys / values [rows] of [len, KVH, hd], present[b]
    bool [len] (positions whose page exists).  Also the largest sum of |terms| of a score and
    the largest |value| of what each query sees, for tolerances: [tokens, H] each."""
    H, hd = q.shape[1:]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mass = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    peak = torch.zeros(q.shape[:2], dtype=torch.float64, device=q.device)
    for b in range(len(lens)):
        q0, q1 = cu[b], cu[b + 1]
        n = q1 - q0
        if n <= 0:
            continue
        k, v = keys[b].double(), values[b].double()
        L, KVH = k.shape[:2]
        per = H // KVH
        x = q[q0:q1].double()
        pos = torch.arange(L, device=q.device)
        last = torch.arange(n, device=q.device) + (lens[b] - n if causal else lens[b])
        seen = (pos[None, :] <= last[:, None]) & (pos[None, :] < lens[b])
        if present is not None:
            seen = seen & present[b][None, :]
        kk, vv = k.repeat_interleave(per, 1), v.repeat_interleave(per, 1)
        s = torch.einsum("nhd,lhd->hnl", x, kk) * scale
        s = torch.where(seen[None], s, -math.inf)
        top = s.amax(-1, keepdim=True) if L else torch.full((H, n, 1), -math.inf, device=q.device)
        p = torch.where(seen[None], torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top)), 0.0)
        total = p.sum(-1, keepdim=True)
        vz = torch.where((seen.any(0))[:, None, None], vv, torch.zeros_like(vv))
        out[q0:q1] = torch.einsum("hnl,lhd->nhd", p / torch.where(total == 0, torch.ones_like(total), total), vz)
        if L:
            kz = torch.where((seen.any(0))[:, None, None], kk, torch.zeros_like(kk))
            mass[q0:q1] = torch.einsum("nhd,hd->nh", x.abs(), kz.abs().amax(0)) * abs(scale)
            peak[q0:q1] = vz.abs().amax(0).amax(-1)[None]
    return out, mass, peak
