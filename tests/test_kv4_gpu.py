"""4-bit paged K/V cache operators against their 64-bit restatement (tests/kv4_reference.py)."""
import math
import random

import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
import moonshine_b200 as mb  # noqa: E402

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def ints(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


# ---------------------------------------------------------------- block tables
@pytest.mark.parametrize("rows,page,old,new,spare", [
    (1, 16, 0, 1, 0), (1, 16, 16, 1, 0), (1, 48, 47, 1, 3), (3, 16, 40, 0, 2), (64, 16, 194, 1, 1),
    (65, 64, 0, 1500, 0), (1023, 16, 300, 7, 0), (1025, 32, 90, 40, 5), (4100, 16, 33, 3, 0), (2, 1, 5, 9, 0),
    (5, 128, 100000, 5000, 4)])
def test_block_tables(rows, page, old, new, spare):
    rng = random.Random(rows * 1000 + page + old)
    lengths = [rng.randint(0, old) for _ in range(rows)]
    added = [rng.choice([0, new, rng.randint(0, new)]) for _ in range(rows)]
    width = max(1, max(-(-(a + b) // page) for a, b in zip(lengths, added)) + rng.randint(0, 2))
    table = [[rng.randint(0, 10 ** 6) for _ in range(width)] for _ in range(rows)]
    takes = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(lengths, added))
    free = [rng.randint(0, 2 ** 30) for _ in range(takes + spare)]
    n_slots = sum(added) + 3 * spare
    want = ref.block_tables(lengths, added, table, page, free, n_slots)
    t = ints(table)
    slots, cu, counts = mb.kv_block_tables(ints(lengths), ints(added), t, page, n_slots, free_pages=ints(free))
    assert t.tolist() == want[0]
    assert slots.tolist() == want[1]
    assert cu.tolist() == want[2] and counts.tolist() == want[3]


def test_block_tables_without_free_pages_left_and_narrow_tables():
    lengths, added = [5, 0, 31, 16, 3], [40, 20, 2, -7, 100]
    table = [[9, 9, 9], [9, 9, 9], [4, 6, 9], [2, 9, 9], [-1, 9, 9]]
    for left in range(8):
        want = ref.block_tables(lengths, added, table, 16, list(range(100, 100 + left)), 200)
        t = ints(table)
        slots, cu, counts = mb.kv_block_tables(ints(lengths), ints(added), t, 16, 200,
                                               free_pages=ints(list(range(100, 100 + left))))
        assert (t.tolist(), slots.tolist(), cu.tolist(), counts.tolist()) == want
    # fewer slots than new tokens: the first ones; pages by number; rows of a wider buffer
    want = ref.block_tables(lengths, added, table, 16, list(range(50)), 33)
    wide = torch.full((5, 8), 77, dtype=torch.int32, device="cuda")
    wide[:, 2:5] = ints(table)
    slots, cu, counts = mb.kv_block_tables(ints(lengths), ints(added), wide[:, 2:5], 16, 33, n_pages=50)
    assert (wide[:, 2:5].tolist(), slots.tolist(), cu.tolist(), counts.tolist()) == want
    assert (wide[:, :2] == 77).all() and (wide[:, 5:] == 77).all()


def test_block_tables_of_no_rows():
    slots, cu, counts = mb.kv_block_tables(ints([]), ints([]), torch.zeros(0, 4, dtype=torch.int32, device="cuda"),
                                           16, 3, n_pages=4)
    assert (slots.tolist(), cu.tolist(), counts.tolist()) == ([-1, -1, -1], [0], [0, 0])


# ---------------------------------------------------------------- store
def random_kv(tokens, heads, hd, dtype, g):
    k = (torch.randn(tokens, heads, hd, generator=g, device="cuda") * 2 + torch.randn(heads, hd, generator=g, device="cuda"))
    return k.to(dtype), torch.randn(tokens, heads, hd, generator=g, device="cuda").to(dtype)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("tokens,heads,hd,page", [(1, 1, 8, 16), (17, 3, 24, 16), (33, 8, 40, 48), (64, 8, 64, 64),
                                                  (45, 2, 72, 16), (31, 5, 96, 32), (130, 4, 128, 64)])
def test_append_and_read(kind, tokens, heads, hd, page):
    g = torch.Generator(device="cuda").manual_seed(tokens * hd)
    k, v = random_kv(tokens, heads, hd, TYPES[kind], g)
    pages = -(-tokens // page) + 2
    pool = mb.kv4_pool(pages, heads, hd, page)
    pool.fill_(0xA5)
    slots = torch.randperm(pages * page, generator=g, device="cuda")[:tokens]
    slots[torch.rand(tokens, generator=g, device="cuda") < 0.1] = -1
    if tokens > 20:
        slots[3] = pages * page  # behind the pool: left out
    mb.kv4_append(pool, k, v, slots)
    here = (slots >= 0) & (slots < pages * page)
    rk, rv = mb.kv4_read(pool, slots, hd, torch.float32)
    ck, sk, bk, wk = ref.quantize(k)
    cv, sv, bv, wv = ref.quantize(v)
    # s c + b is rounded once, to fp32
    assert torch.equal(rk, torch.where(here[:, None, None], wk, 0.0).float())
    assert torch.equal(rv, torch.where(here[:, None, None], wv, 0.0).float())
    hk, hv = mb.kv4_read(pool, slots, hd, TYPES[kind])
    assert torch.equal(hk, rk.to(TYPES[kind])) and torch.equal(hv, rv.to(TYPES[kind]))
    # the page bytes themselves; what no slot names is as it was
    bytes_before = torch.full_like(pool, 0xA5).cpu()
    got = pool.cpu()
    groups = -(-hd // 64)
    touched = {}
    for i, s in enumerate(slots.tolist()):
        if 0 <= s < pages * page:
            touched.setdefault(s // page, {})[s % page] = i
    for p in range(pages):
        for h in range(heads):
            full = torch.zeros(page, hd, dtype=torch.int64), torch.zeros(page, groups, dtype=torch.float64)
            parts = [full[0].clone(), full[1].clone(), full[1].clone(), full[0].clone(), full[1].clone(), full[1].clone()]
            mask = [torch.zeros_like(full[0]), torch.zeros_like(full[1])]
            for at, i in touched.get(p, {}).items():
                for part, src in zip(parts, (ck, sk, bk, cv, sv, bv)):
                    part[at] = src[i, h].cpu()
                mask[0][at] = 15
                mask[1][at] = math.nan  # 0x7e00
            want = ref.page_bytes(*parts)
            used = ref.page_bytes(mask[0], mask[1], mask[1], mask[0], mask[1], mask[1])
            have = bytes(got[p, h].tolist())
            old = bytes(bytes_before[p, h].tolist())
            # meta words of touched positions are wholly overwritten: mark both of their bytes
            for j in range(len(have)):
                if used[j]:
                    assert have[j] == want[j], (p, h, j)
            if not touched.get(p):
                assert have == old


def test_append_leaves_neighbours_as_they_were():
    g = torch.Generator(device="cuda").manual_seed(3)
    heads, hd, page, pages = 3, 72, 32, 4
    pool = mb.kv4_pool(pages, heads, hd, page)
    k, v = random_kv(pages * page, heads, hd, torch.float16, g)
    every = torch.arange(pages * page, device="cuda")
    mb.kv4_append(pool, k, v, every)
    before = mb.kv4_read(pool, every, hd)
    some = ints([5, 17, 63, 100], torch.int64)
    k2, v2 = random_kv(4, heads, hd, torch.float16, g)
    mb.kv4_append(pool, k2, v2, some)
    after = mb.kv4_read(pool, every, hd)
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[some] = False
    for a, b, n in zip(after, before, (k2, v2)):
        assert torch.equal(a[rest], b[rest])
        assert torch.equal(a[some], ref.quantize(n)[3].float())


@pytest.mark.parametrize("kind", list(TYPES))
def test_append_special_values(kind):
    """Constant groups, borders met exactly, huge and tiny ranges, infinities and NaNs."""
    dtype, hd = TYPES[kind], 64
    rows = [torch.zeros(hd), torch.full((hd,), -3.5), torch.arange(hd) % 16 * 1.0, torch.arange(hd) % 31 * 0.5,
            torch.linspace(-65504, 65504, hd), torch.linspace(0, 1e-7, hd), torch.linspace(1000, 1000.01, hd),
            torch.arange(hd) % 31 * 0.5 * 2.0 ** -20 - 1e-3]
    inf = torch.randn(hd)
    inf[3], inf[60] = math.inf, -math.inf
    nan = torch.randn(hd)
    nan[17] = math.nan
    x = torch.stack(rows + [inf, nan, torch.full((hd,), math.nan)]).to(dtype).cuda()[:, None, :]
    pool = mb.kv4_pool(1, 1, hd, 16)
    slots = torch.arange(x.shape[0], device="cuda")
    mb.kv4_append(pool, x, x, slots)
    k, v = mb.kv4_read(pool, slots, hd)
    want = ref.quantize(x)[3].float()
    for got in (k, v):
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


def test_append_strided_and_unaligned_inputs_and_layer_slices():
    g = torch.Generator(device="cuda").manual_seed(9)
    T, H, hd, page, layers = 37, 4, 40, 16, 3
    pools = torch.zeros(5, layers, H, page * ref.position_bytes(hd), dtype=torch.uint8, device="cuda")
    slots = torch.randperm(5 * page, generator=g, device="cuda")[:T]
    by_head = torch.randn(H, T + 1, hd, generator=g, device="cuda").transpose(0, 1)[1:]
    shifted = torch.randn(T * H * hd + 1, generator=g, device="cuda")[1:].view(T, H, hd)
    mb.kv4_append(pools[:, 1], by_head, shifted, slots)
    k, v = mb.kv4_read(pools[:, 1], slots, hd)
    assert torch.equal(k, ref.quantize(by_head)[3].float()) and torch.equal(v, ref.quantize(shifted)[3].float())
    assert not pools[:, 0].any() and not pools[:, 2].any()


# ---------------------------------------------------------------- attention
def build(lens, heads, hd, page, g, extra=2, fill=0xFF):
    """A pool of random pages (every byte `fill` outside the rows' positions: NaN scales), its
    table, and the rows' stored keys and values in fp64."""
    blocks = [-(-n // page) for n in lens]
    pages = sum(blocks) + extra
    pool = mb.kv4_pool(pages, heads, hd, page)
    pool.fill_(fill)
    order = torch.randperm(pages, generator=g, device="cuda").tolist()
    width = max(blocks + [1]) + 1
    table, keys, values, used = [], [], [], 0
    for n, nb in zip(lens, blocks):
        mine = order[used:used + nb]
        used += nb
        table.append(mine + [-1] * (width - nb))
        k, v = random_kv(n, heads, hd, torch.float32, g)
        at = torch.arange(n, device="cuda")
        if n:
            slots = ints(mine, torch.int64)[at // page] * page + at % page
            mb.kv4_append(pool, k, v, slots)
            k, v = (x.double() for x in mb.kv4_read(pool, slots, hd))
        keys.append(k)
        values.append(v)
    return pool, ints(table).view(len(lens), width), keys, values


def tolerance(out, mass, peak, dtype, hd):
    """Half a step of the type for the result (below the smallest normal n all numbers are
    multiples of n eps, so never less than n eps / 2: 2^-25 in fp16), and the roundings before
    it.  A score sums hd
    products and the bias terms in fp32 (each addition 2^-23, tensor cores cut instead of
    rounding) over terms of `mass` in all -- s c and b are each up to twice a key's range, so
    4 mass -- plus fp32's q planes (2^-22); a wrong score shifts a probability, and so the
    result, by twice that times the largest value.  Probabilities in one fp16 plane are off by
    2^-12, in two by 2^-22, of terms s c up to twice the largest value; exp and the fp32 sums
    by 2^-20.  bf16 may take keys and values rounded to fp16, 2^-12 of each."""
    info = torch.finfo(dtype)
    half = info.eps / 2
    score = 4 * mass * ((hd + 16) * 2.0 ** -23 + 2.0 ** -22)
    plane = 2.0 ** -12 if dtype == torch.bfloat16 else 2.0 ** -22
    if dtype == torch.bfloat16:
        score, plane = score + mass * 2.0 ** -12, plane + 2.0 ** -13
    return out.abs().clamp(min=info.smallest_normal) * half + (peak * (2 * score + 2 * plane + 2.0 ** -20)).unsqueeze(-1) + 1e-30


def check(got, want, mass, peak, dtype, hd):
    assert not torch.isnan(got).any()
    off = (got.double() - want).abs() - tolerance(want, mass, peak, dtype, hd)
    assert off.max().item() <= 0, off.max().item()


CASES = [  # rows' lengths, rows' queries, heads, kv_heads, hd, page
    ([1], [1], 1, 1, 8, 16), ([0], [1], 2, 1, 40, 16), ([16], [1], 8, 8, 40, 16), ([17], [1], 8, 8, 64, 16),
    ([375, 1, 0, 750, 64], [1] * 5, 10, 10, 64, 64), ([129, 1500], [1, 1], 8, 8, 40, 32),
    ([5, 40, 1000], [1, 1, 1], 12, 2, 96, 16), ([300, 2, 77], [1, 1, 1], 28, 4, 128, 48),
    ([8191], [1], 16, 4, 128, 64), ([4000, 60], [1, 1], 12, 1, 128, 64),
    ([9, 200, 33], [5, 3, 1], 8, 2, 64, 16), ([3, 64, 0], [5, 4, 2], 6, 6, 40, 16),
    ([100, 257], [17, 33], 14, 2, 128, 32), ([500, 130, 64], [129, 130, 64], 4, 2, 64, 64),
    ([700], [300], 5, 1, 80, 16), ([1200, 90], [64, 90], 16, 4, 24, 16), ([65, 66, 67], [2, 0, 2], 3, 3, 72, 16),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,qs,heads,kv_heads,hd,page", CASES)
def test_attention(lens, qs, heads, kv_heads, hd, page, causal, kind):
    g = torch.Generator(device="cuda").manual_seed(sum(lens) + hd)
    pool, table, keys, values = build(lens, kv_heads, hd, page, g)
    cu = [0]
    for n in qs:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1] + 2, heads, hd, generator=g, device="cuda").to(TYPES[kind])
    out = torch.full_like(q, 7.0)
    one = max(qs) == 1 and min(qs) == 1
    mb.kv4_attention(q, pool, table, ints(lens), cu_q=ints(cu), max_q=max(qs), causal=causal, out=out)
    want, mass, peak = ref.attention(q, keys, values, lens, cu, causal, hd ** -0.5)
    check(out[:cu[-1]], want[:cu[-1]], mass[:cu[-1]], peak[:cu[-1]], TYPES[kind], hd)
    assert (out[cu[-1]:] == 7.0).all()  # tokens of no row
    if one:
        again = mb.kv4_attention(q[:-2], pool, table, ints(lens), causal=causal)
        assert torch.equal(again, out[:-2])  # the same bits with and without cu_q


@pytest.mark.parametrize("kind", ["fp32", "bf16"])
def test_attention_long_context_split(kind):
    """Few rows with long contexts beside short ones: the axis is split and joined."""
    g = torch.Generator(device="cuda").manual_seed(4)
    lens, heads, kv_heads, hd, page = [70001, 3, 0, 4100], 8, 2, 64, 64
    pool, table, keys, values = build(lens, kv_heads, hd, page, g)
    q = torch.randn(4, heads, hd, generator=g, device="cuda").to(TYPES[kind])
    out = mb.kv4_attention(q, pool, table, ints(lens))
    want, mass, peak = ref.attention(q, keys, values, lens, [0, 1, 2, 3, 4], True, hd ** -0.5)
    check(out, want, mass, peak, TYPES[kind], hd)
    assert torch.equal(out, mb.kv4_attention(q, pool, table, ints(lens)))  # the same bits every time


def test_attention_peaked_and_flat_scores():
    """One position far above the rest, and all alike; a scale of the caller's; negative scale."""
    g = torch.Generator(device="cuda").manual_seed(6)
    lens, hd = [900], 64
    pool, table, keys, values = build(lens, 1, hd, 16, g)
    for scale, factor in ((hd ** -0.5, 12.0), (1e-6, 1.0), (0.5, 3.0), (-0.125, 1.0)):
        q = (keys[0][450:451, :, :] * factor).to(torch.float32).contiguous()
        for kind in TYPES.values():
            x = q.to(kind)
            out = mb.kv4_attention(x, pool, table, ints(lens), scale=scale)
            want, mass, peak = ref.attention(x, keys, values, lens, [0, 1], True, scale)
            check(out, want, mass, peak, kind, hd)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 1.0, 300.0])
def test_attention_value_and_query_sizes(size):
    """Values and queries far from 1: fp16 planes keep their relative precision."""
    g = torch.Generator(device="cuda").manual_seed(8)
    hd, n = 64, 333
    k, v = random_kv(n, 2, hd, torch.float32, g)
    pool = mb.kv4_pool(-(-n // 16), 2, hd, 16)
    slots = torch.arange(n, device="cuda")
    mb.kv4_append(pool, k, v * size, slots)
    ks, vs = (x.double() for x in mb.kv4_read(pool, slots, hd))
    table = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda")[None]
    q = torch.randn(1, 4, hd, generator=g, device="cuda") / size
    for kind in (torch.float32, torch.bfloat16):
        out = mb.kv4_attention(q.to(kind), pool, table, ints([n]), scale=size * hd ** -0.5)
        want, mass, peak = ref.attention(q.to(kind), [ks], [vs], [n], [0, 1], True, size * hd ** -0.5)
        check(out, want, mass, peak, kind, hd)


def test_attention_missing_pages_are_not_seen():
    g = torch.Generator(device="cuda").manual_seed(11)
    lens, hd, page = [100, 64, 40], 40, 16
    pool, table, keys, values = build(lens, 2, hd, page, g)
    table[0, 2], table[1, :], table[2, 0] = -1, -5, pool.shape[0]
    present = [torch.ones(n, dtype=torch.bool, device="cuda") for n in lens]
    present[0][32:48] = False
    present[1][:] = False
    present[2][:16] = False
    q = torch.randn(3, 4, hd, generator=g, device="cuda")
    out = mb.kv4_attention(q, pool, table, ints(lens))
    want, mass, peak = ref.attention(q, keys, values, lens, [0, 1, 2, 3], True, hd ** -0.5, present)
    check(out, want, mass, peak, torch.float32, hd)
    assert not out[1].any()
    # lengths past the table's width end with it
    more = mb.kv4_attention(q[:1], pool, table[:1, :7], ints([10 ** 6]), causal=False)
    want, mass, peak = ref.attention(q[:1], keys[:1], values[:1], [100], [0, 1], False, hd ** -0.5, present[:1])
    pool2, t2 = pool, table[:1, :6]
    cut = mb.kv4_attention(q[:1], pool2, t2, ints([10 ** 6]), causal=False)
    want96, mass, peak = ref.attention(q[:1], [keys[0][:96]], [values[0][:96]], [96], [0, 1], False, hd ** -0.5,
                                       [present[0][:96]])
    check(cut, want96, mass, peak, torch.float32, hd)
    assert torch.isnan(more).any()  # the seventh page is only part filled: its other positions are NaN


def test_attention_nan_reaches_only_what_sees_it():
    g = torch.Generator(device="cuda").manual_seed(12)
    hd, n = 64, 50
    k, v = random_kv(n, 2, hd, torch.float32, g)
    v[30, 1, 5] = math.nan
    pool = mb.kv4_pool(4, 2, hd, 16)
    mb.kv4_append(pool, k, v, torch.arange(n, device="cuda"))
    table = ints([[0, 1, 2, 3]])
    q = torch.randn(40, 2, hd, generator=g, device="cuda")
    out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, 40]), max_q=40)
    assert not torch.isnan(out[:, 0]).any()
    sees = torch.arange(40, device="cuda") + n - 40 >= 30
    assert torch.equal(torch.isnan(out[:, 1]).all(-1), sees) and torch.equal(torch.isnan(out[:, 1]).any(-1), sees)


def test_attention_strides_and_layer_slices():
    g = torch.Generator(device="cuda").manual_seed(13)
    lens, hd, page, layers = [90, 33], 64, 16, 3
    pool, table, keys, values = build(lens, 2, hd, page, g)
    pools = torch.full((pool.shape[0], layers, 2, pool.shape[2]), 0xFF, dtype=torch.uint8, device="cuda")
    pools[:, 2] = pool
    wide = torch.full((2, 20), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + table.shape[1]] = table
    big = torch.randn(4, 2, 2 * hd + 1, generator=g, device="cuda")
    q = big.transpose(0, 1)[:, :, 1:hd + 1]  # [2 tokens, 4 heads, hd], unaligned
    room = torch.zeros(2, 4, hd + 3, device="cuda")
    mb.kv4_attention(q, pools[:, 2], wide[:, 3:3 + table.shape[1]], ints(lens), out=room[:, :, 1:hd + 1])
    want, mass, peak = ref.attention(q, keys, values, lens, [0, 1, 2], True, hd ** -0.5)
    check(room[:, :, 1:hd + 1], want, mass, peak, torch.float32, hd)
    assert not room[:, :, 0].any() and not room[:, :, hd + 1:].any()


def test_page_offsets_past_32_bits():
    """Pages further than 4 GiB from the pool's base (a pool that is a slice of a large buffer)."""
    g = torch.Generator(device="cuda").manual_seed(14)
    hd, page, pages, n = 40, 16, 5, 70
    each = page * ref.position_bytes(hd)
    gap = (1 << 30) + (1 << 20)
    buffer = torch.empty(pages * gap, dtype=torch.uint8, device="cuda")
    pool = buffer.as_strided((pages, 1, each), (gap, each, 1))
    k, v = random_kv(n, 1, hd, torch.float32, g)
    table = ints([[4, 2, 0, 3, 1]])
    at = torch.arange(n, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    mb.kv4_append(pool, k, v, slots)
    rk, rv = mb.kv4_read(pool, slots, hd)
    assert torch.equal(rk, ref.quantize(k)[3].float()) and torch.equal(rv, ref.quantize(v)[3].float())
    q = torch.randn(1, 3, hd, generator=g, device="cuda")
    out = mb.kv4_attention(q, pool, table, ints([n]))
    want, mass, peak = ref.attention(q, [rk], [rv], [n], [0, 1], True, hd ** -0.5)
    check(out, want, mass, peak, torch.float32, hd)


# ---------------------------------------------------------------- together
def serving_state(rows, heads, kv_heads, hd, page, width, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pages = rows * width
    return {"pool": mb.kv4_pool(pages, kv_heads, hd, page), "table": torch.full((rows, width), -1, dtype=torch.int32, device="cuda"),
            "free": torch.randperm(pages, generator=g, device="cuda").to(torch.int32),
            "lengths": torch.zeros(rows, dtype=torch.int32, device="cuda"), "g": g}


def test_prompt_then_steps_in_a_replayed_graph():
    """Pages for prompts, then decode steps (tables, append, attention) captured once and
    replayed while lengths and free pages move on in device memory; against fp64 on the values
    that the cache stands for, and the same steps run eagerly give the same bits."""
    rows, heads, kv_heads, hd, page, width = 5, 8, 4, 64, 16, 6
    prompt = [16, 1, 40, 7, 31]
    outs = []
    for captured in (False, True):
        s = serving_state(rows, heads, kv_heads, hd, page, width, 21)
        g = torch.Generator(device="cuda").manual_seed(22)
        T = sum(prompt)
        slots, cu, counts = mb.kv_block_tables(s["lengths"], ints(prompt), s["table"], page, T, free_pages=s["free"])
        k, v = random_kv(T, kv_heads, hd, torch.float32, g)
        mb.kv4_append(s["pool"], k, v, slots)
        q = torch.randn(T, heads, hd, generator=g, device="cuda")
        lens = s["lengths"] + ints(prompt)
        first = mb.kv4_attention(q, s["pool"], s["table"], lens, cu_q=cu, max_q=max(prompt))
        ks, vs = mb.kv4_read(s["pool"], slots, hd)
        edges = cu.tolist()
        keys = [ks[edges[b]:edges[b + 1]] for b in range(rows)]
        values = [vs[edges[b]:edges[b + 1]] for b in range(rows)]
        want, mass, peak = ref.attention(q, keys, values, prompt, edges, True, hd ** -0.5)
        check(first, want, mass, peak, torch.float32, hd)
        s["lengths"].copy_(lens)
        s["free"] = torch.roll(s["free"], -counts[0].item())
        one = torch.ones(rows, dtype=torch.int32, device="cuda")
        kn, vn = torch.empty(rows, kv_heads, hd, device="cuda"), torch.empty(rows, kv_heads, hd, device="cuda")
        qn = torch.empty(rows, heads, hd, device="cuda")
        out = torch.empty_like(qn)
        new_slots = torch.empty(rows, dtype=torch.int64, device="cuda")
        taken = torch.zeros(1, dtype=torch.int64, device="cuda")

        def step():
            sl, _, cn = mb.kv_block_tables(s["lengths"], one, s["table"], page, rows, free_pages=s["free"])
            mb.kv4_append(s["pool"], kn, vn, sl)
            s["lengths"].add_(one)
            mb.kv4_attention(qn, s["pool"], s["table"], s["lengths"], out=out)
            new_slots.copy_(sl)
            # the pages taken leave the free list
            at = (torch.arange(s["free"].shape[0], device="cuda") + cn[0]) % s["free"].shape[0]
            s["free"].copy_(s["free"][at])

        graph = None
        for t in range(20):
            a, b = random_kv(rows, kv_heads, hd, torch.float32, g)
            kn.copy_(a)
            vn.copy_(b)
            qn.copy_(torch.randn(rows, heads, hd, generator=g, device="cuda"))
            if captured and t == 2:
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step()
            if graph is None:
                step()
            else:
                graph.replay()
            ks, vs = mb.kv4_read(s["pool"], new_slots, hd)
            keys = [torch.cat([keys[i], ks[i:i + 1]]) for i in range(rows)]
            values = [torch.cat([values[i], vs[i:i + 1]]) for i in range(rows)]
            n = [p + t + 1 for p in prompt]
            assert s["lengths"].tolist() == n
            want, mass, peak = ref.attention(qn, keys, values, n, list(range(rows + 1)), True, hd ** -0.5)
            check(out, want, mass, peak, torch.float32, hd)
            outs.append(out.clone())
    for a, b in zip(outs[:20], outs[20:]):
        assert torch.equal(a, b)


def test_two_streams_at_once():
    g = torch.Generator(device="cuda").manual_seed(30)
    lens, hd = [30000, 200], 64
    pool, table, keys, values = build(lens, 2, hd, 64, g)
    q = torch.randn(2, 8, hd, generator=g, device="cuda")
    want = mb.kv4_attention(q, pool, table, ints(lens))
    n = ints(lens)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append(mb.kv4_attention(q, pool, table, n))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want) for x in got)


# ---------------------------------------------------------------- many query rows per K/V head
# (heads, kv_heads, hd): one and two groups of 64, whole and partial
MANY = [(8, 2, 40), (4, 4, 64), (5, 1, 80), (14, 2, 128)]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("heads,kv_heads,hd", MANY)
def test_many_queries_missing_pages_and_queries_before_the_first_position(heads, kv_heads, hd, kind):
    g = torch.Generator(device="cuda").manual_seed(hd + heads)
    lens, qs, page = [333, 64, 20, 0, 150], [70, 64, 75, 40, 33], 16
    pool, table, keys, values = build(lens, kv_heads, hd, page, g)
    table[0, 3], table[0, 20], table[1, :], table[4, 0:2] = -1, pool.shape[0], -7, pool.shape[0] + 5
    present = [torch.ones(n, dtype=torch.bool, device="cuda") for n in lens]
    present[0][48:64] = False
    present[0][320:] = False
    present[1][:] = False
    present[4][:32] = False
    cu = [0]
    for n in qs:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], heads, hd, generator=g, device="cuda").to(TYPES[kind])
    for causal in (True, False):
        out = mb.kv4_attention(q, pool, table, ints(lens), cu_q=ints(cu), max_q=max(qs), causal=causal)
        want, mass, peak = ref.attention(q, keys, values, lens, cu, causal, hd ** -0.5, present)
        check(out, want, mass, peak, TYPES[kind], hd)
        assert not out[cu[1]:cu[2]].any() and not out[cu[3]:cu[4]].any()
        if causal:
            assert not out[cu[2]:cu[2] + 55].any()  # 75 queries of 20 positions


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,hd,context", [(8, 2, 64, 30011), (16, 4, 128, 9000), (9, 1, 24, 5000)])
def test_many_queries_split_context(heads, kv_heads, hd, context, kind):
    g = torch.Generator(device="cuda").manual_seed(context)
    lens, qs = [context, 40], [64, 17]
    pool, table, keys, values = build(lens, kv_heads, hd, 64, g)
    q = torch.randn(81, heads, hd, generator=g, device="cuda").to(TYPES[kind])
    args = dict(cu_q=ints([0, 64, 81]), max_q=64)
    out = mb.kv4_attention(q, pool, table, ints(lens), **args)
    want, mass, peak = ref.attention(q, keys, values, lens, [0, 64, 81], True, hd ** -0.5)
    check(out, want, mass, peak, TYPES[kind], hd)
    assert torch.equal(out, mb.kv4_attention(q, pool, table, ints(lens), **args))


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("hd", [64, 96])
def test_many_queries_nan_reaches_only_what_sees_it(hd, kind):
    g = torch.Generator(device="cuda").manual_seed(17)
    n, qn = 200, 150
    k, v = random_kv(n, 2, hd, torch.float32, g)
    v[100, 1, 5], k[180, 0, 3] = math.nan, math.nan
    pool = mb.kv4_pool(13, 2, hd, 16)
    mb.kv4_append(pool, k, v, torch.arange(n, device="cuda"))
    table = torch.arange(13, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(qn, 2, hd, generator=g, device="cuda").to(TYPES[kind])
    q[7, 0, 2] = math.inf
    out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, qn]), max_q=qn)
    at = torch.arange(qn, device="cuda")
    last = at + n - qn
    # a NaN value makes its group of 64 dims NaN, a NaN key or query the whole row
    want = torch.zeros(qn, 2, hd, dtype=torch.bool, device="cuda")
    want[:, 1, :64] = (last >= 100)[:, None]
    want[:, 0] = ((last >= 180) | (at == 7))[:, None]
    assert torch.equal(torch.isnan(out), want)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 300.0])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_many_queries_value_and_query_sizes(size, kind):
    g = torch.Generator(device="cuda").manual_seed(18)
    hd, n, qn = 64, 333, 60
    k, v = random_kv(n, 2, hd, torch.float32, g)
    pool = mb.kv4_pool(-(-n // 16), 2, hd, 16)
    slots = torch.arange(n, device="cuda")
    mb.kv4_append(pool, k, v * size, slots)
    ks, vs = (x.double() for x in mb.kv4_read(pool, slots, hd))
    table = torch.arange(-(-n // 16), dtype=torch.int32, device="cuda")[None]
    small = max(size, 1e-3)  # fp16 queries of 1e-3 .. 300 and back
    q = (torch.randn(qn, 4, hd, generator=g, device="cuda") / small).to(TYPES[kind])
    for sign in (1, -1):
        out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, qn]), max_q=qn, scale=sign * small * hd ** -0.5)
        want, mass, peak = ref.attention(q, [ks], [vs], [n], [0, qn], True, sign * small * hd ** -0.5)
        check(out, want, mass, peak, TYPES[kind], hd)


@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_many_queries_strides_and_max_q(kind):
    """Unaligned strided q and out; queries past max_q and tokens of no row stay as they were."""
    g = torch.Generator(device="cuda").manual_seed(19)
    lens, cu, hd, heads = [90, 300], [1, 41, 121], 64, 4
    pool, table, keys, values = build(lens, 2, hd, 16, g)
    big = torch.randn(heads, 125, 2 * hd + 1, generator=g, device="cuda").to(TYPES[kind])
    q = big.transpose(0, 1)[:, :, 1:hd + 1]
    for max_q in (80, 50):
        room = torch.full((heads, 125, hd + 3), 5.0, device="cuda", dtype=TYPES[kind])
        out = room.transpose(0, 1)[:, :, 1:hd + 1]
        mb.kv4_attention(q, pool, table, ints(lens), cu_q=ints(cu), max_q=max_q, out=out)
        want, mass, peak = ref.attention(q, keys, values, lens, cu, True, hd ** -0.5)
        done = torch.zeros(125, dtype=torch.bool, device="cuda")
        done[1:41] = True
        done[41:41 + max_q] = True
        check(out[done], want[done], mass[done], peak[done], TYPES[kind], hd)
        assert (out[~done] == 5.0).all() and (room[:, :, 0] == 5.0).all() and (room[:, :, hd + 1:] == 5.0).all()


def test_first_call_is_a_captured_one():
    """Nothing of the library has run on the device before the capture."""
    code = """
import torch, moonshine_b200 as mb
n, hd = 9000, 64
pool = mb.kv4_pool(n // 16 + 1, 2, hd, 16)
k = torch.randn(n, 2, hd, device="cuda"); slots = torch.empty(n, dtype=torch.int64, device="cuda")
table = torch.full((1, n // 16 + 1), -1, dtype=torch.int32, device="cuda")
zero = torch.zeros(1, dtype=torch.int32, device="cuda"); many = torch.full((1,), n, dtype=torch.int32, device="cuda")
cu = torch.tensor([0, 40], dtype=torch.int32, device="cuda")
one, q = torch.randn(1, 8, hd, device="cuda"), torch.randn(40, 8, hd, device="cuda").bfloat16()
def run():
    s, _, _ = mb.kv_block_tables(zero, many, table, 16, n, n_pages=pool.shape[0])
    mb.kv4_append(pool, k, k, s)
    return mb.kv4_attention(one, pool, table, many), mb.kv4_attention(q, pool, table, many, cu_q=cu, max_q=40), *mb.kv4_read(pool, s, hd)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = run()
graph.replay()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, run()))
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(mb.__file__)))
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True,
                       timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]


def test_two_graphs_of_split_contexts():
    """Two captured calls, each with its own workspace, replayed on two streams at once."""
    g = torch.Generator(device="cuda").manual_seed(31)
    lens, hd = [20000, 100], 64
    pool, table, keys, values = build(lens, 2, hd, 64, g)
    n, graphs, outs, want = ints(lens), [], [], []
    for i in range(2):
        q = torch.randn(2, 8, hd, generator=g, device="cuda")
        want.append(mb.kv4_attention(q, pool, table, n))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(mb.kv4_attention(q, pool, table, n))
        graphs.append((graph, q))
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for st, (graph, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_many_query_rows_of_a_long_prompt():
    """More groups of query rows than a grid's second dimension holds."""
    g = torch.Generator(device="cuda").manual_seed(32)
    n, heads, hd = 140000, 8, 8
    pool, table, keys, values = build([20], 8, hd, 16, g)
    q = torch.randn(n, heads, hd, generator=g, device="cuda")
    out = mb.kv4_attention(q, pool, table, ints([20]), cu_q=ints([0, n]), max_q=n, causal=False)
    some = torch.cat([torch.arange(50, device="cuda"), torch.arange(n - 50, n, device="cuda")])
    want, mass, peak = ref.attention(q[some], keys, values, [20], [0, 100], False, hd ** -0.5)
    check(out[some], want, mass, peak, torch.float32, hd)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(6, 2, 64, 48), (8, 1, 128, 112), (3, 1, 8, 16), (16, 4, 72, 80)])
def test_many_queries_page_sizes(heads, kv_heads, hd, page, kind):
    """Pages that end inside a stage of 64 positions, and one that holds several."""
    g = torch.Generator(device="cuda").manual_seed(page + hd)
    lens, qs = [517, 48, 113], [65, 48, 80]
    pool, table, keys, values = build(lens, kv_heads, hd, page, g)
    cu = [0, 65, 113, 193]
    q = torch.randn(193, heads, hd, generator=g, device="cuda").to(TYPES[kind])
    out = mb.kv4_attention(q, pool, table, ints(lens), cu_q=ints(cu), max_q=80)
    want, mass, peak = ref.attention(q, keys, values, lens, cu, True, hd ** -0.5)
    check(out, want, mass, peak, TYPES[kind], hd)


@pytest.mark.parametrize("queries", [1, 100])
@pytest.mark.parametrize("kind", ["bf16", "fp32"])
def test_largest_values(kind, queries):
    """Ranges up to +-65504, whose highest code can stand for more than fp16's largest: the scale,
    up to 8736, is rounded by at most 4, 15 times that is 60, and the bias by at most 16, so for
    at most 65580.  Where values are held to 65504, that is off by 76 / 65580 < 2^-9.7."""
    g = torch.Generator(device="cuda").manual_seed(41)
    hd, n = 64, 100
    k, v = random_kv(n, 1, hd, torch.float32, g)
    k, v = k * 2e4, v * 4e4
    v[::3, :, 0], v[::3, :, 1] = 65504, -65504
    k[5, 0, 7], k[5, 0, 8] = 65504, -65504
    pool = mb.kv4_pool(7, 1, hd, 16)
    slots = torch.arange(n, device="cuda")
    mb.kv4_append(pool, k, v, slots)
    ks, vs = (x.double() for x in mb.kv4_read(pool, slots, hd))
    assert 65504 < vs.max() <= 65580
    table = torch.arange(7, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(queries, 1, hd, generator=g, device="cuda").to(TYPES[kind])
    scale = 1e-4 * hd ** -0.5
    out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, queries]), max_q=queries, scale=scale)
    want, mass, peak = ref.attention(q, [ks], [vs], [n], [0, queries], True, scale)
    # where K and V are rounded to fp16 the tolerance has 2^-12 of keys and 2 (2^-12 + 2^-13) of
    # values; 2^-9.7 more is 2^2.3 < 5 times and 2^1.3 / 1.5 < 1.7 times that
    held = kind == "bf16" and queries > 32
    check(out, want, mass * (6 if held else 1), peak * (2.7 if held else 1), TYPES[kind], hd)
