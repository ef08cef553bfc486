"""4-bit paged K/V cache operators at inputs where they can go wrong: rows that end inside a warp,
values at the end of fp16's range, NaNs beside what nobody sees, queries of unlike sizes."""
import math

import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
import moonshine_b200 as mb  # noqa: E402
from test_kv4_gpu import TYPES, build, check, ints, random_kv, tolerance  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("queries", [65, 75, 97, 127])
@pytest.mark.parametrize("hd,context", [(72, 200), (128, 130), (96, 6000)])
def test_rows_that_end_inside_a_warp(hd, context, queries, kind):
    """Two groups of dims, the last warp of rows part filled; whole contexts and split ones."""
    g = torch.Generator(device="cuda").manual_seed(hd + queries)
    pool, table, keys, values = build([context], 1, hd, 16, g)
    q = torch.randn(queries, 1, hd, generator=g, device="cuda").to(TYPES[kind])
    out = mb.kv4_attention(q, pool, table, ints([context]), cu_q=ints([0, queries]), max_q=queries)
    want, mass, peak = ref.attention(q, keys, values, [context], [0, queries], True, hd ** -0.5)
    check(out, want, mass, peak, TYPES[kind], hd)


def test_a_wait_that_runs_out_is_reported(tmp_path):
    """The decoder step's form, built with waits that give up at once (kv4_give_up.cu): the status
    word says so, for ms_generate_batch to throw, and no result is a number."""
    import os
    import shutil
    import subprocess
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    here = os.path.dirname(os.path.abspath(__file__))
    kernels = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(mb.__file__))), "csrc", "kernels")
    exe = str(tmp_path / "give_up")
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O2", "-I", kernels, "-o", exe,
                    os.path.join(here, "kv4_give_up.cu")], check=True, timeout=300)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.split() == ["5", "0"], (r.returncode, r.stdout)


# ---------------------------------------------------------------- the end of fp16's range
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("queries", [1, 70])
def test_largest_code_past_fp16(queries, kind, which):
    """A group from 34108.25 to 65504: s = 2094, b = 34112, and its code 15 stands for 65522, fp16's
    infinity.  Where bf16 takes keys and values as fp16 it is held to 65504, off by 18 / 65522 <
    2^-11.8: of keys beside the 2^-12 that the tolerance has (2.2 times that), of values beside
    2 (2^-12 + 2^-13) (1.4 times that).  Queries that do not see the position are as without it."""
    g = torch.Generator(device="cuda").manual_seed(51)
    hd, n = 64, 100
    k, v = random_kv(n, 1, hd, torch.float32, g)
    k, v = k * (1e3 if which == "k" else 1), v * (1e3 if which == "v" else 1)
    (k if which == "k" else v)[80, 0] = torch.linspace(34108.25, 65504, hd, device="cuda")
    pool = mb.kv4_pool(7, 1, hd, 16)
    slots = torch.arange(n, device="cuda")
    mb.kv4_append(pool, k, v, slots)
    ks, vs = (x.double() for x in mb.kv4_read(pool, slots, hd))
    assert (ks if which == "k" else vs)[80].max() == 34112 + 15 * 2094
    table = torch.arange(7, dtype=torch.int32, device="cuda")[None]
    q = torch.randn(queries, 1, hd, generator=g, device="cuda").to(TYPES[kind])
    scale = hd ** -0.5 * (1e-4 if which == "k" else 1)
    out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, queries]), max_q=queries, scale=scale)
    want, mass, peak = ref.attention(q, [ks], [vs], [n], [0, queries], True, scale)
    if kind == "fp16":  # results past fp16's largest are infinite
        want = want.to(torch.float16).double()
        assert torch.equal(torch.isinf(out), torch.isinf(want))
        out, want = torch.where(torch.isinf(out), 0, out), torch.where(torch.isinf(want), 0, want)
    held = kind == "bf16" and queries > 32
    check(out, want, mass * (2.2 if held else 1), peak * (1.4 if held else 1), TYPES[kind], hd)


def test_groups_that_reach_past_the_largest_value():
    """fp32 groups near +-65504 with values beyond: clamped before they are coded."""
    g = torch.Generator(device="cuda").manual_seed(50)
    hd, n = 64, 400
    lo = 65504 - 2.0 ** (torch.rand(n, 1, 1, generator=g, device="cuda") * 16 - 4)
    x = lo + (66000 - lo) * torch.rand(n, 1, hd, generator=g, device="cuda")
    x[:, :, 0] = lo[:, :, 0]
    x[::4, :, 5] = 1e6
    x[1::4, :, 5] = math.inf
    x[2::8] = -x[2::8]
    x[0, 0, :], x[0, 0, 1:3] = 65400, torch.tensor([65300.0, 1e6])
    x[1, 0, :], x[1, 0, 1:3] = 65500, torch.tensor([65490.0, 70000])
    slots = torch.randperm(n, generator=g, device="cuda")
    for order in (torch.arange(n, device="cuda"), slots):  # whole tiles, and token by token
        pool = mb.kv4_pool(n // 16, 1, hd, 16)
        mb.kv4_append(pool, x, -x, order)
        k, v = mb.kv4_read(pool, order, hd)
        assert torch.equal(k, ref.quantize(x)[3].float()) and torch.equal(v, ref.quantize(-x)[3].float())


# ---------------------------------------------------------------- NaN
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("lens,queries,per", [(3, 5, 1), (3, 5, 3), (20, 75, 1), (1, 130, 2)])
def test_a_query_that_is_nan_and_sees_nothing(lens, queries, per, kind):
    """Zeros, whatever the query holds; one that sees something is NaN, the others as without it."""
    g = torch.Generator(device="cuda").manual_seed(queries)
    hd, blind = 64, queries - lens
    pool, table, keys, values = build([lens], 2, hd, 16, g)
    q = torch.randn(queries, 2 * per, hd, generator=g, device="cuda").to(TYPES[kind])
    clean = mb.kv4_attention(q, pool, table, ints([lens]), cu_q=ints([0, queries]), max_q=queries)
    q[0, 0, 3], q[blind - 1, 1, 2] = math.nan, math.inf
    q[-1, 0, 7] = -math.inf
    out = mb.kv4_attention(q, pool, table, ints([lens]), cu_q=ints([0, queries]), max_q=queries)
    assert not out[:blind].any() and torch.isnan(out[-1, 0]).all()
    out[-1, 0] = clean[-1, 0]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("queries", [1, 6, 100])
@pytest.mark.parametrize("at", [40, 99])
@pytest.mark.parametrize("gap", [False, True])
def test_a_nan_value_reaches_all_that_see_it(gap, at, queries, kind):
    """By visibility, not by the size of its probability: every other position's underflows here.
    In a whole tile and in the last, part-filled one; beside a missing page and not."""
    g = torch.Generator(device="cuda").manual_seed(at)
    hd, n = 96, 100
    k, v = random_kv(n, 1, hd, torch.float32, g)
    k[5] = 3 * torch.sign(torch.randn(1, hd, generator=g, device="cuda"))
    v[at, 0, 70] = math.nan
    pool = mb.kv4_pool(7, 1, hd, 16)
    slots = torch.arange(n, device="cuda")
    mb.kv4_append(pool, k, v, slots)
    table = torch.arange(7, dtype=torch.int32, device="cuda")[None]
    if gap:
        table[0, 4] = -1
    q = (k[5:6].expand(queries, 1, hd) * 40).to(TYPES[kind])
    ks = mb.kv4_read(pool, slots, hd)[0].double()
    scores = (ks[:, 0] @ q[0, 0].double()) * hd ** -0.5
    rest = torch.cat([scores[:5], scores[6:]])
    assert scores[5] - rest.max() > 300  # exp(-300) is 0 in fp32
    out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, queries]), max_q=queries, causal=False)
    assert torch.isnan(out[:, :, 64:]).all() and not torch.isnan(out[:, :, :64]).any()
    # nobody sees it: as if it were not there
    one = mb.kv4_attention(q, pool, table, ints([at]), cu_q=ints([0, queries]), max_q=queries, causal=False)
    assert not torch.isnan(one).any()


# ---------------------------------------------------------------- queries of unlike sizes
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("queries", [1, 4, 16, 100])
@pytest.mark.parametrize("hd", [64, 128])
def test_one_large_query_channel(hd, queries, kind):
    """One channel of q 1000 times the others, its keys the same at all positions (the group's
    minimum, -4, so code 0 and exactly b): it moves no probability, the small channels decide.
    Two positions, so the result is the mean of two values under a difference of scores.

    A score is exact but for fp32 sums: of a group the codes' sum (4 products of 16 dims on the
    tensor cores, each cut by 2^-23 of its largest term), and 3 operations of 2^-24 that join it
    with the bias, 11 in units of 2^-24 of the terms, and one more that adds the second group; terms
    are below 15 s and 2 |b| times |q| each.  bf16 with many queries takes keys rounded by 2^-12
    (those of the large channel are exact).  Two scores' errors move the result by at most a
    quarter of the values' difference each, so by |score error| times the largest value."""
    g = torch.Generator(device="cuda").manual_seed(hd + queries)
    n, heads = 2, 3
    k = (torch.randn(n, 1, hd, generator=g, device="cuda") * 1.5).clamp(-3.9, 3.9)
    k[:, :, 0] = -4.0
    k[:, :, 64:65] = -4.0
    v = torch.randn(n, 1, hd, generator=g, device="cuda")
    pool = mb.kv4_pool(1, 1, hd, 16)
    slots = torch.arange(n, device="cuda")
    mb.kv4_append(pool, k, v, slots)
    ks, vs = (x.double() for x in mb.kv4_read(pool, slots, hd))
    assert (ks[:, 0, 0] == -4).all()
    q = torch.randn(queries, heads, hd, generator=g, device="cuda")
    q[:, :, 0] = 1000.0
    q = q.to(TYPES[kind])
    table = ints([[0]])
    out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, queries]), max_q=queries, causal=False)
    want, _, peak = ref.attention(q, [ks], [vs], [n], [0, queries], False, hd ** -0.5)
    size, groups = q.double().abs(), -(-hd // 64)
    terms = (size.sum(-1) * (8 + 2 * 4)) * hd ** -0.5  # 15 s is at most 8
    score = terms * (11 + groups) * 2.0 ** -24
    if kind == "bf16" and queries * heads > 32:
        score = score + size[:, :, 1:].sum(-1) * 4 * 2.0 ** -12 * hd ** -0.5
    plane = 2.0 ** -12 + 2.0 ** -13 if kind == "bf16" else 2.0 ** -22
    half = torch.finfo(TYPES[kind]).eps / 2
    tol = want.abs() * half + (peak * (score + 2 * plane + 2.0 ** -20)).unsqueeze(-1)
    off = (out.double() - want).abs() - tol
    assert off.max().item() <= 0, off.max().item()


# ---------------------------------------------------------------- the end of fp32's range
@pytest.mark.parametrize("kind", ["fp32", "bf16"])
@pytest.mark.parametrize("queries", [1, 6, 100])
@pytest.mark.parametrize("sign", [1.0, -1.0])
def test_scores_at_the_end_of_fp32(sign, queries, kind):
    """Queries of 1e35, whose scores fit: the position with the largest one alone, its value but for the
    roundings of one probability (2^-12 + 2^-13 in bf16, 2^-22 in fp32).  Queries of 3e38, whose scores do
    not: NaN, as a sum of infinities is, and not the zeros of a query that sees nothing."""
    g = torch.Generator(device="cuda").manual_seed(60)
    hd, n = 64, 40
    k = 1 + torch.rand(n, 1, hd, generator=g, device="cuda")
    v = torch.randn(n, 1, hd, generator=g, device="cuda")
    pool = mb.kv4_pool(3, 1, hd, 16)
    slots = torch.arange(n, device="cuda")
    mb.kv4_append(pool, k, v, slots)
    ks, vs = (x.double() for x in mb.kv4_read(pool, slots, hd))
    table = ints([[0, 1, 2]])
    for size, fits in ((1e35, True), (3e38, False)):
        q = torch.full((queries, 1, hd), sign * size, device="cuda").to(TYPES[kind])
        out = mb.kv4_attention(q, pool, table, ints([n]), cu_q=ints([0, queries]), max_q=queries, causal=False)
        if fits:
            want = vs[(ks[:, 0].sum(-1) * sign).argmax()].expand(queries, 1, hd)
            plane = 2.0 ** -12 + 2.0 ** -13 if kind == "bf16" else 2.0 ** -22
            tol = want.abs() * torch.finfo(TYPES[kind]).eps / 2 + vs.abs().max() * (2 * plane + 2.0 ** -20)
            assert ((out.double() - want).abs() <= tol).all()
        else:
            assert torch.isnan(out).all()


# ---------------------------------------------------------------- the batched decoder step's form
@pytest.fixture(scope="module")
def step_attention(tmp_path_factory):
    import ctypes as C
    import os
    import subprocess
    so = str(tmp_path_factory.mktemp("kv4_step") / "kv4_step.so")
    here, package = os.path.dirname(os.path.abspath(__file__)), os.path.dirname(os.path.abspath(mb.__file__))
    mb._L()
    subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-I/usr/local/cuda/include",
                    "-I" + os.path.join(os.path.dirname(package), "csrc", "kernels"), os.path.join(here, "kv4_step.cpp"),
                    os.path.join(package, "libmoonshine_b200.so"), "-Wl,-rpath," + package, "-o", so], check=True)
    f, P, I = C.CDLL(so).step_attention, C.c_void_p, C.c_int
    f.restype, f.argtypes = C.c_int64, [P, I, I, I, I, P, P, I, I, P, I, P, C.c_float, C.c_int64, P, P, P]
    return f


@pytest.mark.parametrize("split", [False, True])
@pytest.mark.parametrize("lens,kv_heads,per,hd", [([40, 0, 7], 8, 1, 40), ([375, 64], 10, 1, 64), ([100, 33, 1], 2, 3, 40),
                                                  ([129, 750, 20], 2, 5, 64), ([300], 1, 8, 56), ([9000, 80], 2, 8, 64)])
def test_decoder_step(lens, kv_heads, per, hd, split, step_attention):
    """fp32 queries, one channel of each 300 times the others; the result in bf16, or as the sum of two
    bf16 planes, which keep 2^-17 of it."""
    g = torch.Generator(device="cuda").manual_seed(sum(lens) + per)
    page, heads, rows = 64, kv_heads * per, len(lens)
    pool, table, keys, values = build(lens, kv_heads, hd, page, g)
    q = torch.randn(rows, heads, hd, generator=g, device="cuda")
    q[:, :, 5] *= 300
    n = rows * heads * hd
    out = torch.full((2, rows, heads, hd), 7.0, dtype=torch.bfloat16, device="cuda")
    status, length = torch.zeros(1, dtype=torch.int32, device="cuda"), ints(lens)
    args = (pool.data_ptr(), pool.shape[0], kv_heads, hd, page, q.data_ptr(), out.data_ptr(), heads, rows, table.data_ptr(),
            table.shape[1], length.data_ptr(), hd ** -0.5, n if split else 0)
    work = torch.empty(max(step_attention(*args, None, None, None), 16), dtype=torch.uint8, device="cuda")
    assert step_attention(*args, work.data_ptr(), status.data_ptr(), torch.cuda.current_stream().cuda_stream) == 0
    want, mass, peak = ref.attention(q, keys, values, lens, list(range(rows + 1)), False, hd ** -0.5)
    got = out[0].double() + (out[1].double() if split else 0)
    # fp32's roundings before the result and its planes' 2^-17, or bf16's
    if split:
        off = (got - want).abs() - tolerance(want, mass, peak, torch.float32, hd) - want.abs() * 2.0 ** -17
        assert off.max().item() <= 0, off.max().item()
    else:
        check(got, want, mass, peak, torch.bfloat16, hd)
        assert (out[1] == 7.0).all()
    assert status.item() == 0
