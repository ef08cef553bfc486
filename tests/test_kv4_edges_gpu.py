"""4-bit paged K/V cache operators at inputs where they can go wrong: rows that end inside a warp,
values at the end of fp16's range, NaNs beside what nobody sees, queries of unlike sizes."""
import math

import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
import moonshine_b200 as mb  # noqa: E402
from test_kv4_gpu import TYPES, build, check, ints, random_kv  # noqa: E402

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
