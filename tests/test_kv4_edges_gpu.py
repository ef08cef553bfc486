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
