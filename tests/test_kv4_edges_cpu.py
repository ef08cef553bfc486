"""Refusals of the 4-bit K/V cache operators that the argument structs leave open, without GPU work."""
import pytest

torch = pytest.importorskip("torch")

import moonshine_b200 as mb  # noqa: E402
from test_kv4_cpu import attention_struct, pool_struct, refused  # noqa: E402


@pytest.mark.parametrize("max_q", [0, 1, 7])
@pytest.mark.parametrize("changes,text", [
    (dict(q=None), "null q"), (dict(out=None), "null q"), (dict(lens=None), "null q"), (dict(block_table=None), "null block_table"),
    (dict(rows=4), "one token per row"), (dict(q_tokens=1), "one token per row"), (dict(q=(1 << 20) + 2), "aligned"),
    (dict(width=(1 << 26) + 1), "2^30"), (dict(out_head_stride=63), "strides"), (dict(out=1 << 20), "may not be q")])
def test_without_cu_q_max_q_has_no_say(changes, text, max_q):
    """One token per row: every check is made, whatever max_q holds."""
    L, p = mb._L(), pool_struct()
    args = attention_struct(max_q=max_q, **changes)
    assert L.ms_kv4_attention_workspace(p, args) == -1
    assert text in L.ms_last_error().decode()
    refused(L.ms_kv4_attention(p, args, None, 0, -1, None), text)


def test_largest_page_size():
    """Pages of more than 2^30 positions are refused (in a process of its own: the call once did
    not return)."""
    code = """
import ctypes as C, moonshine_b200 as mb
from moonshine_b200 import kv4
L = mb._L()
for page_size in (2 ** 30 + 16, 2 ** 31 - 16):
    pool = C.byref(kv4._Kv4Pool(base=None, page_stride=0, head_stride=0, pages=0, kv_heads=1, head_dim=64, page_size=page_size))
    t = C.byref(kv4._Kv4Tokens(k=1 << 20, v=1 << 21, slots=1 << 20, tokens=3, k_token_stride=64, k_head_stride=64,
                               v_token_stride=64, v_head_stride=64, dtype=0, reserved=0))
    for call in (L.ms_kv4_append, L.ms_kv4_read):
        assert call(pool, t, -1, None) == 1 and b"page_size" in L.ms_last_error()
"""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(mb.__file__)))
    r = subprocess.run([sys.executable, "-c", code], env={**os.environ, "PYTHONPATH": root}, capture_output=True, text=True,
                       timeout=60)
    assert r.returncode == 0, r.stderr[-2000:]


def test_tensors_that_want_a_gradient():
    """The operators have none: a call that would cut the graph is refused, one under no_grad is not
    (it goes on to the next check, which CPU tensors fail)."""
    pool, slots = torch.zeros(4, 2, 16 * 72, dtype=torch.uint8), torch.zeros(3, dtype=torch.int64)
    table, lens = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    x, y = torch.zeros(3, 2, 64), torch.zeros(3, 2, 64, requires_grad=True)
    for k, v, name in ((y, x, "k"), (x, y, "v"), (y * 2, x, "k")):
        with pytest.raises(ValueError, match=name + " requires a gradient"):
            mb.kv4_append(pool, k, v, slots)
    for q, out, name in ((y, None, "q"), (x, y, "out")):
        with pytest.raises(ValueError, match=name + " requires a gradient"):
            mb.kv4_attention(q, pool, table, lens, out=out)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        mb.kv4_append(pool, y, y, slots)
    with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):
        mb.kv4_attention(y, pool, table, lens, out=y)
    with pytest.raises(ValueError, match="CUDA"):
        mb.kv4_attention(y.detach(), pool, table, lens)
