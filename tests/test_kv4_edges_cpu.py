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
