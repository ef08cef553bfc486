"""Refusals and host-side parts of the 4-bit K/V cache operators: no GPU work is reached."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

import kv4_reference as ref  # noqa: E402
import moonshine_b200 as mb  # noqa: E402
from moonshine_b200 import kv4  # noqa: E402

INVALID, CAPACITY, UNSUPPORTED = 1, 9, 8


def test_position_bytes():
    for hd in (8, 24, 40, 64, 72, 96, 128):
        assert mb.kv4_position_bytes(hd) == ref.position_bytes(hd)
    for hd in (0, 4, 60, 136, -8):
        with pytest.raises(ValueError, match="head_dim"):
            mb.kv4_position_bytes(hd)


def test_tile_layout_covers_every_byte_once():
    """Code words and (scale, bias) words of a tile of 16 positions fill it without overlap."""
    for hd in range(8, 129, 8):
        seen = []
        for r in range(16):
            for value in (0, 1):
                seen += [ref.code_byte(hd, w, r, value) for w in range(hd // 8)]
                seen += [ref.meta_byte(hd, n, r, value) for n in range(-(-hd // 64))]
        assert sorted(seen) == list(range(0, 16 * ref.position_bytes(hd), 4))


def test_reference_quantizer_on_known_groups():
    x = torch.arange(16.0)[None]
    c, s, b, v = ref.quantize(x)
    assert c[0].tolist() == list(range(16)) and (s.item(), b.item()) == (1.0, 0.0) and torch.equal(v, x.double())
    x = torch.tensor([[0.0, 0.5, 1.49, 1.5, 15.0]])  # a value on a border goes up
    assert ref.quantize(x)[0][0].tolist() == [0, 1, 1, 2, 15]
    assert ref.quantize(torch.full((1, 5), 2.0))[3].tolist() == [[2.0] * 5]


def pool_struct(**changes):
    p = dict(base=1 << 20, page_stride=2 * 16 * 72, head_stride=16 * 72, pages=4, kv_heads=2, head_dim=64, page_size=16)
    p.update(changes)
    return C.byref(kv4._Kv4Pool(**p))


def tokens_struct(**changes):
    t = dict(k=1 << 20, v=1 << 21, slots=1 << 20, tokens=3, k_token_stride=128, k_head_stride=64, v_token_stride=128,
             v_head_stride=64, dtype=0, reserved=0)
    t.update(changes)
    return C.byref(kv4._Kv4Tokens(**t))


def refused(status, text, code=INVALID):
    assert status == code, status
    assert text in mb._L().ms_last_error().decode()


@pytest.mark.parametrize("changes,text,code", [
    (dict(head_dim=60), "multiple of 8", UNSUPPORTED), (dict(head_dim=136), "multiple of 8", UNSUPPORTED),
    (dict(page_size=8), "page_size", INVALID), (dict(page_size=0), "page_size", INVALID),
    (dict(pages=-1), "pages", INVALID), (dict(kv_heads=0), "kv_heads", INVALID), (dict(base=None), "null pool", INVALID),
    (dict(base=(1 << 20) + 8), "16 bytes", INVALID), (dict(page_stride=2 * 16 * 72 + 8), "16 bytes", INVALID),
    (dict(head_stride=16 * 72 - 16), "head_stride", INVALID), (dict(page_stride=16), "page_stride", INVALID)])
def test_pool_refusals(changes, text, code):
    L, p = mb._L(), pool_struct(**changes)
    refused(L.ms_kv4_append(p, tokens_struct(), -1, None), text, code)
    refused(L.ms_kv4_read(p, tokens_struct(), -1, None), text, code)
    refused(L.ms_kv4_attention(p, attention_struct(), None, 0, -1, None), text, code)
    assert L.ms_kv4_attention_workspace(p, attention_struct()) == -1


def attention_struct(**changes):
    a = dict(q=1 << 20, out=1 << 21, q_tokens=3, q_token_stride=256, q_head_stride=64, out_token_stride=256,
             out_head_stride=64, block_table=1 << 20, table_stride=4, lens=1 << 20, cu_q=None, dtype=0, heads=4, rows=3,
             width=4, max_q=1, causal=1, scale=0.0, reserved=0)
    a.update(changes)
    return C.byref(kv4._Kv4AttentionArgs(**a))


@pytest.mark.parametrize("changes,text", [
    (dict(dtype=3), "dtype"), (dict(rows=-1), "negative"), (dict(heads=3), "multiple of kv_heads"),
    (dict(heads=0), "multiple of kv_heads"), (dict(q=None), "null q"), (dict(lens=None), "null q"),
    (dict(block_table=None), "null block_table"), (dict(rows=4), "one token per row"), (dict(q=(1 << 20) + 2), "aligned"),
    (dict(scale=float("nan")), "finite"), (dict(width=(1 << 26) + 1), "2^30"), (dict(out_head_stride=63), "strides"), (dict(out_token_stride=0), "strides"), (dict(out=1 << 20), "may not be q"), (dict(rows=70000), "65535")])
def test_attention_refusals(changes, text):
    L, p = mb._L(), pool_struct()
    refused(L.ms_kv4_attention(p, attention_struct(**changes), None, 0, -1, None), text)


def test_queries_that_do_not_fit_a_launch():
    L, p = mb._L(), pool_struct()
    many = dict(q_tokens=10 ** 7, max_q=10 ** 7, cu_q=1 << 20)
    refused(L.ms_kv4_attention(p, attention_struct(**many), None, 0, -1, None), "several calls", UNSUPPORTED)
    assert L.ms_kv4_attention_workspace(p, attention_struct(**many)) == -1
    # max_q counts up to the tokens that there are
    assert L.ms_kv4_attention_workspace(p, attention_struct(q_tokens=200, max_q=10 ** 9, cu_q=1 << 20)) == 0
    assert L.ms_kv4_attention_workspace(p, attention_struct(q_tokens=10 ** 6, max_q=10 ** 6, cu_q=1 << 20)) == 0


def test_workspace_is_bounded():
    """Parts of long contexts take at most 256 MB, whatever the number of query tokens."""
    L, p = mb._L(), pool_struct(page_size=64, page_stride=2 * 64 * 72, head_stride=64 * 72)
    for tokens in (1, 100, 5000, 10 ** 5):
        n = L.ms_kv4_attention_workspace(p, attention_struct(dtype=2, q_tokens=tokens, max_q=tokens, cu_q=1 << 20, rows=2,
                                                             width=1 << 14))
        assert 0 <= n <= 256 << 20, (tokens, n)


def test_empty_calls_do_nothing():
    L, p = mb._L(), pool_struct()
    for changes in (dict(rows=0), dict(q_tokens=0, cu_q=1 << 20), dict(max_q=0, cu_q=1 << 20)):
        assert L.ms_kv4_attention(p, attention_struct(**changes), None, 0, -1, None) == 0
    none = tokens_struct(k=None, v=None, slots=None, tokens=0)
    assert L.ms_kv4_append(p, none, -1, None) == 0
    assert L.ms_kv4_read(p, none, -1, None) == 0
    assert L.ms_kv4_append(pool_struct(pages=0, base=None), tokens_struct(), -1, None) == 0


@pytest.mark.parametrize("changes,text", [
    (dict(dtype=5), "dtype"), (dict(k=None), "null k"), (dict(v=None), "null k"), (dict(slots=None), "null k"),
    (dict(v=(1 << 20) + 1, dtype=1), "aligned"), (dict(tokens=-3), "negative")])
def test_store_refusals(changes, text):
    L, p = mb._L(), pool_struct()
    refused(L.ms_kv4_append(p, tokens_struct(**changes), -1, None), text)
    refused(L.ms_kv4_read(p, tokens_struct(**changes), -1, None), text)
    refused(L.ms_kv4_append(None, tokens_struct(), -1, None), "null pool")
    refused(L.ms_kv4_read(p, tokens_struct(k_head_stride=32), -1, None), "strides")
    refused(L.ms_kv4_read(p, tokens_struct(v_token_stride=0), -1, None), "strides")
    refused(L.ms_kv4_append(p, None, -1, None), "null tokens")


@pytest.mark.parametrize("changes,text", [
    (dict(lengths=None), "null lengths"), (dict(new_tokens=None), "null lengths"), (dict(rows=-1), "negative"),
    (dict(page_size=0), "page_size"), (dict(block_table=None), "null block_table"), (dict(table_stride=3), "table_stride"),
    (dict(slots=None), "null slots"), (dict(n_slots=1 << 31), "n_slots"), (dict(cu_new=None), "null cu_new"),
    (dict(counts=None), "null cu_new"), (dict(n_free=-1), "negative")])
def test_table_refusals(changes, text):
    x = 1 << 20
    t = dict(lengths=x, new_tokens=x, free_pages=x, block_table=x, slots=x, cu_new=x, counts=x, table_stride=4, n_slots=7,
             rows=3, width=4, page_size=16, n_free=9)
    t.update(changes)
    refused(mb._L().ms_kv_block_tables(C.byref(kv4._KvTables(**t)), -1, None), text)
    refused(mb._L().ms_kv_block_tables(None, -1, None), "null arguments")


def test_python_refusals():
    i32, i64 = (lambda *n: torch.zeros(*n, dtype=torch.int32)), (lambda *n: torch.zeros(*n, dtype=torch.int64))
    pool = torch.zeros(4, 2, 16 * 72, dtype=torch.uint8)
    with pytest.raises(ValueError, match="CUDA"):
        mb.kv4_append(pool, torch.zeros(3, 2, 64), torch.zeros(3, 2, 64), i64(3))
    with pytest.raises(ValueError, match="uint8"):
        mb.kv4_read(pool.float(), i64(3), 64)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        mb.kv4_append(pool, torch.zeros(3, 2, 64, dtype=torch.float64), torch.zeros(3, 2, 64), i64(3))
    with pytest.raises(ValueError, match="CUDA"):
        mb.kv4_attention(torch.zeros(3, 4, 64), pool, i32(3, 4), i32(3))
    with pytest.raises(ValueError, match="3 dimensions"):
        mb.kv4_attention(torch.zeros(3, 256), pool, i32(3, 4), i32(3))
    with pytest.raises(ValueError, match="CUDA"):
        mb.kv_block_tables(i32(3), i32(3), i32(3, 4), 16, 5, n_pages=4)
    with pytest.raises(ValueError, match="int32"):
        mb.kv_block_tables(i32(3), i32(3), i64(3, 4), 16, 5, n_pages=4)
    with pytest.raises(ValueError, match="page_size"):
        mb.kv4_pool(4, 2, 64, 24)
    for scale in (0, 1e-60, float("nan")):
        with pytest.raises(ValueError, match="scale"):
            mb.kv4_attention(torch.zeros(3, 4, 64), pool, i32(3, 4), i32(3), scale=scale)


def test_structs_have_the_library_layout():
    L = mb._L()
    packs = {"ms_kv_tables": kv4._TABLES, "ms_kv4_pool": kv4._POOL, "ms_kv4_tokens": kv4._TOKENS,
             "ms_kv4_attention_args": kv4._ATTENTION}
    for name, cls in kv4.STRUCTS:
        size = C.sizeof(cls)
        assert L.ms_struct_size(name.encode()) == size
        # the packed form the calls pass: every field at its place
        values = [float(i + 1) if t is C.c_float else i + 1 for i, (_, t) in enumerate(cls._fields_)]
        assert packs[name](*values).ljust(size, b"\0") == bytes(cls(*values))
