"""4-bit paged K/V cache operators on torch CUDA tensors (ms_kv_* of include/moonshine_b200.h).

    pool = kv4_pool(pages, kv_heads, head_dim, page_size)             # uint8 [pages, kv_heads, page bytes]
    slots, cu, counts = kv_block_tables(lengths, new, table, page_size, max_new, free_pages=free)
    kv4_append(pool, k, v, slots)                                     # k, v [tokens, kv_heads, head_dim]
    out = kv4_attention(q, pool, table, lens, cu_q=cu, max_q=longest) # q [tokens, heads, head_dim]
    k, v = kv4_read(pool, slots, head_dim)                            # the values that the codes stand for

Every call enqueues on the current stream of its tensors' device and returns without waiting,
so all of them can be captured into a CUDA graph, which replays with the lengths, tables and
pages that the device memory then holds.  All tensors of a call are on one CUDA device.  A
slice of a larger buffer can be the pool (one layer of [pages, layers, kv_heads, bytes]) as
long as its strides are multiples of 16 bytes.  No call has a gradient.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple


class _Kv4Pool(C.Structure):
    _fields_ = [("base", C.c_void_p), ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("pages", C.c_int32),
                ("kv_heads", C.c_int32), ("head_dim", C.c_int32), ("page_size", C.c_int32)]


class _Kv4AttentionArgs(C.Structure):
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("q_tokens", C.c_int64), ("q_token_stride", C.c_int64),
                ("q_head_stride", C.c_int64), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64),
                ("block_table", C.c_void_p), ("table_stride", C.c_int64), ("lens", C.c_void_p), ("cu_q", C.c_void_p),
                ("dtype", C.c_int32), ("heads", C.c_int32), ("rows", C.c_int32), ("width", C.c_int32),
                ("max_q", C.c_int32), ("causal", C.c_int32), ("scale", C.c_float), ("reserved", C.c_int32)]


_P, _I, _L = C.c_void_p, C.c_int32, C.c_int64
SIGNATURES = {
    "ms_kv4_position_bytes": (_I, [_I]),
    "ms_kv_block_tables": (C.c_int, [_P, _P, _I, _I, _P, _I, _P, _I, _L, _P, _L, _P, _P, _I, _P]),
    "ms_kv4_append": (C.c_int, [C.POINTER(_Kv4Pool), _P, _P, _I, _L, _L, _L, _L, _L, _P, _I, _P]),
    "ms_kv4_read": (C.c_int, [C.POINTER(_Kv4Pool), _P, _P, _I, _L, _L, _L, _L, _L, _P, _I, _P]),
    "ms_kv4_attention_workspace": (_L, [C.POINTER(_Kv4Pool), C.POINTER(_Kv4AttentionArgs)]),
    "ms_kv4_attention": (C.c_int, [C.POINTER(_Kv4Pool), C.POINTER(_Kv4AttentionArgs), _P, _L, _I, _P]),
}
STRUCTS = (("ms_kv4_pool", _Kv4Pool), ("ms_kv4_attention_args", _Kv4AttentionArgs))

_bound = None


def _api():
    """(torch, the library, the package's status check, dtype codes), bound on first use."""
    global _bound
    if _bound is None:
        import torch

        from . import _L as lib, _check
        _bound = (torch, lib(), _check, {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    return _bound


def _on(t, name, dtype, device=None, ndim=None):
    """Refuses a tensor of another type, device or rank."""
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if not t.is_cuda or (device is not None and t.device != device):
        raise ValueError(f"{name} must be on {'a CUDA device' if device is None else device}, not on {t.device}")
    if ndim is not None and t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")


def _flat(t, name, dtype, device, numel=None):
    """_on for a contiguous vector (of `numel` entries)."""
    _on(t, name, dtype, device, 1)
    if numel is not None and t.shape[0] != numel:
        raise ValueError(f"{name} must have {numel} entries, not {t.shape[0]}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _pool(torch, lib, pool, head_dim):
    _on(pool, "pool", torch.uint8, None, 3)
    pages, heads, nbytes = pool.shape
    each = lib.ms_kv4_position_bytes(head_dim)
    if each == 0:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, not {head_dim}")
    if nbytes == 0 or nbytes % (16 * each) or pool.stride(2) != 1:
        raise ValueError(f"pool must be [pages, kv_heads, page_size * {each}] for head_dim {head_dim}, its last "
                         f"dimension contiguous and page_size a multiple of 16; got {tuple(pool.shape)}")
    return _Kv4Pool(pool.data_ptr(), pool.stride(0), pool.stride(1), pages, heads, head_dim, nbytes // each)


def _vectors(t, name, dtype, device, shape):
    """Refuses all but [tokens, heads, head_dim] with a contiguous head_dim; its strides."""
    _on(t, name, dtype, device, 3)
    if t.shape != shape:
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")
    return t.stride(0), t.stride(1)


def _code(codes, dtype, name):
    code = codes.get(dtype)
    if code is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {dtype}")
    return code


def kv4_position_bytes(head_dim: int) -> int:
    """Bytes of one position's K and V for one head: head_dim + 8 * ceil(head_dim / 64)."""
    n = _api()[1].ms_kv4_position_bytes(int(head_dim))
    if n == 0:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, not {head_dim}")
    return n


def kv4_pool(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
    """An empty pool: uint8 [pages, kv_heads, page_size * kv4_position_bytes(head_dim)]."""
    if page_size <= 0 or page_size % 16:
        raise ValueError(f"page_size must be a positive multiple of 16, not {page_size}")
    torch = _api()[0]
    return torch.zeros(pages, kv_heads, page_size * kv4_position_bytes(head_dim), dtype=torch.uint8, device=device)


def kv_block_tables(lengths, new_tokens, block_table, page_size: int, max_new: int, free_pages=None,
                    n_pages: Optional[int] = None) -> Tuple:
    """Pages and slots for the new tokens of every row (ms_kv_block_tables).

    ``lengths`` and ``new_tokens`` are int32 [rows]; ``block_table`` int32 [rows, width] is
    updated in place: rows take pages from ``free_pages`` (int32; or the pages
    0 .. ``n_pages`` - 1) in row order, and entries behind a row's pages become -1.  Returns
    slots int64 [max_new] (-1 without a page and behind the last token), cu_new int32
    [rows + 1] and counts int32 [2] = (pages needed, new tokens), all on the device."""
    torch, lib, check, _ = _api()
    _on(block_table, "block_table", torch.int32, None, 2)
    device = block_table.device
    rows, width = block_table.shape
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table's rows must be contiguous")
    _flat(lengths, "lengths", torch.int32, device, rows)
    _flat(new_tokens, "new_tokens", torch.int32, device, rows)
    if (free_pages is None) == (n_pages is None):
        raise ValueError("give either free_pages or n_pages")
    if free_pages is not None:
        _flat(free_pages, "free_pages", torch.int32, device)
    slots = torch.empty(max_new, dtype=torch.int64, device=device)
    sums = torch.empty(rows + 3, dtype=torch.int32, device=device)
    cu_new, counts = sums[:rows + 1], sums[rows + 1:]
    index = device.index
    check(lib.ms_kv_block_tables(lengths.data_ptr(), new_tokens.data_ptr(), rows, page_size,
                                 None if free_pages is None else free_pages.data_ptr(),
                                 n_pages if free_pages is None else free_pages.shape[0], block_table.data_ptr(), width,
                                 block_table.stride(0), slots.data_ptr(), max_new, cu_new.data_ptr(),
                                 counts.data_ptr(), index, torch.cuda.current_stream(index).cuda_stream))
    return slots, cu_new, counts


def kv4_append(pool, k, v, slots) -> None:
    """Quantizes k and v [tokens, kv_heads, head_dim] into their ``slots`` (int64 [tokens];
    -1: left out) of the pool (ms_kv4_append)."""
    torch, lib, check, codes = _api()
    code = _code(codes, k.dtype, "k")
    if k.dim() != 3:
        raise ValueError(f"k must have 3 dimensions, not {k.dim()}")
    p = _pool(torch, lib, pool, k.shape[2])
    device = pool.device
    shape = (k.shape[0], p.kv_heads, p.head_dim)
    ks, vs = _vectors(k, "k", k.dtype, device, shape), _vectors(v, "v", k.dtype, device, shape)
    _flat(slots, "slots", torch.int64, device, shape[0])
    index = device.index
    check(lib.ms_kv4_append(p, k.data_ptr(), v.data_ptr(), code, shape[0], *ks, *vs, slots.data_ptr(), index,
                            torch.cuda.current_stream(index).cuda_stream))


def kv4_read(pool, slots, head_dim: int, dtype=None) -> Tuple:
    """(k, v) [tokens, kv_heads, head_dim] of the ``slots``: the values that the stored codes
    stand for, rounded to ``dtype`` (float32), zeros for a slot outside the pool (ms_kv4_read)."""
    torch, lib, check, codes = _api()
    dtype = torch.float32 if dtype is None else dtype
    code = _code(codes, dtype, "dtype")
    p = _pool(torch, lib, pool, int(head_dim))
    device = pool.device
    _flat(slots, "slots", torch.int64, device)
    k = torch.empty(slots.shape[0], p.kv_heads, p.head_dim, dtype=dtype, device=device)
    v = torch.empty_like(k)
    index, st, sh = device.index, k.stride(0), k.stride(1)
    check(lib.ms_kv4_read(p, k.data_ptr(), v.data_ptr(), code, slots.shape[0], st, sh, st, sh, slots.data_ptr(), index,
                          torch.cuda.current_stream(index).cuda_stream))
    return k, v


def kv4_attention(q, pool, block_table, lens, cu_q=None, max_q: Optional[int] = None, causal: bool = True,
                  scale: Optional[float] = None, out=None):
    """softmax(scale q k^T) v over the pages of each row (ms_kv4_attention).

    ``q`` [tokens, heads, head_dim]; row b's tokens are ``cu_q[b]`` .. ``cu_q[b + 1]`` (int32
    [rows + 1], with ``max_q`` the longest row; None: one token per row).  ``lens`` int32 [rows]
    counts the row's positions, under ``causal`` including those of its queries: query i of n
    sees the positions up to lens - n + i.  ``scale`` defaults to head_dim^-1/2.  Returns
    ``out`` (made like q if not given; tokens of no row are left as they are)."""
    torch, lib, check, codes = _api()
    code = _code(codes, q.dtype, "q")
    if q.dim() != 3:
        raise ValueError(f"q must have 3 dimensions, not {q.dim()}")
    p = _pool(torch, lib, pool, q.shape[2])
    device = pool.device
    qs = _vectors(q, "q", q.dtype, device, q.shape)
    if q.shape[1] == 0 or q.shape[1] % p.kv_heads:
        raise ValueError(f"q's {q.shape[1]} heads are no multiple of the pool's {p.kv_heads}")
    _on(block_table, "block_table", torch.int32, device, 2)
    rows, width = block_table.shape
    if width > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table's rows must be contiguous")
    _flat(lens, "lens", torch.int32, device, rows)
    if cu_q is None:
        if q.shape[0] != rows:
            raise ValueError(f"without cu_q q holds one token per row: {q.shape[0]} tokens for {rows} rows")
        max_q = 1
    else:
        _flat(cu_q, "cu_q", torch.int32, device, rows + 1)
        if max_q is None:
            raise ValueError("cu_q needs max_q, the most tokens of a row")
    if scale is not None and not scale:
        raise ValueError("scale must not be 0")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=device)
    os = _vectors(out, "out", q.dtype, device, q.shape)
    a = _Kv4AttentionArgs(q.data_ptr(), out.data_ptr(), q.shape[0], *qs, *os, block_table.data_ptr(),
                          block_table.stride(0), lens.data_ptr(), None if cu_q is None else cu_q.data_ptr(), code,
                          q.shape[1], rows, width, max_q, bool(causal), scale or 0.0, 0)
    need = lib.ms_kv4_attention_workspace(p, a)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need > 0 else None
    index = device.index
    check(lib.ms_kv4_attention(p, a, None if work is None else work.data_ptr(), max(need, 0), index,
                               torch.cuda.current_stream(index).cuda_stream))
    return out
