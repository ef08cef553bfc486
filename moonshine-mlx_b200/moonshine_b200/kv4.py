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
long as its strides are multiples of 16 bytes.  No call has a gradient: outside of
torch.no_grad() tensors that require one are refused.
"""
from __future__ import annotations

import ctypes as C
import struct
from typing import Optional, Tuple


class _Kv4Pool(C.Structure):
    _fields_ = [("base", C.c_void_p), ("page_stride", C.c_int64), ("head_stride", C.c_int64), ("pages", C.c_int32),
                ("kv_heads", C.c_int32), ("head_dim", C.c_int32), ("page_size", C.c_int32)]


class _KvTables(C.Structure):
    _fields_ = [("lengths", C.c_void_p), ("new_tokens", C.c_void_p), ("free_pages", C.c_void_p),
                ("block_table", C.c_void_p), ("slots", C.c_void_p), ("cu_new", C.c_void_p), ("counts", C.c_void_p),
                ("table_stride", C.c_int64), ("n_slots", C.c_int64), ("rows", C.c_int32), ("width", C.c_int32),
                ("page_size", C.c_int32), ("n_free", C.c_int32)]


class _Kv4Tokens(C.Structure):
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("slots", C.c_void_p), ("tokens", C.c_int64),
                ("k_token_stride", C.c_int64), ("k_head_stride", C.c_int64), ("v_token_stride", C.c_int64),
                ("v_head_stride", C.c_int64), ("dtype", C.c_int32), ("reserved", C.c_int32)]


class _Kv4AttentionArgs(C.Structure):
    _fields_ = [("q", C.c_void_p), ("out", C.c_void_p), ("q_tokens", C.c_int64), ("q_token_stride", C.c_int64),
                ("q_head_stride", C.c_int64), ("out_token_stride", C.c_int64), ("out_head_stride", C.c_int64),
                ("block_table", C.c_void_p), ("table_stride", C.c_int64), ("lens", C.c_void_p), ("cu_q", C.c_void_p),
                ("dtype", C.c_int32), ("heads", C.c_int32), ("rows", C.c_int32), ("width", C.c_int32),
                ("max_q", C.c_int32), ("causal", C.c_int32), ("scale", C.c_float), ("reserved", C.c_int32)]


# Structs go to the library as packed bytes: a decode step of a small batch is a few
# microseconds on the GPU, about what a ctypes structure costs to fill field by field.
STRUCTS = (("ms_kv_tables", _KvTables), ("ms_kv4_pool", _Kv4Pool), ("ms_kv4_tokens", _Kv4Tokens),
           ("ms_kv4_attention_args", _Kv4AttentionArgs))
_POOL = struct.Struct("Pqqiiii").pack
_TABLES = struct.Struct("PPPPPPPqqiiii").pack
_TOKENS = struct.Struct("PPPqqqqqii").pack
_ATTENTION = struct.Struct("PPqqqqqPqPPiiiiiifi").pack

_P, _I = C.c_void_p, C.c_int32
SIGNATURES = {
    "ms_kv4_position_bytes": (_I, [_I]),
    "ms_kv_block_tables": (C.c_int, [_P, _I, _P]),
    "ms_kv4_append": (C.c_int, [_P, _P, _I, _P]),
    "ms_kv4_read": (C.c_int, [_P, _P, _I, _P]),
    "ms_kv4_attention_workspace": (C.c_int64, [_P, _P]),
    "ms_kv4_attention": (C.c_int, [_P, _P, _P, C.c_int64, _I, _P]),
}


class _Api:
    """torch, the library's functions and what the calls look up, bound on first use."""

    def __init__(self):
        import torch

        from . import _L, _check
        lib = _L()
        self.torch, self.check, self.lib = torch, _check, lib
        self.codes = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
        self.u8, self.i32, self.i64 = torch.uint8, torch.int32, torch.int64
        self.each = {hd: lib.ms_kv4_position_bytes(hd) for hd in range(8, 129, 8)}
        self.stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
        if self.stream is None:
            self.stream = lambda index: torch.cuda.current_stream(index).cuda_stream


_bound: Optional[_Api] = None


def _api() -> _Api:
    global _bound
    if _bound is None:
        _bound = _Api()
    return _bound


# ---------------------------------------------------------------- refusals, in words
# A call tests all of its arguments in one expression and comes here only when that fails.
def _on(t, name, dtype, device, ndim):
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")
    if not t.is_cuda or t.get_device() != device:
        raise ValueError(f"{name} must be on a CUDA device, all tensors of a call on the same; it is on {t.device}")


def _vector(t, name, dtype, device, numel=None):
    _on(t, name, dtype, device, 1)
    if numel is not None and t.shape[0] != numel:
        raise ValueError(f"{name} must have {numel} entries, not {t.shape[0]}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _tokens(t, name, dtype, device, shape):
    _on(t, name, dtype, device, 3)
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must be {tuple(shape)}, not {tuple(t.shape)}")
    if t.stride(2) != 1:
        raise ValueError(f"{name}'s last dimension must be contiguous")


def _no_gradient(a, t, name):
    if t.requires_grad and a.torch.is_grad_enabled():
        raise ValueError(f"{name} requires a gradient and this call has none: detach it, or call under torch.no_grad()")


def _pages(a, pool, head_dim):
    if head_dim not in a.each:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, not {head_dim}")
    _on(pool, "pool", a.u8, pool.get_device(), 3)
    each = a.each[head_dim]
    if pool.shape[2] == 0 or pool.shape[2] % (16 * each) or pool.stride(2) != 1:
        raise ValueError(f"pool must be [pages, kv_heads, page_size * {each}] for head_dim {head_dim}, its last "
                         f"dimension contiguous and page_size a multiple of 16; it is {tuple(pool.shape)}")


def _table(a, block_table, device):
    _on(block_table, "block_table", a.i32, device, 2)
    if block_table.shape[1] > 1 and block_table.stride(1) != 1:
        raise ValueError("block_table's rows must be contiguous")


def _floats(a, t, name, ndim=3):
    if t.dtype not in a.codes:
        raise ValueError(f"{name} must be float32, float16 or bfloat16, not {t.dtype}")
    if t.dim() != ndim:
        raise ValueError(f"{name} must have {ndim} dimensions, not {t.dim()}")


# ---------------------------------------------------------------- the operators
def kv4_position_bytes(head_dim: int) -> int:
    """Bytes of one position's K and V for one head: head_dim + 8 * ceil(head_dim / 64)."""
    each = _api().each
    if head_dim not in each:
        raise ValueError(f"head_dim must be a multiple of 8 from 8 to 128, not {head_dim}")
    return each[head_dim]


def kv4_pool(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, device="cuda"):
    """An empty pool: uint8 [pages, kv_heads, page_size * kv4_position_bytes(head_dim)]."""
    if page_size <= 0 or page_size % 16:
        raise ValueError(f"page_size must be a positive multiple of 16, not {page_size}")
    a = _api()
    return a.torch.zeros(pages, kv_heads, page_size * kv4_position_bytes(head_dim), dtype=a.u8, device=device)


def kv_block_tables(lengths, new_tokens, block_table, page_size: int, max_new: int, free_pages=None,
                    n_pages: Optional[int] = None) -> Tuple:
    """Pages and slots for the new tokens of every row (ms_kv_block_tables).

    ``lengths`` and ``new_tokens`` are int32 [rows]; ``block_table`` int32 [rows, width] is
    updated in place: rows take pages from ``free_pages`` (int32; or the pages
    0 .. ``n_pages`` - 1) in row order, and entries behind a row's pages become -1.  Returns
    slots int64 [max_new] (-1 without a page and behind the last token), cu_new int32
    [rows + 1] and counts int32 [2] = (pages needed, new tokens), all on the device."""
    a = _bound or _api()
    i32 = a.i32
    device = block_table.get_device()
    if (free_pages is None) == (n_pages is None):
        raise ValueError("give either free_pages or n_pages")
    shape, step = block_table.shape, block_table.stride()
    if not (device >= 0 and len(shape) == 2 and lengths.dtype is i32 and new_tokens.dtype is i32
            and block_table.dtype is i32 and lengths.get_device() == device and new_tokens.get_device() == device
            and lengths.shape == new_tokens.shape == shape[:1] and lengths.is_contiguous()
            and new_tokens.is_contiguous() and (step[1] == 1 or shape[1] <= 1)
            and (free_pages is None or (free_pages.dtype is i32 and free_pages.get_device() == device
                                        and free_pages.dim() == 1 and free_pages.is_contiguous()))):
        _table(a, block_table, device)
        _vector(lengths, "lengths", i32, device, shape[0])
        _vector(new_tokens, "new_tokens", i32, device, shape[0])
        if free_pages is not None:
            _vector(free_pages, "free_pages", i32, device)
    rows, width = shape
    slots = a.torch.empty(max_new, dtype=a.i64, device=block_table.device)
    cu_new, counts = lengths.new_empty(rows + 1), lengths.new_empty(2)
    status = a.lib.ms_kv_block_tables(
        _TABLES(lengths.data_ptr(), new_tokens.data_ptr(), 0 if free_pages is None else free_pages.data_ptr(),
                block_table.data_ptr(), slots.data_ptr(), cu_new.data_ptr(), counts.data_ptr(), step[0], max_new, rows,
                width, page_size, n_pages if free_pages is None else free_pages.shape[0]),
        device, a.stream(device))
    if status:
        a.check(status)
    return slots, cu_new, counts


def kv4_append(pool, k, v, slots) -> None:
    """Quantizes k and v [tokens, kv_heads, head_dim] into their ``slots`` (int64 [tokens];
    -1: left out) of the pool (ms_kv4_append)."""
    a = _bound or _api()
    code = a.codes.get(k.dtype)
    device = pool.get_device()
    shape, ks, vs, ps = k.shape, k.stride(), v.stride(), pool.shape
    if k.requires_grad or v.requires_grad:
        _no_gradient(a, k, "k")
        _no_gradient(a, v, "v")
    if not (code is not None and device >= 0 and len(shape) == 3 and len(ps) == 3 and shape[2] in a.each
            and shape[1] == ps[1] and v.shape == shape and v.dtype is k.dtype and ks[2] == vs[2] == 1
            and k.get_device() == v.get_device() == slots.get_device() == device and pool.dtype is a.u8
            and slots.dtype is a.i64 and slots.shape == shape[:1] and slots.is_contiguous()
            and ps[2] > 0 and ps[2] % (16 * a.each[shape[2]]) == 0 and pool.stride(2) == 1):
        _floats(a, k, "k")
        _pages(a, pool, shape[2])
        want = (shape[0], ps[1], shape[2])
        _tokens(k, "k", k.dtype, device, want)
        _tokens(v, "v", k.dtype, device, want)
        _vector(slots, "slots", a.i64, device, shape[0])
    status = a.lib.ms_kv4_append(
        _POOL(pool.data_ptr(), *pool.stride()[:2], ps[0], ps[1], shape[2], ps[2] // a.each[shape[2]]),
        _TOKENS(k.data_ptr(), v.data_ptr(), slots.data_ptr(), shape[0], ks[0], ks[1], vs[0], vs[1], code, 0),
        device, a.stream(device))
    if status:
        a.check(status)


def kv4_read(pool, slots, head_dim: int, dtype=None) -> Tuple:
    """(k, v) [tokens, kv_heads, head_dim] of the ``slots``: the values that the stored codes
    stand for, rounded to ``dtype`` (float32), zeros for a slot outside the pool (ms_kv4_read)."""
    a = _bound or _api()
    if dtype is None:
        dtype = a.torch.float32
    code = a.codes.get(dtype)
    if code is None:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    device, ps = pool.get_device(), pool.shape
    if not (device >= 0 and len(ps) == 3 and head_dim in a.each and pool.dtype is a.u8 and slots.dtype is a.i64
            and slots.get_device() == device and slots.dim() == 1 and slots.is_contiguous() and ps[2] > 0
            and ps[2] % (16 * a.each[head_dim]) == 0 and pool.stride(2) == 1):
        _pages(a, pool, head_dim)
        _vector(slots, "slots", a.i64, device)
    tokens, heads = slots.shape[0], ps[1]
    k = a.torch.empty((tokens, heads, head_dim), dtype=dtype, device=pool.device)
    v = a.torch.empty_like(k)
    step = heads * head_dim
    status = a.lib.ms_kv4_read(
        _POOL(pool.data_ptr(), *pool.stride()[:2], ps[0], heads, head_dim, ps[2] // a.each[head_dim]),
        _TOKENS(k.data_ptr(), v.data_ptr(), slots.data_ptr(), tokens, step, head_dim, step, head_dim, code, 0),
        device, a.stream(device))
    if status:
        a.check(status)
    return k, v


def kv4_attention(q, pool, block_table, lens, cu_q=None, max_q: Optional[int] = None, causal: bool = True,
                  scale: Optional[float] = None, out=None):
    """softmax(scale q k^T) v over the pages of each row (ms_kv4_attention).

    ``q`` [tokens, heads, head_dim]; row b's tokens are ``cu_q[b]`` .. ``cu_q[b + 1]`` (int32
    [rows + 1], with ``max_q`` the longest row; None: one token per row).  ``lens`` int32 [rows]
    counts the row's positions, under ``causal`` including those of its queries: query i of n
    sees the positions up to lens - n + i.  ``scale`` defaults to head_dim^-1/2.  Returns
    ``out`` (made like q if not given; tokens of no row are left as they are)."""
    a = _bound or _api()
    code = a.codes.get(q.dtype)
    device = pool.get_device()
    shape, ps, qs, ts, tp = q.shape, pool.shape, q.stride(), block_table.shape, block_table.stride()
    if scale is not None and not abs(scale) >= 1e-37:
        raise ValueError(f"scale must be None or at least 1e-37 in magnitude, not {scale}")
    if cu_q is None:
        max_q = 1
    elif max_q is None:
        raise ValueError("cu_q needs max_q, the most tokens of a row")
    if out is None:
        out = a.torch.empty(shape, dtype=q.dtype, device=q.device)
    if q.requires_grad or out.requires_grad:
        _no_gradient(a, q, "q")
        _no_gradient(a, out, "out")
    os = out.stride()
    if not (code is not None and device >= 0 and len(shape) == 3 and len(ps) == 3 and len(ts) == 2
            and shape[2] in a.each and shape[1] > 0 and ps[1] > 0 and shape[1] % ps[1] == 0 and qs[2] == os[2] == 1
            and out.shape == shape and out.dtype is q.dtype and pool.dtype is a.u8 and block_table.dtype is a.i32
            and lens.dtype is a.i32 and q.get_device() == block_table.get_device() == device
            and lens.get_device() == out.get_device() == device and (tp[1] == 1 or ts[1] <= 1)
            and lens.shape == ts[:1] and lens.is_contiguous() and ps[2] > 0 and ps[2] % (16 * a.each[shape[2]]) == 0
            and pool.stride(2) == 1
            and (shape[0] == ts[0] if cu_q is None else
                 cu_q.dtype is a.i32 and cu_q.get_device() == device and cu_q.dim() == 1
                 and cu_q.shape[0] == ts[0] + 1 and cu_q.is_contiguous())):
        _floats(a, q, "q")
        _pages(a, pool, shape[2])
        _tokens(q, "q", q.dtype, device, shape)
        if shape[1] == 0 or ps[1] == 0 or shape[1] % ps[1]:
            raise ValueError(f"q's {shape[1]} heads are no multiple of the pool's {ps[1]}")
        _tokens(out, "out", q.dtype, device, shape)
        _table(a, block_table, device)
        _vector(lens, "lens", a.i32, device, ts[0])
        if cu_q is not None:
            _vector(cu_q, "cu_q", a.i32, device, ts[0] + 1)
        elif shape[0] != ts[0]:
            raise ValueError(f"without cu_q q holds one token per row: {shape[0]} tokens for {ts[0]} rows")
    pages = _POOL(pool.data_ptr(), *pool.stride()[:2], ps[0], ps[1], shape[2], ps[2] // a.each[shape[2]])
    args = _ATTENTION(q.data_ptr(), out.data_ptr(), shape[0], qs[0], qs[1], os[0], os[1], block_table.data_ptr(), tp[0],
                      lens.data_ptr(), 0 if cu_q is None else cu_q.data_ptr(), code, shape[1], ts[0], ts[1], max_q,
                      1 if causal else 0, scale or 0.0, 0)
    need = a.lib.ms_kv4_attention_workspace(pages, args)
    work = None if need <= 0 else a.torch.empty(need, dtype=a.u8, device=q.device)
    status = a.lib.ms_kv4_attention(pages, args, None if work is None else work.data_ptr(), need, device,
                                    a.stream(device))
    if status:
        a.check(status)
    return out
