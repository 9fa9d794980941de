"""A paged key/value cache on MI355X: appending a step's keys and values, attention over the pages, and the same where
the batch shares a long prefix. The serving form of the contiguous caches of deepgengraph_amd.attention, with a length per
sequence.

The cache is two pools of pages, k_pages and v_pages [num_pages, page_size, Hkv, D] (any strides with a contiguous head
dimension: a [num_pages, Hkv, page_size, D] pool is passed as its transpose(1, 2)). Key j of sequence b is row
j % page_size of page block_table[b, j // page_size] (int32 [B, width]). kv_lens (int32 [B]) are the keys each sequence
holds, the step's own included. A step's tokens come as [B, Sq, heads, D], or, where the sequences bring different numbers
of them, one after the other as [T, heads, D] with cu_q (int32 [B + 1]): sequence b's are cu_q[b] .. cu_q[b + 1] - 1.

Lengths and table are read on the device: a call looks at no tensor from the host, launches on the current stream and can
be captured into a graph, whose replays read the lengths, the table and the pages anew. Unsupported types, shapes and
strides raise RuntimeError before any launch. No counterpart in the reference, whose decode cases read one contiguous
cache of one length for all sequences (deepgengraph_exp/cases/kernels/attn.py:18-34).
"""
from __future__ import annotations

import functools
import math
import struct

import torch

from . import _lib

_I32 = torch.int32
_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_STRIDES_19, _STRIDES_13 = struct.Struct("19q"), struct.Struct("13q")


# A step's small calls take the GPU 5 to 15 us, and the host about as long: the checks below look at each property once,
# in the cheapest form, and leave what the library checks itself (sizes, strides, alignment) to it.
def _device(*tensors):
    """The common GPU's index; None stands for an argument that was not given."""
    index = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != index or index < 0:
            _lib.require_gpu(*tensors)  # says what is wrong
    return index


def _launch(dev: int, name: str, *args):
    """The library call, with the tensors' device current (streams and kernels belong to one)."""
    if _current_device() == dev:
        return _lib.call(name, *args, _lib.stream_handle(dev))
    with torch.cuda.device(dev):
        return _lib.call(name, *args, _lib.stream_handle(dev))


def _tokens(op: str, name: str, t: torch.Tensor, cu_q):
    """(batch, token, head) strides of a step's tokens."""
    st = t.stride()
    if len(st) != (4 if cu_q is None else 3):
        raise RuntimeError(f"{op}: {name} must be {'[B, Sq, heads, D]' if cu_q is None else '[T, heads, D] with cu_q'}, "
                           f"got shape {tuple(t.shape)}")
    if st[-1] != 1:
        raise RuntimeError(f"{op}: {name}'s head dimension must be contiguous (stride {st[-1]})")
    return st[:3] if cu_q is None else (0, st[0], st[1])


def _cache(op: str, k_pages, v_pages, block_table, kv_lens, cu_q, B: int):
    """Checks of the pools, the table and the lengths; (shape of the pools, table width, strides of both pools)."""
    shape, ks, vs = k_pages.shape, k_pages.stride(), v_pages.stride()
    if len(shape) != 4 or v_pages.shape != shape or v_pages.dtype is not k_pages.dtype:
        raise RuntimeError(f"{op}: k_pages {tuple(shape)} {k_pages.dtype} and v_pages {tuple(v_pages.shape)} "
                           f"{v_pages.dtype} must be two [pages, page_size, Hkv, D] of one kind")
    if ks[3] != 1 or vs[3] != 1:
        raise RuntimeError(f"{op}: the pages' head dimension must be contiguous (strides {ks[3]}, {vs[3]})")
    table = block_table.shape
    if block_table.dtype is not _I32 or len(table) != 2 or table[0] != B or (table[1] > 1 and block_table.stride(1) != 1):
        raise RuntimeError(f"{op}: block_table must be int32 [{B}, width] with unit column stride")
    if kv_lens.dtype is not _I32 or kv_lens.shape != (B,) or not kv_lens.is_contiguous():
        raise RuntimeError(f"{op}: kv_lens must be contiguous int32 [{B}]")
    return shape, table[1], ks[:3] + vs[:3]


def _batch(op: str, t: torch.Tensor, cu_q):
    """(B, T, Sq) of a step's tokens; Sq 0 with cu_q."""
    if cu_q is None:
        return t.shape[0], t.shape[0] * t.shape[1], t.shape[1]
    if cu_q.dtype is not _I32 or cu_q.dim() != 1 or cu_q.shape[0] < 1 or not cu_q.is_contiguous():
        raise RuntimeError(f"{op}: cu_q must be contiguous int32 [B + 1]")
    return cu_q.shape[0] - 1, t.shape[0], 0


@functools.lru_cache(maxsize=4096)
def _workspace_bytes(op: str, *sizes: int) -> int:
    need = _lib.load().dgg_attn_paged_workspace_bytes(*sizes)
    if need < 0:
        raise RuntimeError(f"{op}: {_lib.load().dgg_last_error().decode(errors='replace')}")
    return need


def paged_append(key: torch.Tensor, value: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor,
                 block_table: torch.Tensor, kv_lens: torch.Tensor, *, query: torch.Tensor | None = None,
                 cu_q: torch.Tensor | None = None, rope_theta: float | None = None,
                 query_out: torch.Tensor | None = None) -> torch.Tensor | None:
    """Stores a step's key and value rows [B, Sq, Hkv, D] (or [T, Hkv, D] with cu_q) in the pages, in place, in one launch:
    token i of sequence b goes to position kv_lens[b] - Sq + i. With rope_theta the keys are rotated on the way by their
    position, as rotary_embedding_online rotates them (NeoX pairs (j, j + D/2), angle pos / theta^(2j/D); the angle is
    taken in 64 bits here, which matters at far positions), and so is `query` (the step's query rows, same leading shape),
    whose rotated copy is returned (in query_out, if given, which may be query itself). key, value and query may be views
    of one projection's result.

    float32, float16, bfloat16; D a multiple of 16 up to 512; any page size. A token whose position lies outside the
    table's row, or on a page number outside the pool, is not stored (its query row is rotated all the same); rows from
    cu_q[B] on are not touched. Two tokens of one call must not share a place: a page that two sequences share is
    written by neither."""
    op = "paged_append"
    dev = _device(key, value, k_pages, v_pages, block_table, kv_lens, query, cu_q, query_out)
    k_st, v_st = _tokens(op, "key", key, cu_q), _tokens(op, "value", value, cu_q)
    B, T, Sq = _batch(op, key, cu_q)
    (n_pages, page, Hkv, D), width, pool_st = _cache(op, k_pages, v_pages, block_table, kv_lens, cu_q, B)
    shape, dtype = key.shape, key.dtype
    if value.shape != shape or shape[-2] != Hkv or shape[-1] != D:
        raise RuntimeError(f"{op}: key {tuple(shape)} and value {tuple(value.shape)} do not match pages of {Hkv} heads "
                           f"of {D}")
    if value.dtype is not dtype or k_pages.dtype is not dtype:
        raise RuntimeError(f"{op}: key, value and page dtypes differ")
    if rope_theta is not None and not rope_theta > 0:
        raise RuntimeError(f"{op}: rope_theta must be > 0 (got {rope_theta})")
    Hq, q_st, o_st, q_ptr, o_ptr = 0, (0, 0, 0), (0, 0, 0), None, None
    if query is not None:
        if rope_theta is None:
            raise RuntimeError(f"{op}: a query is taken to be rotated: give rope_theta")
        q_st = _tokens(op, "query", query, cu_q)
        q_shape = query.shape
        if q_shape[:-2] != shape[:-2] or q_shape[-1] != D or query.dtype is not dtype:
            raise RuntimeError(f"{op}: query {tuple(q_shape)} {query.dtype} does not match key {tuple(shape)} {dtype}")
        if query_out is None:
            query_out = torch.empty_like(query)
        elif query_out.shape != q_shape or query_out.dtype is not dtype:
            raise RuntimeError(f"{op}: query_out must match query in shape and dtype")
        o_st = _tokens(op, "query_out", query_out, cu_q)
        Hq, q_ptr, o_ptr = q_shape[-2], query.data_ptr(), query_out.data_ptr()
    elif query_out is not None:
        raise RuntimeError(f"{op}: query_out without a query")
    strides = _STRIDES_19.pack(*q_st, *k_st, *v_st, *o_st, *pool_st, block_table.stride(0))
    _launch(dev, "dgg_paged_append", q_ptr, key.data_ptr(), value.data_ptr(), o_ptr, k_pages.data_ptr(),
              v_pages.data_ptr(), block_table.data_ptr(), kv_lens.data_ptr(), _lib.ptr(cu_q), B, T, Sq, Hq, Hkv, D,
              n_pages, page, width, strides, rope_theta or 0.0, _lib.dtype_code(dtype))
    return query_out


def _attend(op: str, q, k_pages, v_pages, block_table, kv_lens, prefix_len, cu_q, causal, softcap, window, scale,
            return_lse, out):
    dev = _device(q, k_pages, v_pages, block_table, kv_lens, cu_q, out)
    q_st = _tokens(op, "q", q, cu_q)
    B, T, Sq = _batch(op, q, cu_q)
    (n_pages, page, Hkv, D), width, pool_st = _cache(op, k_pages, v_pages, block_table, kv_lens, cu_q, B)
    shape, dtype = q.shape, q.dtype
    Hq = shape[-2]
    if shape[-1] != D or dtype is not k_pages.dtype:
        raise RuntimeError(f"{op}: q {tuple(shape)} {dtype} does not match pages {tuple(k_pages.shape)} {k_pages.dtype}")
    if out is None:
        out = torch.empty_like(q)
    elif out.shape != shape or out.dtype is not dtype:
        raise RuntimeError(f"{op}: out must match q in shape and dtype")
    o_st = _tokens(op, "out", out, cu_q)
    ws_bytes = _workspace_bytes(op, B, T, Sq, Hq, Hkv, D, prefix_len)
    ws = q.new_empty(ws_bytes // 2 + 8)  # (of 16-bit elements; another type is refused below)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=q.device) if return_lse else None
    strides = _STRIDES_13.pack(*q_st, *pool_st, *o_st, block_table.stride(0))
    _launch(dev, "dgg_attn_paged", q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr(), _lib.ptr(lse),
              block_table.data_ptr(), kv_lens.data_ptr(), _lib.ptr(cu_q), ws.data_ptr(), ws_bytes, B, T, Sq, Hq, Hkv, D,
              n_pages, page, width, prefix_len, strides, 1.0 / math.sqrt(D) if scale is None else scale, softcap or 0.0,
              window or 0, _lib.ATTN_CAUSAL if causal else 0, _lib.dtype_code(dtype))
    if not return_lse:
        return out
    return out, lse if cu_q is not None else lse.view(B, Sq, Hq).transpose(1, 2)


def paged_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                    kv_lens: torch.Tensor, *, cu_q: torch.Tensor | None = None, causal: bool = True,
                    softcap: float = 0.0, window: int = 0, scale: float | None = None, return_lse: bool = False,
                    out: torch.Tensor | None = None):
    """attention() of every sequence's query rows over its own pages: q [B, Sq, Hq, D] (or [T, Hq, D] with cu_q) ->
    out of q's shape and, with return_lse, the natural-log lse, fp32 [B, Hq, Sq] ([T, Hq] with cu_q). Decode rows, drafted
    tokens and prompt chunks of any lengths go into one call; scores, bottom-right causal mask (query i of a sequence's n
    sees keys up to kv_lens[b] - n + i), soft-cap, window and grouped heads as attention() has them.

    float16 and bfloat16, D 64, 128 or 256, page sizes that are multiples of 16, up to 4,096 sequences. A kv_lens beyond
    the table's row is taken as what that row can name, and keys on a page number outside the pool are not seen (a window's
    pages may be given back by writing -1 into the table). A row that sees no key gets 0 and lse -inf; rows from cu_q[B]
    on are not written. out may be q itself. Memory behind a sequence's last key may hold anything, NaN included."""
    return _attend("paged_attention", q, k_pages, v_pages, block_table, kv_lens, 0, cu_q, causal, softcap, window, scale,
                   return_lse, out)


def shared_prefix_attention(q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, block_table: torch.Tensor,
                            kv_lens: torch.Tensor, prefix_len: int, *, cu_q: torch.Tensor | None = None,
                            causal: bool = True, softcap: float = 0.0, window: int = 0, scale: float | None = None,
                            return_lse: bool = False, out: torch.Tensor | None = None):
    """paged_attention() for a batch whose sequences begin with the same prefix_len keys (a system prompt, a document, the
    branches of a search): the prefix is read once for all rows of the batch, as the keys of sequence 0 (the other rows
    of block_table are not looked at there), the rest of each sequence from its own pages, and the two are joined
    by their log-sum-exp. prefix_len is a number of whole pages; kv_lens and positions count the prefix. Results and other
    arguments as paged_attention(), which computes the same from tables that repeat the prefix's pages."""
    return _attend("shared_prefix_attention", q, k_pages, v_pages, block_table, kv_lens, int(prefix_len), cu_q, causal,
                   softcap, window, scale, return_lse, out)
