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

import math

import torch

from . import _lib
from .attention import _check_bshd


def _tokens(name: str, t: torch.Tensor, cu_q):
    """(B, T, Sq, [batch, token, head] strides) of a step's tokens; Sq 0 with cu_q."""
    st = t.stride()
    if t.dim() != (4 if cu_q is None else 3):
        raise RuntimeError(f"{name}: expected {'[B, Sq, heads, D]' if cu_q is None else '[T, heads, D] with cu_q'}, got "
                           f"shape {tuple(t.shape)}")
    if st[-1] != 1:
        raise RuntimeError(f"{name}: head dimension must be contiguous (stride {st[-1]})")
    if cu_q is None:
        return t.shape[0], t.shape[0] * t.shape[1], t.shape[1], st[:3]
    return cu_q.shape[0] - 1, t.shape[0], 0, (0, st[0], st[1])


def _cache(op: str, k_pages, v_pages, block_table, kv_lens, cu_q, B: int):
    """Checks of the pools, the table and the lengths."""
    _check_bshd("k_pages", k_pages)
    _check_bshd("v_pages", v_pages)
    if v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype:
        raise RuntimeError(f"{op}: k_pages {tuple(k_pages.shape)} {k_pages.dtype} and v_pages {tuple(v_pages.shape)} "
                           f"{v_pages.dtype} differ")
    if block_table.dtype != torch.int32 or block_table.dim() != 2 or block_table.shape[0] != B or (
            block_table.shape[1] > 1 and block_table.stride(1) != 1):
        raise RuntimeError(f"{op}: block_table must be int32 [{B}, width] with unit column stride")
    if kv_lens.dtype != torch.int32 or kv_lens.shape != (B,) or not kv_lens.is_contiguous():
        raise RuntimeError(f"{op}: kv_lens must be contiguous int32 [{B}]")


def _check_cu(op: str, cu_q):
    if cu_q is not None and (cu_q.dtype != torch.int32 or cu_q.dim() != 1 or cu_q.shape[0] < 1
                             or not cu_q.is_contiguous()):
        raise RuntimeError(f"{op}: cu_q must be contiguous int32 [B + 1]")


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
    dev = _lib.require_gpu(key, value, k_pages, v_pages, block_table, kv_lens, query, cu_q, query_out)
    _check_cu(op, cu_q)
    B, T, Sq, k_st = _tokens("key", key, cu_q)
    _, _, _, v_st = _tokens("value", value, cu_q)
    _cache(op, k_pages, v_pages, block_table, kv_lens, cu_q, B)
    n_pages, page, Hkv, D = k_pages.shape
    if value.shape != key.shape or tuple(key.shape[-2:]) != (Hkv, D):
        raise RuntimeError(f"{op}: key {tuple(key.shape)} and value {tuple(value.shape)} do not match pages of "
                           f"{Hkv} heads of {D}")
    if not (key.dtype == value.dtype == k_pages.dtype):
        raise RuntimeError(f"{op}: key, value and page dtypes differ")
    Hq, q_st, o_st = 0, (0, 0, 0), (0, 0, 0)
    if query is not None:
        if rope_theta is None:
            raise RuntimeError(f"{op}: a query is taken to be rotated: give rope_theta")
        _, _, _, q_st = _tokens("query", query, cu_q)
        if query.shape[:-2] != key.shape[:-2] or query.shape[-1] != D or query.dtype != key.dtype:
            raise RuntimeError(f"{op}: query {tuple(query.shape)} {query.dtype} does not match key {tuple(key.shape)}")
        if query_out is None:
            query_out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        elif query_out.shape != query.shape or query_out.dtype != query.dtype:
            raise RuntimeError(f"{op}: query_out must match query in shape and dtype")
        _, _, _, o_st = _tokens("query_out", query_out, cu_q)
        Hq = query.shape[-2]
    elif query_out is not None:
        raise RuntimeError(f"{op}: query_out without a query")
    if rope_theta is not None and not rope_theta > 0:
        raise RuntimeError(f"{op}: rope_theta must be > 0 (got {rope_theta})")
    strides = _lib.int64_array([*q_st, *k_st, *v_st, *o_st, *k_pages.stride()[:3], *v_pages.stride()[:3],
                                block_table.stride(0)])
    _lib.call("dgg_paged_append", _lib.ptr(query), _lib.ptr(key), _lib.ptr(value), _lib.ptr(query_out),
              _lib.ptr(k_pages), _lib.ptr(v_pages), _lib.ptr(block_table), _lib.ptr(kv_lens), _lib.ptr(cu_q), B, T, Sq,
              Hq, Hkv, D, n_pages, page, block_table.shape[1], strides, float(rope_theta or 0.0),
              _lib.dtype_code(key.dtype), _lib.stream_handle(dev))
    return query_out


def _attend(op: str, q, k_pages, v_pages, block_table, kv_lens, prefix_len, cu_q, causal, softcap, window, scale,
            return_lse, out):
    dev = _lib.require_gpu(q, k_pages, v_pages, block_table, kv_lens, cu_q, out)
    _check_cu(op, cu_q)
    B, T, Sq, q_st = _tokens("q", q, cu_q)
    _cache(op, k_pages, v_pages, block_table, kv_lens, cu_q, B)
    n_pages, page, Hkv, D = k_pages.shape
    Hq = q.shape[-2]
    if q.shape[-1] != D or q.dtype != k_pages.dtype:
        raise RuntimeError(f"{op}: q {tuple(q.shape)} {q.dtype} does not match pages {tuple(k_pages.shape)} "
                           f"{k_pages.dtype}")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype:
        raise RuntimeError(f"{op}: out must match q in shape and dtype")
    _, _, _, o_st = _tokens("out", out, cu_q)
    scale = 1.0 / math.sqrt(D) if scale is None else float(scale)
    need = _lib.load().dgg_attn_paged_workspace_bytes(B, T, Sq, Hq, Hkv, D, int(prefix_len))
    if need < 0:
        raise RuntimeError(f"{op}: {_lib.load().dgg_last_error().decode(errors='replace')}")
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    lse = torch.empty(T, Hq, dtype=torch.float32, device=q.device) if return_lse else None
    strides = _lib.int64_array([*q_st, *k_pages.stride()[:3], *v_pages.stride()[:3], *o_st, block_table.stride(0)])
    _lib.call("dgg_attn_paged", _lib.ptr(q), _lib.ptr(k_pages), _lib.ptr(v_pages), _lib.ptr(out), _lib.ptr(lse),
              _lib.ptr(block_table), _lib.ptr(kv_lens), _lib.ptr(cu_q), _lib.ptr(ws), ws.numel(), B, T, Sq, Hq, Hkv, D,
              n_pages, page, block_table.shape[1], int(prefix_len), strides, scale, float(softcap or 0.0),
              int(window or 0), _lib.ATTN_CAUSAL if causal else 0, _lib.dtype_code(q.dtype), _lib.stream_handle(dev))
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
    on are not written. Memory behind a sequence's last key may hold anything, NaN included."""
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
    prefix_len, page = int(prefix_len), k_pages.shape[1] if k_pages.dim() == 4 else 1
    if prefix_len < 0 or prefix_len % max(page, 1) or prefix_len > block_table.shape[-1] * page:
        raise RuntimeError(f"shared_prefix_attention: prefix_len {prefix_len} must be whole pages of {page} keys that the "
                           "block table names")
    return _attend("shared_prefix_attention", q, k_pages, v_pages, block_table, kv_lens, prefix_len, cu_q, causal,
                   softcap, window, scale, return_lse, out)
