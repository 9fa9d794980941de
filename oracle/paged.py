"""The paged-cache operators in 64 bits on the CPU — TEST INFRASTRUCTURE ONLY (see oracle/__init__.py). Plain loops over
sequences and heads, from the definitions in include/dgg.h; no counterpart in the reference."""
from __future__ import annotations

import math

import torch


def spans(kv_lens, cu_q, B, Sq):
    """(first token, tokens, keys) of every sequence."""
    cu = [b * Sq for b in range(B + 1)] if cu_q is None else [int(x) for x in cu_q]
    return [(cu[b], cu[b + 1] - cu[b], int(kv_lens[b])) for b in range(B)]


def rotate(x, pos, theta):
    """x [n, heads, D] rotated by positions pos [n], NeoX pairs."""
    D = x.shape[-1]
    ang = pos.double()[:, None, None] * theta ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], dim=-1)


def append(key, value, k_pages, v_pages, table, kv_lens, *, query=None, cu_q=None, rope_theta=None):
    """The pools after the call and the rotated query, float64 (query rows of no sequence: as given)."""
    B = table.shape[0]
    Sq = 0 if cu_q is not None else key.shape[1]
    k, v = (t.reshape(-1, *t.shape[-2:]).double() for t in (key, value))
    q = query.reshape(-1, *query.shape[-2:]).double().clone() if query is not None else None
    kp, vp = k_pages.double().clone(), v_pages.double().clone()
    n_pages, page = kp.shape[:2]
    for b, (t0, n, kv) in enumerate(spans(kv_lens, cu_q, B, Sq)):
        pos = torch.arange(kv - n, kv)
        kr = rotate(k[t0:t0 + n], pos, rope_theta) if rope_theta else k[t0:t0 + n]
        if q is not None:
            q[t0:t0 + n] = rotate(q[t0:t0 + n], pos, rope_theta)
        for i in range(n):
            j = kv - n + i
            if 0 <= j < table.shape[1] * page and 0 <= int(table[b, j // page]) < n_pages:
                kp[int(table[b, j // page]), j % page] = kr[i]
                vp[int(table[b, j // page]), j % page] = v[t0 + i]
    return kp, vp, (q.view(query.shape) if q is not None else None)


def attention(q, k_pages, v_pages, table, kv_lens, *, cu_q=None, prefix_len=0, causal=True, softcap=0.0, window=0,
              scale=None):
    """(out, lse, spread, slack) in float64, [T, Hq, D] / [T, Hq]: spread = sum_j p |v| of each output and slack a bound
    on the relative error that 32-bit scores leave in a probability, for tolerances. Rows of no sequence are NaN."""
    B = table.shape[0]
    Sq = 0 if cu_q is not None else q.shape[1]
    qf = q.reshape(-1, *q.shape[-2:]).double()
    T, Hq, D = qf.shape
    n_pages, page, Hkv, _ = k_pages.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((T, Hq, D), math.nan, dtype=torch.float64)
    spread, lse, slack = out.clone(), out[..., 0].clone(), out[..., 0].clone()
    for b, (t0, n, kv) in enumerate(spans(kv_lens, cu_q, B, Sq)):
        kv = min(max(kv, 0), table.shape[1] * page)
        j = torch.arange(kv)
        ids = torch.where(j < prefix_len, table[0].long()[j // page], table[b].long()[j // page])
        real = (ids >= 0) & (ids < n_pages)
        ids = ids.clamp(0, max(n_pages - 1, 0))
        i = torch.arange(n)[:, None] + kv - n
        seen = real[None].expand(n, kv).clone()
        if causal:
            seen &= j[None] <= i
        if window:
            seen &= i - j[None] < window
        used = seen.any(0)  # the others' memory may hold anything
        for h in range(Hq):
            kh = k_pages[ids, j % page, h // (Hq // Hkv)].double()
            vh = v_pages[ids, j % page, h // (Hq // Hkv)].double()
            kh[~used] = 0
            vh[~used] = 0
            x = qf[t0:t0 + n, h] @ kh.T * scale
            mag = (qf[t0:t0 + n, h].abs() @ kh.abs().T * scale).amax(-1) if kv else torch.zeros(n, dtype=torch.float64)
            if softcap:
                x = softcap * torch.tanh(x / softcap)
            x = x.masked_fill(~seen, -math.inf)
            ls = torch.logsumexp(x, -1) if kv else torch.full((n,), -math.inf, dtype=torch.float64)
            p = torch.exp(x - torch.where(ls.isinf(), torch.zeros_like(ls), ls)[:, None])
            out[t0:t0 + n, h] = p @ vh
            spread[t0:t0 + n, h] = p @ vh.abs()
            lse[t0:t0 + n, h] = ls
            # a dot product of D terms in fp32 is off by at most (D + 2) 2^-24 of the sum of its terms' magnitudes; the
            # soft-cap's exponential and reciprocal by a few 2^-23 of the cap; twice, for the row's sum is off as well
            slack[t0:t0 + n, h] = 2 * ((D + 2) * 2.0 ** -24 * mag + 8 * softcap * 2.0 ** -23) + 2.0 ** -18
    return out, lse, spread, slack
