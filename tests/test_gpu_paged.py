"""The paged cache on the GPU against 64-bit oracles: append with rotary, attention over pages, shared prefixes.

Tolerance of the attention, per element: the output is rounded once (u = eps / 2 of its type, relative), the
probabilities are rounded to the same type before the matrix instruction (u of sum p |v|), and the 32-bit scores leave a
relative error `slack` in them (oracle/paged.py): |err| <= u |o| + (u + slack) (1 + u) sum p |v|. The lse is 32-bit: slack
plus 2^-20 of its size."""
import math

import pytest
import torch

from deepgengraph_amd import paged
from oracle import paged as op

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _cache(g, kv_lens, page, Hkv, D, dtype, *, layout="row", extra_width=1, spare_pages=3, shared=0, garbage=math.nan):
    """Pools whose unused rows hold `garbage`, a table of scattered pages whose unused entries are no pages, on the CPU."""
    B, cap = len(kv_lens), max(list(kv_lens) + [1])
    width = -(-cap // page) + extra_width
    n = sum(-(-kv // page) for kv in kv_lens) + spare_pages
    order = torch.randperm(n, generator=g)
    table = torch.full((B, width), -7, dtype=torch.int32)
    table[:, 1::2] = 1 << 30
    kp, vp = (torch.full((n, page, Hkv, D), garbage, dtype=dtype) for _ in range(2))
    at = 0
    for b, kv in enumerate(kv_lens):
        for i in range(-(-kv // page)):
            if b > 0 and (i + 1) * page <= shared:
                table[b, i] = table[0, i]
                continue
            pg = int(order[at])
            at += 1
            table[b, i] = pg
            rows = min(page, kv - i * page)
            kp[pg, :rows] = torch.randn(rows, Hkv, D, generator=g).to(dtype)
            vp[pg, :rows] = torch.randn(rows, Hkv, D, generator=g).to(dtype)
    return kp, vp, table


def _to(gpu, kp, vp, table, kv_lens, layout="row"):
    if layout == "head":
        kd, vd = (t.transpose(1, 2).contiguous().to(gpu).transpose(1, 2) for t in (kp, vp))
    else:
        kd, vd = kp.to(gpu), vp.to(gpu)
    return kd, vd, table.to(gpu), torch.tensor(kv_lens, dtype=torch.int32, device=gpu)


def _check(out, lse, ref, what):
    ro, rl, spread, slack = ref
    u = torch.finfo(out.dtype).eps / 2
    o = out.reshape(ro.shape).double().cpu()
    live = ~rl.isnan()
    bound = u * ro.abs() + (u + slack[..., None]) * (1 + u) * spread + torch.finfo(out.dtype).tiny
    err = (o - ro).abs()
    assert torch.isfinite(o[live]).all(), f"{what}: not finite"
    worst = (err / bound)[live].max().item() if live.any() else 0.0
    assert worst <= 1, f"{what}: {worst:.2f} times the bound (err {err[live].max():.3e})"
    if lse is not None:
        ls = (lse if lse.dim() == 2 else lse.transpose(1, 2).reshape(rl.shape)).double().cpu()
        none = rl.isinf()
        assert torch.equal(ls[live & none], rl[live & none]), f"{what}: lse of rows without a key"
        e = (ls - rl).abs() - slack - rl.abs() * 2.0 ** -20
        assert (e[live & ~none] <= 0).all(), f"{what}: lse off by {(ls - rl).abs()[live & ~none].max():.3e}"


def _run(gpu, kv_lens, q_lens, *, page=16, Hq=4, Hkv=2, D=128, dtype=torch.bfloat16, seed=0, ragged=None, layout="row",
         prefix=0, tail=0, qscale=1.0, **kw):
    g = _gen(seed)
    B = len(kv_lens)
    ragged = len(set(q_lens)) > 1 if ragged is None else ragged
    kp, vp, table = _cache(g, kv_lens, page, Hkv, D, dtype, shared=prefix)
    T = sum(q_lens) + tail
    q = (torch.randn(T, Hq, D, generator=g) * qscale).to(dtype)
    cu = None
    if ragged:
        cu = torch.tensor([sum(q_lens[:b]) for b in range(B + 1)], dtype=torch.int32)
    else:
        q = q.view(B, q_lens[0], Hq, D)
    kd, vd, td, ld = _to(gpu, kp, vp, table, kv_lens, layout)
    cud = cu.to(gpu) if cu is not None else None
    f = paged.paged_attention if not prefix else lambda *a, **k: paged.shared_prefix_attention(*a, prefix, **k)
    mark = torch.full(q.shape, 7.0, dtype=dtype, device=gpu)
    out, lse = f(q.to(gpu), kd, vd, td, ld, cu_q=cud, return_lse=True, out=mark, **kw)
    ref = op.attention(q, kp, vp, table, kv_lens, cu_q=cu, prefix_len=prefix, **kw)
    what = f"kv {kv_lens} q {q_lens} page {page} H {Hq}/{Hkv} D {D} {dtype} {layout} prefix {prefix} {kw}"
    _check(out, lse, ref, what)
    if tail:
        assert (out[sum(q_lens):] == 7.0).all(), what + ": rows behind the last sequence were written"
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (7, 1)])
def test_decode(gpu, dtype, D, heads):
    _run(gpu, [1, 31, 32, 33, 100, 517], [1] * 6, D=D, Hq=heads[0], Hkv=heads[1], dtype=dtype)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 256])
@pytest.mark.parametrize("layout", ["row", "head"])
def test_pages_and_layouts(gpu, page, layout):
    _run(gpu, [5, 255, 256, 257, 900], [1] * 5, page=page, layout=layout, seed=page)
    _run(gpu, [300, 47, 513], [17, 40, 129], page=page, layout=layout, seed=page + 1)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("heads", [(2, 2), (4, 1)])
def test_chunks(gpu, D, heads):
    # a prompt from its first token, a chunk behind keys, a single token, a sequence without tokens, one without keys
    _run(gpu, [150, 700, 333, 64, 0, 40], [150, 200, 1, 0, 0, 33], D=D, Hq=heads[0], Hkv=heads[1], tail=5)
    _run(gpu, [129, 300], [70, 70], D=D, Hq=heads[0], Hkv=heads[1], seed=3, dtype=torch.float16)


def test_rows_without_keys(gpu):
    # more tokens than keys: the first rows see nothing; a sequence of length zero; all of them
    _run(gpu, [3, 0, 20], [5, 5, 5])
    _run(gpu, [0, 0], [1, 1])
    _run(gpu, [0, 9, 0], [3, 2, 0], causal=False)


@pytest.mark.parametrize("kw", [dict(window=1), dict(window=33), dict(window=100, softcap=20.0), dict(softcap=5.0),
                                dict(causal=False), dict(causal=False, window=50), dict(scale=0.3),
                                dict(window=1 << 40)])
@pytest.mark.parametrize("D", [64, 256])
def test_options(gpu, kw, D):
    _run(gpu, [1, 95, 400, 33], [1, 1, 1, 1], D=D, **kw)
    _run(gpu, [130, 95, 400], [130, 1, 45], D=D, seed=1, **kw)


def test_large_scores(gpu):
    _run(gpu, [700, 40], [1, 1], qscale=60.0, dtype=torch.float16)


def test_long_and_uneven(gpu):
    # one long sequence among short ones: many slices for it, one for the others
    _run(gpu, [9001] + [17 + b for b in range(40)], [1] * 41, Hq=4, Hkv=1, D=64)
    _run(gpu, [5000, 20, 3], [64, 1, 3], Hq=4, Hkv=1, D=128)


def test_many_sequences(gpu):
    kv = [(b * 37) % 90 for b in range(150)]
    _run(gpu, kv, [1] * 150, Hq=2, Hkv=1, D=64)
    _run(gpu, kv, [min(k, b % 4) for b, k in enumerate(kv)], Hq=2, Hkv=1, D=64)
    _run(gpu, kv[:70], [1] * 70, Hq=2, Hkv=2, D=128, ragged=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_prefix(gpu, dtype, D):
    _run(gpu, [300, 257, 256 + 90, 500], [1] * 4, prefix=256, D=D, dtype=dtype)
    _run(gpu, [300, 290, 500], [20, 33, 1], prefix=256, D=D, dtype=dtype, Hq=4, Hkv=1, tail=2)


@pytest.mark.parametrize("page", [16, 48, 64])
def test_prefix_pages(gpu, page):
    _run(gpu, [page * 5 + 3, page * 5 + 1, page * 9], [1] * 3, prefix=page * 5, page=page)
    _run(gpu, [page * 5 + 30] * 40, [1] * 40, prefix=page * 5, page=page, Hq=4, Hkv=2, D=64)


def test_prefix_that_covers_everything(gpu):
    # sequences that end inside the prefix or with it, whose own part is empty, and padded ones
    _run(gpu, [256, 256, 100, 0], [1] * 4, prefix=256)
    _run(gpu, [256, 130, 0], [8, 8, 8], prefix=128, window=64)
    _run(gpu, [600, 540], [1, 1], prefix=512, window=40, softcap=10.0)
    _run(gpu, [600, 540], [30, 2], prefix=512, causal=False)


@pytest.mark.parametrize("heads", [(256, 256), (256, 128)])
def test_large_row_groups(gpu, heads):
    # chunks that fill the chip run in row groups of 256
    q = 256 * 256 // heads[1] * heads[1] // heads[0]
    _run(gpu, [q + 137], [q], Hq=heads[0], Hkv=heads[1], seed=heads[1])
    _run(gpu, [300, 129], [128, 128], Hq=heads[0], Hkv=heads[1], dtype=torch.float16, window=90)


def test_row_groups_cut_and_uncut(gpu):
    # uneven chunks whose row groups nearly fill the chip, so that only the longest are cut; and long ones among short
    _run(gpu, [130 * (b % 3 + 1) for b in range(24)], [100] * 24, Hq=8, Hkv=8, D=64)
    _run(gpu, [2000, 70, 65, 900], [65, 70, 65, 33], Hq=4, Hkv=1, D=256, dtype=torch.float16)
    _run(gpu, [40, 2100], [33, 34], Hq=2, Hkv=1)


def test_most_sequences(gpu):
    # the most that a call takes: each lane looks at 64 of them
    kv = [(b * 7) % 33 for b in range(4096)]
    _run(gpu, kv, [1] * 4096, Hq=1, Hkv=1, D=64)
    n = [0 if b % 5 == 1 else 1 + (b % 7 == 3) * 2 for b in range(1000)]
    n[500] = 60
    _run(gpu, [max(k, m) for k, m in zip(kv, n)], n, Hq=2, Hkv=1, D=64, ragged=True, tail=3)


def test_prefix_with_many_sequences(gpu):
    _run(gpu, [96 + b % 40 for b in range(130)], [1] * 130, prefix=96, Hq=2, Hkv=1, D=64)
    _run(gpu, [96 + b % 40 for b in range(130)], [b % 3 for b in range(130)], prefix=96, Hq=2, Hkv=2, D=64)


@pytest.mark.parametrize("D,heads", [(64, (48, 48)), (128, (160, 160)), (128, (8, 2)), (256, (32, 16))])
@pytest.mark.parametrize("P,more,kw", [(1024, [1, 2, 17], {}), (16, [500, 3, 700], {}), (512, [200, 300, 400], dict(window=90)),
                                       (512, [0, 0, 5], dict(window=600))])
def test_prefix_and_decode_rows(gpu, D, heads, P, more, kw):
    # nearly all keys in the prefix, nearly none, a prefix that no window reaches, sequences that hold nothing else; up
    # to as many heads as workgroups that are resident at once
    B = 34 if heads[0] == heads[1] else 18
    kv = [P + more[b % 3] for b in range(B)]
    _run(gpu, kv, [1] * B, Hq=heads[0], Hkv=heads[1], D=D, prefix=P, seed=D + P, **kw)
    if heads[0] > 100:
        return  # (the oracle takes its time)
    _run(gpu, kv, [1, 0] + [1] * (B - 2), Hq=heads[0], Hkv=heads[1], D=D, prefix=P, seed=D + P, tail=3, **kw)


def test_prefix_is_the_first_sequences(gpu):
    # the other rows of the table are not looked at inside the prefix
    g = _gen(5)
    kv = [200, 190, 170]
    kp, vp, table = _cache(g, kv, 16, 2, 64, torch.float16, shared=160)
    q = torch.randn(3, 1, 4, 64, generator=g).half()
    args = _to(gpu, kp, vp, table, kv)
    a = paged.shared_prefix_attention(q.to(gpu), *args, 160)
    t2 = table.clone()
    t2[1:, :10] = -1
    b = paged.shared_prefix_attention(q.to(gpu), args[0], args[1], t2.to(gpu), args[3], 160)
    assert torch.equal(a, b)


def test_holes_and_long_lengths(gpu):
    # page numbers outside the pool hide their keys; a kv_len beyond the table is the table's capacity
    g = _gen(6)
    kv = [300, 90, 64]
    for page in (16, 32):
        kp, vp, table = _cache(g, kv, page, 2, 128, torch.bfloat16, extra_width=0)
        table[0, 0], table[0, 3], table[0, 4], table[1, 1] = -1, 1 << 20, -5, -1
        table[2, :] = -1
        for q_len in (1, 40):
            q = torch.randn(3, q_len, 4, 128, generator=g).bfloat16()
            kd, vd, td, ld = _to(gpu, kp, vp, table, kv)
            out, lse = paged.paged_attention(q.to(gpu), kd, vd, td, ld, return_lse=True)
            _check(out, lse, op.attention(q, kp, vp, table, kv), f"holes page {page} q {q_len}")
    kp, vp, table = _cache(g, [96, 96], 16, 2, 128, torch.bfloat16, extra_width=0)
    q = torch.randn(2, 3, 4, 128, generator=g).bfloat16()
    kd, vd, td, ld = _to(gpu, kp, vp, table, [5000, 96])
    out, lse = paged.paged_attention(q.to(gpu), kd, vd, td, ld, return_lse=True)
    _check(out, lse, op.attention(q, kp, vp, table, [5000, 96]), "kv_len beyond the table")


@pytest.mark.parametrize("prefix", [0, 16])
def test_offsets_that_name_tokens_twice(gpu, prefix):
    # a cu_q that descends: more tokens than the call has; nothing is computed
    g = _gen(12)
    kv = [40, 33, 64, 20]
    kp, vp, table = _cache(g, kv, 16, 1, 64, torch.float16)
    args = _to(gpu, kp, vp, table, kv)
    q = torch.randn(48, 2, 64, generator=g).half().to(gpu)
    cu = torch.tensor([0, 48, 0, 48, 10], dtype=torch.int32, device=gpu)
    mark = torch.full_like(q, 7.0)
    kw = dict(cu_q=cu, out=mark)
    paged.shared_prefix_attention(q, *args, prefix, **kw) if prefix else paged.paged_attention(q, *args, **kw)
    assert (mark == 7.0).all()


def test_strided_inputs(gpu):
    # q as a slice of a projection, out with wider rows, a table that is part of a larger one
    g = _gen(8)
    kv = [70, 260]
    kp, vp, table = _cache(g, kv, 16, 2, 64, torch.float16)
    kd, vd, td, ld = _to(gpu, kp, vp, table, kv)
    qkv = torch.randn(2, 3, 8 * 64, generator=g).half()
    q = qkv[..., 64: 64 + 4 * 64].unflatten(-1, (4, 64))
    wide = torch.zeros(2, 3, 6, 64, dtype=torch.float16, device=gpu)
    big = torch.full((5, table.shape[1] + 9), -1, dtype=torch.int32, device=gpu)
    big[1:3, 4:4 + table.shape[1]] = td
    view = qkv.to(gpu)[..., 64: 64 + 4 * 64].unflatten(-1, (4, 64))
    out = paged.paged_attention(view, kd, vd, big[1:3, 4:4 + table.shape[1]], ld, out=wide[:, :, 1:5])
    _check(out, None, op.attention(q, kp, vp, table, kv), "strided")
    assert (wide[:, :, 0] == 0).all() and (wide[:, :, 5] == 0).all()
    # [Sq, B] order: tokens of a batch far apart
    q2 = torch.randn(3, 2, 4, 64, generator=g).half().transpose(0, 1)
    out = paged.paged_attention(q2.to(gpu), kd, vd, td, ld)
    _check(out, None, op.attention(q2, kp, vp, table, kv), "transposed tokens")


def test_far_offsets(gpu):
    # pages beyond 2^32 bytes of the pool
    page, Hkv, D = 256, 8, 128
    n = (1 << 32) // (page * Hkv * D * 2) + 40
    kd = torch.zeros(n, page, Hkv, D, dtype=torch.bfloat16, device=gpu)
    vd = torch.zeros_like(kd)
    g = _gen(9)
    kv = [700, 300]
    kp, vp, table = _cache(g, kv, page, Hkv, D, torch.bfloat16)
    far = torch.arange(n - kp.shape[0], n)
    kd[far], vd[far] = kp.to(gpu), vp.to(gpu)
    q = torch.randn(2, 1, 8, D, generator=g).bfloat16()
    td = torch.where((table >= 0) & (table < kp.shape[0]), table + (n - kp.shape[0]), table)
    ld = torch.tensor(kv, dtype=torch.int32, device=gpu)
    out = paged.paged_attention(q.to(gpu), kd, vd, td.to(gpu), ld)
    _check(out, None, op.attention(q, kp, vp, table, kv), "far pages")
    key, val = (torch.randn(2, 1, Hkv, D, generator=g).bfloat16() for _ in range(2))
    paged.paged_append(key.to(gpu), val.to(gpu), kd, vd, td.to(gpu), ld, rope_theta=1e4)
    rk, rv, _ = op.append(key, val, kp, vp, table, kv, rope_theta=1e4)
    _same_pool(kd[far], rk, 2 ** -8, "far append k")
    _same_pool(vd[far], rv, 0, "far append v")


def _same_pool(got, ref, u, what):
    # one rounding (u) of a value computed in 32 bits: x cos - y sin with errors of 2^-22 of |x| + |y| <= 16
    got = got.double().cpu()
    nan = ref.isnan()
    assert torch.equal(nan, got.isnan()), what + ": rows that were not to be written"
    bad = (got - ref).abs()[~nan] > u * ref.abs()[~nan] + (2.0 ** -22 * 16 if u else 0)
    assert not bad.any(), f"{what}: {int(bad.sum())} values off, {(got - ref).abs()[~nan].max():.3e}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("page,D,layout", [(16, 128, "row"), (1, 64, "row"), (24, 256, "head"), (64, 80, "head")])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("theta", [None, 10000.0])
def test_append(gpu, dtype, page, D, layout, ragged, theta):
    g = _gen(page + D)
    kv = [1, 40, 77, 300, 25]
    n = [1, 0, 33, 2, 25] if ragged else [1] * 5
    Hq, Hkv, B = 6, 2, 5
    kp, vp, table = _cache(g, kv, page, Hkv, D, dtype)
    T = sum(n) + (3 if ragged else 0)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(dtype)
    cu = torch.tensor([sum(n[:b]) for b in range(B + 1)], dtype=torch.int32) if ragged else None

    def split(t):
        t = t if ragged else t.view(B, 1, -1)
        return [x.unflatten(-1, (-1, D)) for x in t.split([Hq * D, Hkv * D, Hkv * D], dim=-1)]

    q, k, v = split(qkv)
    qd, kd_, vd_ = split(qkv.to(gpu))
    kd, vd, td, ld = _to(gpu, kp, vp, table, kv, layout)
    query = dict(query=qd) if theta else {}
    rot = paged.paged_append(kd_, vd_, kd, vd, td, ld, cu_q=cu.to(gpu) if ragged else None, rope_theta=theta, **query)
    rk, rv, rq = op.append(k, v, kp, vp, table, kv, query=q if theta else None, cu_q=cu, rope_theta=theta)
    u = torch.finfo(dtype).eps / 2
    _same_pool(kd, rk, u if theta else 0, "k pool")
    _same_pool(vd, rv, 0, "v pool")
    if theta:
        live = sum(n)
        _same_pool(rot.reshape(T, Hq, D)[:live], rq.reshape(T, Hq, D)[:live], u, "query")
        assert torch.equal(qkv.to(gpu)[:, :Hq * D].reshape(T, Hq, D), qd.reshape(T, Hq, D))  # left as it was
    else:
        assert rot is None


@pytest.mark.parametrize("T_per", [1, 300])
def test_append_far_positions(gpu, T_per):
    # a position of 130,000: 32-bit angles would be off by a hundredth of a radian
    g = _gen(4)
    page, Hkv, D, kv = 64, 2, 128, [130000, 1000]
    width = -(-kv[0] // page)
    table = torch.randperm(2 * width, generator=g).view(2, width).to(torch.int32)
    kp = torch.zeros(2 * width, page, Hkv, D)
    k, v = (torch.randn(2, T_per, Hkv, D, generator=g) for _ in range(2))
    q = torch.randn(2, T_per, 4, D, generator=g)
    kd, vd, td, ld = _to(gpu, kp, kp, table, kv)
    out = q.to(gpu)
    rot = paged.paged_append(k.to(gpu), v.to(gpu), kd, vd, td, ld, query=out, query_out=out, rope_theta=500000.0)
    assert rot is out
    rk, rv, rq = op.append(k, v, kp, kp, table, kv, query=q, rope_theta=500000.0)
    _same_pool(kd, rk, 2 ** -24, "k")
    _same_pool(vd, rv, 0, "v")
    _same_pool(rot, rq, 2 ** -24, "q in place")


def test_append_what_has_no_place(gpu):
    # positions before 0 or behind the table, and page numbers outside the pool: nothing is written for them
    g = _gen(11)
    kv, page, Hkv, D = [2, 50, 64, 40], 16, 1, 64
    kp, vp, table = _cache(g, kv, page, Hkv, D, torch.float16, extra_width=0)
    table[2, 3], table[3, 2] = -1, 1 << 20
    k, v = (torch.randn(4, 5, Hkv, D, generator=g).half() for _ in range(2))
    lens = [2, 66, 64, 40]  # sequence 1: two of the five positions lie behind the table
    kd, vd, td, ld = _to(gpu, kp, vp, table, lens)
    paged.paged_append(k.to(gpu), v.to(gpu), kd, vd, td, ld)
    rk, rv, _ = op.append(k, v, kp, vp, table, lens)
    _same_pool(kd, rk, 0, "k")
    _same_pool(vd, rv, 0, "v")


def test_refusals(gpu):
    g = _gen(1)
    kv = [40, 20]
    kp, vp, table = _cache(g, kv, 16, 2, 64, torch.float16)
    kd, vd, td, ld = _to(gpu, kp, vp, table, kv)
    q = torch.randn(2, 1, 4, 64, generator=g).half().to(gpu)
    k = torch.randn(2, 1, 2, 64, generator=g).half().to(gpu)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=gpu)
    at = paged.paged_attention

    def no(f, *a, **kw):
        with pytest.raises(RuntimeError):
            f(*a, **kw)

    no(at, q.cpu(), kd, vd, td, ld)
    no(at, q.float(), kd.float(), vd.float(), td, ld)
    no(at, q.bfloat16(), kd, vd, td, ld)
    no(at, q, kd, vd.float(), td, ld)
    no(at, q, kd, vd[:, :8], td, ld)
    no(at, q, kd, vd, td.long(), ld)
    no(at, q, kd, vd, td, ld.long())
    no(at, q, kd, vd, td[:1], ld)
    no(at, q, kd, vd, td.t(), ld)
    no(at, q[:, 0], kd, vd, td, ld)
    no(at, q, kd, vd, td, ld, cu_q=cu)
    no(at, q[:, 0], kd, vd, td, ld, cu_q=cu.long())
    no(at, q[..., :3, :], kd, vd, td, ld)
    no(at, q[..., ::2], kd[..., ::2], vd[..., ::2], td, ld)
    no(at, q[..., :32], kd[..., :32], vd[..., :32], td, ld)
    no(at, q, kd[:, :8], vd[:, :8], td, ld)
    no(at, q, kd, vd, td, ld, window=-1)
    no(at, q, kd, vd, td, ld, softcap=-1.0)
    no(at, q, kd, vd, td, ld, scale=0.0)
    no(at, q, kd, vd, td, ld, out=q.float())
    sh = paged.shared_prefix_attention
    no(sh, q, kd, vd, td, ld, 8)
    no(sh, q, kd, vd, td, ld, -16)
    no(sh, q, kd, vd, td, ld, 16 * (td.shape[1] + 1))
    ap = paged.paged_append
    no(ap, k, k.float(), kd, vd, td, ld)
    no(ap, k.float(), k.float(), kd, vd, td, ld)
    no(ap, k, k, kd, vd, td, ld, query=q)
    no(ap, k, k, kd, vd, td, ld, query=q[:1], rope_theta=1e4)
    no(ap, k, k, kd, vd, td, ld, rope_theta=-1.0)
    no(ap, k, k, kd, vd, td, ld, query_out=q)
    no(ap, q, q, kd, vd, td, ld)
    no(ap, k, k, kd, vd, td, ld, cu_q=cu)
    # nothing to do
    assert at(q[:0], kd, vd, td[:0], ld[:0]).shape == (0, 1, 4, 64)
    assert at(q[:, :0], kd, vd, td, ld).shape == (2, 0, 4, 64)
    # without pages nobody has a key
    assert (at(q, kd[:0], vd[:0], td, ld) == 0).all()


def test_two_streams(gpu):
    """Calls on two streams at once, each with a workspace of its own, give what they give one after the other."""
    g = _gen(31)
    kv = [700, 90, 1500, 33]
    kp, vp, table = _cache(g, kv, 16, 2, 128, torch.bfloat16)
    args = _to(gpu, kp, vp, table, kv)
    qs = [torch.randn(4, n, 8, 128, generator=g).bfloat16().to(gpu) for n in (1, 24)]
    want = [paged.paged_attention(q, *args) for q in qs]
    streams = [torch.cuda.Stream() for _ in qs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(paged.paged_attention(qs[i], *args))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("prefix", [0, 32])
def test_llama_block_over_a_paged_cache(gpu, prefix):
    """A prompt in uneven chunks, then decode steps, through the attention block: with the identity as its output
    projection the block returns the attention of the projected rows, which the 64-bit oracle computes from the same
    projections (the norm and the projection are the block's own, tested elsewhere)."""
    from deepgengraph_amd import llama, ops

    g = _gen(17)
    B, H, Hk, D, page, width = 3, 4, 2, 128, 16, 8
    hidden = H * D
    w_norm = (1 + 0.02 * torch.randn(hidden, generator=g)).bfloat16().to(gpu)
    w_qkv = (0.05 * torch.randn(hidden + 2 * Hk * D, hidden, generator=g)).bfloat16().to(gpu)
    block = llama.LlamaAttentionBlock(w_norm, w_qkv, torch.eye(hidden).bfloat16().to(gpu), heads=H, kv_heads=Hk)
    table = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32)
    if prefix:
        table[1:, : prefix // page] = table[0, : prefix // page]
    kp = torch.randn(B * width, page, Hk, D, generator=g).bfloat16()
    vp = torch.randn(B * width, page, Hk, D, generator=g).bfloat16()
    kd, vd, td = kp.to(gpu), vp.to(gpu), table.to(gpu)
    lens = [prefix] * B
    for n in ([20, 1, 33], [1, 30, 2], [1, 1, 1], [1, 1, 1]):
        lens = [a + b for a, b in zip(lens, n)]
        ld = torch.tensor(lens, dtype=torch.int32, device=gpu)
        same = len(set(n)) == 1
        cu = None if same else torch.tensor([0, n[0], n[0] + n[1], sum(n)], dtype=torch.int32)
        x = torch.randn(*((B, n[0]) if same else (sum(n),)), hidden, generator=g).bfloat16().to(gpu)
        y = block.paged_step(x, kd, vd, td, ld, cu_q=None if cu is None else cu.to(gpu), prefix_len=prefix)
        h = torch.empty_like(x)
        ops.rms_norm(h, x, w_norm, block.eps)
        q, k, v = (t.unflatten(-1, (-1, D)) for t in
                   torch.matmul(h, w_qkv.t()).cpu().split([hidden, Hk * D, Hk * D], dim=-1))
        rk, rv, rq = op.append(k, v, kp, vp, table, lens, query=q, cu_q=cu, rope_theta=1e4)
        _same_pool(kd, rk, 2 ** -8, f"keys {n}")
        _same_pool(vd, rv, 0, f"values {n}")
        kp, vp = kd.cpu(), vd.cpu()
        # the query that the attention saw (the same rows are stored once more)
        qd, kd2, vd2 = (t.to(gpu) for t in (q, k, v))
        seen = paged.paged_append(kd2, vd2, kd, vd, td, ld, query=qd, cu_q=None if cu is None else cu.to(gpu),
                                  rope_theta=1e4).cpu()
        _same_pool(seen, rq, 2 ** -8, f"queries {n}")
        ref = op.attention(seen, kp, vp, table, lens, cu_q=cu, prefix_len=prefix)
        _check(y.unflatten(-1, (H, D)), None, ref, f"step {n}")


@pytest.mark.parametrize("prefix", [0, 48])
@pytest.mark.parametrize("n,kv", [([1, 1, 1], [300, 60, 2000]), ([1, 150, 9], [300, 160, 2000]), ([70, 70], [500, 80])])
def test_output_over_the_query(gpu, n, kv, prefix):
    """The output may take the query's place: one unit, cut keys and a shared prefix give what they give elsewhere."""
    g = _gen(41)
    kp, vp, table = _cache(g, kv, 16, 2, 128, torch.bfloat16, shared=prefix)
    args = _to(gpu, kp, vp, table, kv)
    same = len(set(n)) == 1
    cu = None if same else torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32, device=gpu)
    q = torch.randn(*((len(n), n[0]) if same else (sum(n),)), 8, 128, generator=g).bfloat16().to(gpu)
    call = dict(cu_q=cu)
    f = paged.paged_attention if not prefix else lambda *a, **k: paged.shared_prefix_attention(*a, prefix, **k)
    want = f(q, *args, **call)
    assert f(q, *args, out=q, **call) is q
    assert torch.equal(q, want)


@pytest.mark.parametrize("D", [64, 128])
def test_ragged_batch_captured(gpu, D):
    """A batch of fixed capacity, captured once and replayed with other numbers of tokens per sequence: decode rows, chunks,
    sequences without tokens, all rows or few of them in use. Every replay against the eager calls and the oracle; rows
    behind the last sequence stay as they are."""
    g = _gen(43)
    B, T, Hq, Hkv, page, width, P = 5, 160, 8, 2, 16, 40, 32
    table = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32)
    table[1:, : P // page] = table[0, : P // page]
    kp, vp = (torch.randn(B * width, page, Hkv, D, generator=g).bfloat16() for _ in range(2))
    kd, vd, td = kp.to(gpu), vp.to(gpu), table.to(gpu)
    ld = torch.full((B,), 100, dtype=torch.int32, device=gpu)
    cu = torch.zeros(B + 1, dtype=torch.int32, device=gpu)
    q = torch.randn(T, Hq, D, generator=g).bfloat16().to(gpu)
    outs = [torch.zeros_like(q) for _ in range(2)]

    def step(o1, o2):
        return (paged.paged_attention(q, kd, vd, td, ld, cu_q=cu, return_lse=True, out=o1)[1],
                paged.shared_prefix_attention(q, kd, vd, td, ld, P, cu_q=cu, return_lse=True, out=o2)[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*outs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        lses = step(*outs)
    for r, (n, kv) in enumerate([([1, 1, 1, 1, 1], [640, 33, 200, 1, 90]), ([1, 150, 0, 8, 1], [300, 182, 77, 600, 0]),
                                 ([0, 0, 0, 0, 0], [50, 50, 50, 50, 50]), ([0, 0, 160, 0, 0], [40, 0, 640, 40, 40]),
                                 ([9, 1, 33, 70, 4], [41, 1, 65, 102, 640])]):
        cu.copy_(torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32))
        ld.copy_(torch.tensor(kv, dtype=torch.int32))
        q.copy_(torch.randn(q.shape, generator=g).bfloat16())
        for o in outs:
            o.fill_(7.0)
        graph.replay()
        eager = [torch.full_like(q, 7.0) for _ in range(2)]
        el = step(*eager)
        torch.cuda.synchronize()
        live = sum(n)
        want = op.attention(q.cpu(), kp, vp, table, kv, cu_q=cu.cpu())
        for i in range(2):
            assert torch.equal(outs[i], eager[i]), f"replay {r}: output {i}"
            assert torch.equal(lses[i][:live], el[i][:live]), f"replay {r}: lse {i}"
            assert (outs[i][live:] == 7.0).all(), f"replay {r}: rows behind the last sequence"
            _check(outs[i], lses[i], want, f"replay {r}, form {i}")


def test_step_together_captured(gpu):
    """Append and attention as a decode step, captured once and replayed with other lengths, tables and inputs, against the
    eager calls; another stream in between."""
    g = _gen(21)
    B, Hq, Hkv, D, page, width = 3, 4, 2, 64, 16, 20
    table = torch.randperm(B * width, generator=g).view(B, width).to(torch.int32)
    kp0, vp0 = (torch.randn(B * width, page, Hkv, D, generator=g).half() for _ in range(2))

    def step(qkv, kd, vd, td, ld):
        q, k, v = (x.unflatten(-1, (-1, D)) for x in qkv.split([Hq * D, Hkv * D, Hkv * D], dim=-1))
        q = paged.paged_append(k, v, kd, vd, td, ld, query=q, rope_theta=1e4)
        return (paged.paged_attention(q, kd, vd, td, ld, return_lse=True),
                paged.shared_prefix_attention(q, kd, vd, td, ld, 32))

    kd, vd, td = kp0.to(gpu), vp0.to(gpu), table.to(gpu)
    ld = torch.tensor([40, 33, 50], dtype=torch.int32, device=gpu)
    x = torch.zeros(B, 1, (Hq + 2 * Hkv) * D, dtype=torch.float16, device=gpu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, kd, vd, td, ld)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (o1, lse), o2 = step(x, kd, vd, td, ld)
    ke, ve = kp0.to(gpu), vp0.to(gpu)
    kd.copy_(ke), vd.copy_(ve)
    for r, lens in enumerate([[41, 34, 51], [300, 35, 0], [320, 33, 160], [42, 310, 52]]):
        x.copy_(torch.randn(x.shape, generator=g).half())
        ld.copy_(torch.tensor(lens, dtype=torch.int32))
        td.copy_(table[torch.randperm(B, generator=g)])
        graph.replay()
        (e1, el), e2 = step(x, ke, ve, td, ld)
        torch.cuda.synchronize()
        assert torch.equal(o1, e1) and torch.equal(o2, e2) and torch.equal(lse, el), f"replay {r}"
        assert torch.equal(kd, ke) and torch.equal(vd, ve), f"replay {r}: pages"
        want = op.attention(paged_q(x, ke, ve, td, ld, Hq, Hkv, D), ke.cpu(), ve.cpu(), td.cpu(), lens)
        _check(o1, lse, want, f"replay {r}")


def paged_q(x, kd, vd, td, ld, Hq, Hkv, D):
    """The step's rotated queries (the keys' places are written again with the same values)."""
    q, k, v = (t.unflatten(-1, (-1, D)) for t in x.split([Hq * D, Hkv * D, Hkv * D], dim=-1))
    return paged.paged_append(k, v, kd, vd, td, ld, query=q, rope_theta=1e4).cpu()
