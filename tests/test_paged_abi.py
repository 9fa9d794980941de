"""Refusals of the paged-cache entry points, on the CPU: each bad argument returns its documented status before anything
is launched, so none of these calls touches a device. And the oracle of the GPU tests against a second form."""
import ctypes
import math

import pytest
import torch

from deepgengraph_amd import _lib
from oracle import attention as oa
from oracle import paged as op

OK, E_DTYPE, E_SHAPE, E_STRIDE, E_ALIGN, E_UNSUP, E_LAUNCH, E_NULL, E_WS = 0, -1, -2, -3, -4, -5, -6, -7, -8
FAKE = ctypes.c_void_p(0x10000)  # 16-byte aligned, never dereferenced: validation fails first
MIS = ctypes.c_void_p(0x10002)


@pytest.fixture(scope="module")
def lib():
    if not _lib.LIB_PATH.exists():
        from deepgengraph_amd import build

        build.build()
    return _lib.load()


def _attn(lib, strides=None, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, o=FAKE, lse=None, table=FAKE, lens=FAKE, cu=None, ws=FAKE, ws_bytes=1 << 40, B=2, T=2,
             Sq=1, Hq=4, Hkv=2, D=128, pages=8, page=16, width=4, prefix=0, scale=0.1, softcap=0.0, window=0, flags=1,
             dtype=_lib.DGG_BF16)
    a.update(kw)
    st = _lib.int64_array(strides or [512, 512, 128, 4096, 256, 128, 4096, 256, 128, 512, 512, 128, 4])
    return lib.dgg_attn_paged(a["q"], a["k"], a["v"], a["o"], a["lse"], a["table"], a["lens"], a["cu"], a["ws"],
                              a["ws_bytes"], a["B"], a["T"], a["Sq"], a["Hq"], a["Hkv"], a["D"], a["pages"], a["page"],
                              a["width"], a["prefix"], None if strides == [] else st, a["scale"], a["softcap"],
                              a["window"], a["flags"], a["dtype"], None)


def test_attention_refusals(lib):
    assert _attn(lib, dtype=_lib.DGG_F32) == E_DTYPE
    assert _attn(lib, dtype=9) == E_DTYPE
    assert _attn(lib, B=-1) == E_SHAPE
    assert _attn(lib, B=5000, T=5000) == E_SHAPE
    assert b"4096" in lib.dgg_last_error()
    assert _attn(lib, T=3) == E_SHAPE
    assert _attn(lib, T=1 << 24, Sq=1 << 23) == E_SHAPE
    assert _attn(lib, cu=FAKE) == E_SHAPE  # both Sq and cu_q
    assert _attn(lib, Sq=0) == E_SHAPE     # neither
    assert _attn(lib, Hq=3) == E_SHAPE
    assert _attn(lib, Hkv=0) == E_SHAPE
    assert _attn(lib, D=96) == E_UNSUP
    assert _attn(lib, pages=-1) == E_SHAPE
    assert _attn(lib, page=8) == E_SHAPE
    assert _attn(lib, page=0) == E_SHAPE
    assert _attn(lib, width=-1) == E_SHAPE
    assert _attn(lib, width=1 << 30) == E_SHAPE
    assert _attn(lib, prefix=8) == E_SHAPE
    assert _attn(lib, prefix=-16) == E_SHAPE
    assert _attn(lib, prefix=80) == E_SHAPE
    assert _attn(lib, scale=0.0) == E_SHAPE
    assert _attn(lib, scale=math.nan) == E_SHAPE
    assert _attn(lib, softcap=-1.0) == E_SHAPE
    assert _attn(lib, window=-1) == E_SHAPE
    assert _attn(lib, flags=_lib.ATTN_REF_ROUNDING) == E_UNSUP
    assert _attn(lib, strides=[512, 512, 128, 4096, 256, 4, 4096, 256, 128, 512, 512, 128, 4]) == E_STRIDE
    assert _attn(lib, strides=[512, 512, 128, 4096, 256, 128, 4096, 256, 128, 512, 512, 128, -4]) == E_STRIDE
    for name in ("q", "k", "v", "o", "table", "lens", "ws"):
        assert _attn(lib, **{name: None}) == E_NULL, name
    for name in ("q", "k", "v", "o", "ws"):
        assert _attn(lib, **{name: MIS}) == E_ALIGN, name
    need = lib.dgg_attn_paged_workspace_bytes(2, 2, 1, 4, 2, 128, 0)
    assert need > 0 and _attn(lib, ws_bytes=need - 1) == E_WS
    assert lib.dgg_attn_paged_workspace_bytes(2, 3, 1, 4, 2, 128, 0) == -1
    assert lib.dgg_attn_paged_workspace_bytes(0, 0, 0, 4, 2, 128, 0) == 0
    assert _attn(lib, B=0, T=0, q=None) == OK


def _append(lib, strides=None, **kw):
    a = dict(q=FAKE, k=FAKE, v=FAKE, qo=FAKE, kp=FAKE, vp=FAKE, table=FAKE, lens=FAKE, cu=None, B=2, T=2, Sq=1, Hq=4, Hkv=2,
             D=128, pages=8, page=16, width=4, theta=1e4, dtype=_lib.DGG_BF16)
    a.update(kw)
    st = _lib.int64_array(strides or [512, 512, 128] * 4 + [4096, 256, 128] * 2 + [4])
    return lib.dgg_paged_append(a["q"], a["k"], a["v"], a["qo"], a["kp"], a["vp"], a["table"], a["lens"], a["cu"], a["B"],
                                a["T"], a["Sq"], a["Hq"], a["Hkv"], a["D"], a["pages"], a["page"], a["width"], st,
                                a["theta"], a["dtype"], None)


def test_append_refusals(lib):
    assert _append(lib, dtype=9) == E_DTYPE
    assert _append(lib, T=3) == E_SHAPE
    assert _append(lib, B=-1) == E_SHAPE
    assert _append(lib, T=1 << 24, Sq=1 << 23) == E_SHAPE
    assert _append(lib, cu=FAKE) == E_SHAPE
    assert _append(lib, Sq=0) == E_SHAPE
    assert _append(lib, Hkv=0) == E_SHAPE
    assert _append(lib, Hq=-1) == E_SHAPE
    assert _append(lib, D=24) == E_UNSUP
    assert _append(lib, D=1024) == E_UNSUP
    assert _append(lib, pages=-1) == E_SHAPE
    assert _append(lib, page=0) == E_SHAPE
    assert _append(lib, width=1 << 31) == E_SHAPE
    assert _append(lib, theta=-1.0) == E_SHAPE
    assert _append(lib, theta=math.inf) == E_SHAPE
    assert _append(lib, theta=0.0) == E_SHAPE  # a query, but no rotation
    assert _append(lib, strides=[512, 512, 4] * 4 + [4096, 256, 128] * 2 + [4]) == E_STRIDE
    assert _append(lib, strides=[512, 512, 128] * 4 + [4096, 256, 128] * 2 + [-4]) == E_STRIDE
    for name in ("q", "k", "v", "qo", "kp", "vp", "table", "lens"):
        assert _append(lib, **{name: None}) == E_NULL, name
    for name in ("q", "k", "v", "qo", "kp", "vp"):
        assert _append(lib, **{name: MIS}) == E_ALIGN, name
    assert _append(lib, B=0, T=0, q=None) == OK


def test_sizes_whose_products_pass_64_bits(lib):
    # the products of the checks wrap around to sizes that would be right
    for f in (_attn, _append):
        assert f(lib, B=4096, T=4096, Sq=(1 << 52) + 1) == E_SHAPE
        assert f(lib, width=1 << 60) == E_SHAPE
        assert f(lib, width=(1 << 60) + 4) == E_SHAPE
    assert lib.dgg_attn_paged_workspace_bytes(4096, 4096, (1 << 52) + 1, 4, 2, 128, 0) == -1


def test_oracle_against_the_contiguous_one():
    """The paged oracle over pages in order is the contiguous oracle's attention of each sequence."""
    g = torch.Generator().manual_seed(0)
    q, kv = torch.randn(2, 3, 4, 16, generator=g), [19, 32]
    kp, vp = (torch.randn(4, 16, 2, 16, generator=g) for _ in range(2))
    table = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)
    for opt in (dict(), dict(window=5), dict(softcap=2.0)):
        out, lse, _, _ = op.attention(q, kp, vp, table, kv, **opt)
        for b, n in enumerate(kv):
            k, v = (t[2 * b: 2 * b + 2].reshape(1, 32, 2, 16)[:, :n] for t in (kp, vp))
            ref, rl = oa.attention(q[b: b + 1], k, v, return_lse=True, **opt)
            assert torch.allclose(out[3 * b: 3 * b + 3], ref[0].double(), atol=2e-6)
            assert torch.allclose(lse[3 * b: 3 * b + 3], rl[0].t().double(), atol=2e-6)


def test_oracle_append():
    """Rotation keeps lengths and turns the product of two rotated rows with their distance; rows land in their pages."""
    g = torch.Generator().manual_seed(1)
    kp = torch.zeros(3, 16, 1, 8)
    table = torch.tensor([[2, 0]], dtype=torch.int32)
    k = torch.randn(1, 4, 1, 8, generator=g)
    a, v, _ = op.append(k, k, kp, kp, table, [18], rope_theta=100.0)
    for i, pos in enumerate(range(14, 18)):
        row = a[int(table[0, pos // 16]), pos % 16, 0]
        assert torch.allclose(row.norm(), k[0, i, 0].double().norm())
        assert torch.equal(v[int(table[0, pos // 16]), pos % 16, 0], k[0, i, 0].double())
    one = torch.ones(1, 1, 1, 8)
    x, y = (op.rotate(one[0], torch.tensor([p]), 100.0)[0, 0] for p in (5, 12))
    z, w = (op.rotate(one[0], torch.tensor([p]), 100.0)[0, 0] for p in (905, 912))
    assert torch.allclose(x @ y, z @ w)
    assert int((a != 0).any(-1).sum()) == 4
