"""The operators of a paged key/value cache, as measured work: appending rotated keys and values, attention over the
pages, and the same where a batch shares a long prefix (deepgengraph_amd.paged).

    listed()             the named cases
    draw(rng)            one more case of the same ranges
    prepare(case, seed)  what a serving program holds before the call, on the GPU
    run(state)           one pass; its outputs
    work(case)           bytes and operations one pass cannot do without
    exact(case, seed)    the outputs in 64 bits, in plain torch

`own` false: run() computes the operators from elementary torch operations in 32 bits. `own` true: it makes the calls
that a user makes.

A case is one layer of one step of a server. Its batch has B sequences; sequence b brings q_len[b] new tokens and then
holds kv_len[b] keys, the new ones included, in pages of `page` tokens that its row of the block table names. Fields:

    op        append, attention, prefix
    B, q      sequences, and new tokens per sequence (the most of them, where `mix` says that they differ)
    mix       same: every sequence brings q tokens ([B, q, heads, D] tensors)
              some: about one sequence in eight brings up to q tokens and the others one ([tokens, heads, D] tensors)
              all: every sequence brings its own number, up to q
    L, low    the longest sequence, and the shortest as a share of it (lengths are even over their logarithm)
    P         keys that all sequences share, in the pages of the first one (prefix)
    H, Hkv, D, page, dtype, softcap, window, theta, layout, lse, vary
              layout: row = pages [n, page, Hkv, D], head = pages [n, Hkv, page, D]; vary: draws the lengths
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}

_BASE = dict(q=1, mix="same", low=1.0, P=0, H=32, Hkv=8, D=128, page=16, dtype="bf16", softcap=0.0, window=0,
             theta=10000.0, layout="row", lse=False, vary=1)


def _case(**kw):
    return {**_BASE, **kw}


def listed():
    return [
        # A decode step of 64 users: one token each is rotated and stored. Small, so that launches and latency count.
        _case(name="append_step", op="append", B=64, L=32768, low=1 / 64),
        # Eight prompts of uneven length enter the cache: a copy of a few hundred megabytes.
        _case(name="append_prompts", op="append", B=8, q=2048, mix="all", L=4096, low=1 / 4, Hkv=32, page=64,
              dtype="f16"),
        # One user's chat: one row over one sequence of no round length. The smallest attention.
        _case(name="decode_one", op="attention", B=1, L=4001),
        # 64 users of very different lengths: a decode step bound by the reading of the cache.
        _case(name="decode_batch", op="attention", B=64, L=32768, low=1 / 64, dtype="f16", vary=2),
        # The same without grouped heads: four times the cache per key.
        _case(name="decode_mha", op="attention", B=16, L=8192, low=1 / 2, Hkv=32, page=64, vary=3),
        # Verification of drafted tokens: eight rows per sequence, with the log-sum-exp.
        _case(name="verify", op="attention", B=8, q=8, L=16384, low=1 / 8, page=32, lse=True, vary=4),
        # Gemma-2's attention: wide heads, soft-cap and a window that hides the start of the longer sequences.
        _case(name="decode_gemma2", op="attention", B=32, L=8192, low=1 / 16, H=16, Hkv=8, D=256, softcap=50.0,
              window=4096, layout="head", vary=5),
        # A mixed step: some prompts' chunks among the decode rows.
        _case(name="mixed_step", op="attention", B=32, q=512, mix="some", L=8192, low=1 / 16, page=64, vary=6),
        # Chunks of long prompts: bound by the matrix products.
        _case(name="prompt_chunk", op="attention", B=4, q=1024, L=8192, low=1 / 2, vary=7),
        # A decode step of 64 users behind one system prompt or document of 8K tokens.
        _case(name="prefix_step", op="prefix", B=64, P=8192, L=9216, low=8200 / 9216, vary=8),
        # The same without grouped heads behind a document of 32K.
        _case(name="prefix_mha", op="prefix", B=32, P=32768, L=33792, low=32832 / 33792, Hkv=32, page=64, dtype="f16",
              vary=9),
        # The users' questions themselves, all read against the document.
        _case(name="prefix_questions", op="prefix", B=16, q=64, mix="all", P=16384, L=16640, low=16448 / 16640,
              vary=10),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], evenly over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attention", "attention", "attention", "prefix", "prefix"])
    heads = rng.choice([(32, 8, 128), (32, 8, 128), (32, 32, 128), (16, 8, 256), (16, 16, 64), (12, 12, 64)])
    c = dict(op=op, H=heads[0], Hkv=heads[1], D=heads[2], page=rng.choice([16, 16, 32, 64, 128, 256]),
             dtype=rng.choice(["bf16", "f16"]), layout=rng.choice(["row", "row", "head"]), lse=rng.random() < 0.3,
             low=rng.choice([1.0, 1 / 2, 1 / 8, 1 / 64]), vary=rng.randrange(1 << 20))
    if op == "append":
        c["dtype"] = rng.choice(["bf16", "bf16", "f16", "f32"])
        c["lse"] = False
        c["B"] = _log(rng, 1, 128)
        c["mix"] = rng.choice(["same", "same", "all"])
        c["q"] = 1 if rng.random() < 0.4 else _log(rng, 2, max(2, min(2048, 8192 // c["B"])))
        c["L"] = max(c["q"], _log(rng, 64, 131072 * 1024 // max(1024, c["Hkv"] * c["D"])))
        c["theta"] = rng.choice([10000.0, 10000.0, 500000.0])
        return _case(**c)
    c["B"] = _log(rng, 1, 64)
    shape = rng.choice(["decode", "decode", "verify", "mixed", "prompt"])
    c["q"] = _log(rng, *{"decode": (1, 1), "verify": (2, 16), "mixed": (32, 512), "prompt": (32, 1024)}[shape])
    if shape in ("mixed", "prompt"):  # long chunks: fewer sequences
        c["B"] = _log(rng, 1, 32 if shape == "mixed" else max(1, 2048 // c["q"]))
        c["mix"] = "some" if shape == "mixed" else rng.choice(["same", "all"])
    # the keys of all sequences together stay within those of the listed cases
    top = 300000 * 8 * 128 // (c["Hkv"] * c["D"])
    c["L"] = max(c["q"], _log(rng, 16, min(32768, max(64, top // c["B"]))))
    long_rows = shape in ("mixed", "prompt")
    if long_rows:
        c["L"] = max(c["q"], min(c["L"], 8192))
    if op == "prefix":
        c["P"] = max(1, _log(rng, 64, 4096 if long_rows else 16384) // c["page"]) * c["page"]  # whole pages are shared
        own_keys = max(c["q"], min(c["L"], 1024))
        c["L"] = c["P"] + own_keys
        c["low"] = (c["P"] + max(c["q"], int(own_keys * c["low"]))) / c["L"]
    elif heads[2] == 256 and rng.random() < 0.7:
        c["softcap"], c["window"] = 50.0, rng.choice([0, 512, 4096])
    return _case(**c)


# --------------------------------------------------------------------------------------------------------------------
# Inputs
# --------------------------------------------------------------------------------------------------------------------
def _lens(case):
    """(q_len, kv_len) of every sequence: of the case, not of the seed."""
    rng = random.Random(case["vary"] * 1000003 + case["B"])
    q, L, mix = case["q"], case["L"], case["mix"]
    out = []
    for b in range(case["B"]):
        n = q
        if mix == "some":
            n = _log(rng, max(1, q // 8), q) if rng.random() < 0.125 or b == 0 else 1
        elif mix == "all":
            n = _log(rng, max(1, q // 16), q)
        kv = L if b == 0 else _log(rng, max(1, int(round(L * case["low"]))), L)
        out.append((n, max(n, kv)))
    return out


def _ragged(case):
    return case["mix"] != "same"


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _randn(g, dtype, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=dtype if dtype != torch.float32 else None)


def _inputs(case, seed):
    """The tensors of a case, from the seed alone. Every sequence has pages of its own, in no order, apart from the
    pages of a shared prefix. Appending looks at the last pages of a sequence only: there all earlier ones are one
    document's."""
    g, dt = _gen(seed), _DTYPES[case["dtype"]]
    lens, page, Hkv, D, H = _lens(case), case["page"], case["Hkv"], case["D"], case["H"]
    width = -(-case["L"] // page)
    if case["op"] == "append":
        shared = [max(0, kv - n) // page for n, kv in lens]
    else:
        shared = [case["P"] // page] * len(lens)
    common = max(shared) if case["op"] != "attention" else 0
    n_pages = common + sum(-(-kv // page) - min(s, common) for s, (_, kv) in zip(shared, lens))
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    host = torch.zeros(len(lens), width, dtype=torch.int64)
    at = common
    for b, (s, (_, kv)) in enumerate(zip(shared, lens)):
        s, used = min(s, common), -(-kv // page)
        host[b, :s] = torch.arange(s)
        host[b, s:used] = torch.arange(at, at + used - s)
        at += used - s
    table = order[host.cuda()]  # entries behind a sequence's last page name some page, as a reused table's do
    pages = []
    for _ in range(2):
        shape = (n_pages, page, Hkv, D) if case["layout"] == "row" else (n_pages, Hkv, page, D)
        t = torch.empty(shape, dtype=dt, device="cuda").normal_(generator=g)
        pages.append(t if case["layout"] == "row" else t.transpose(1, 2))
    tokens = sum(n for n, _ in lens)
    starts = [0]
    for n, _ in lens:
        starts.append(starts[-1] + n)
    s = dict(k_pages=pages[0], v_pages=pages[1], table=table,
             kv_lens=torch.tensor([kv for _, kv in lens], dtype=torch.int32).cuda(),
             cu_q=torch.tensor(starts, dtype=torch.int32).cuda() if _ragged(case) else None)
    lead = (tokens,) if _ragged(case) else (case["B"], case["q"])
    if case["op"] == "append":  # views of the projection's result
        qkv = _randn(g, dt, *lead, (H + 2 * Hkv) * D)
        s["q"] = qkv[..., : H * D].unflatten(-1, (H, D))
        s["k"] = qkv[..., H * D: (H + Hkv) * D].unflatten(-1, (Hkv, D))
        s["v"] = qkv[..., (H + Hkv) * D:].unflatten(-1, (Hkv, D))
    else:
        s["q"] = _randn(g, dt, *lead, H, D)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = dict(case)
    s["lens"] = _lens(case)  # the scheduler knows the lengths
    return s


# --------------------------------------------------------------------------------------------------------------------
# One pass
# --------------------------------------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    return _plain_append(state, case) if case["op"] == "append" else _plain_attention(state, case)


def _run_own(s, case):
    from deepgengraph_amd import paged

    if case["op"] == "append":
        q = paged.paged_append(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], query=s["q"],
                               cu_q=s["cu_q"], rope_theta=case["theta"])
        return q, s["k_pages"], s["v_pages"]
    options = dict(cu_q=s["cu_q"], softcap=case["softcap"], window=case["window"], return_lse=case["lse"])
    if case["op"] == "prefix":
        return paged.shared_prefix_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], case["P"],
                                             **options)
    return paged.paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["kv_lens"], **options)


def _flat(t):
    """[B, q, heads, D] or [tokens, heads, D] as [tokens, heads, D]."""
    return t.reshape(-1, *t.shape[-2:])


def _plain_append(s, case):
    dev, page, D = s["k"].device, case["page"], case["D"]
    q_len = (s["cu_q"][1:] - s["cu_q"][:-1]).long() if s["cu_q"] is not None else torch.full(
        (case["B"],), case["q"], device=dev)
    k, v, q = _flat(s["k"]), _flat(s["v"]), _flat(s["q"])
    T = k.shape[0]
    seq = torch.repeat_interleave(torch.arange(case["B"], device=dev), q_len, output_size=T)
    first = torch.cumsum(q_len, 0) - q_len
    pos = s["kv_lens"].long()[seq] - q_len[seq] + torch.arange(T, device=dev) - first[seq]
    freq = case["theta"] ** (-torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
    ang = pos.double().unsqueeze(1) * freq  # in 64 bits: 32 leave a hundredth of a radian at position 100,000
    cos, sin = ang.cos().float().unsqueeze(1), ang.sin().float().unsqueeze(1)

    def rotate(t):
        a, b = t.float().chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(t.dtype)

    where = s["table"][seq, pos // page].long()
    s["k_pages"][where, pos % page] = rotate(k)
    s["v_pages"][where, pos % page] = v
    return rotate(q).view(s["q"].shape), s["k_pages"], s["v_pages"]


def _plain_attention(s, case):
    """Sequence by sequence and KV head by KV head: gather the pages, scores, mask, softmax, product."""
    page, D, H, Hkv = case["page"], case["D"], case["H"], case["Hkv"]
    G = H // Hkv
    q = _flat(s["q"])
    out = torch.empty_like(q)
    lse = torch.empty(q.shape[0], H, dtype=torch.float32, device=q.device)
    t0 = 0
    for b, (n, kv) in enumerate(s["lens"]):
        ids = s["table"][b, : -(-kv // page)].long()
        k = s["k_pages"][ids].flatten(0, 1)[:kv].float()
        v = s["v_pages"][ids].flatten(0, 1)[:kv].float()
        i = torch.arange(n, device=q.device).unsqueeze(1) + (kv - n)
        j = torch.arange(kv, device=q.device).unsqueeze(0)
        hidden = j > i
        if case["window"]:
            hidden |= i - j >= case["window"]
        step = Hkv if G * n * kv * Hkv <= 1 << 26 else 1
        for h in range(0, Hkv, step):
            qh = q[t0: t0 + n, h * G: (h + step) * G].float().view(n, step, G, D)
            qh = qh.permute(1, 2, 0, 3).reshape(step, G * n, D)
            kh = k[:, h: h + step].permute(1, 2, 0).contiguous()
            x = torch.matmul(qh, kh) / math.sqrt(D)
            if case["softcap"]:
                x = case["softcap"] * torch.tanh(x / case["softcap"])
            x = x.view(step, G, n, kv).masked_fill_(hidden, -math.inf)
            m = x.amax(-1, keepdim=True)
            p = torch.exp(x - m)
            total = p.sum(-1, keepdim=True)
            o = torch.matmul((p / total).view(step, G * n, kv), v[:, h: h + step].permute(1, 0, 2).contiguous())
            out[t0: t0 + n, h * G: (h + step) * G] = o.view(step * G, n, D).transpose(0, 1).to(q.dtype)
            lse[t0: t0 + n, h * G: (h + step) * G] = (m + total.log()).view(step * G, n).t()
        t0 += n
    out = out.view(s["q"].shape)
    if not case["lse"]:
        return out
    return out, lse if _ragged(case) else lse.view(case["B"], case["q"], H).transpose(1, 2)


# --------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# --------------------------------------------------------------------------------------------------------------------
def work(case):
    e, D, H, Hkv, P = _SIZE[case["dtype"]], case["D"], case["H"], case["Hkv"], case["P"]
    lens = _lens(case)
    tokens = sum(n for n, _ in lens)
    if case["op"] == "append":
        return {"bytes": int(2 * e * tokens * (H + 2 * Hkv) * D), "flops": 3.0 * tokens * (H + Hkv) * D}
    window = case["window"]
    keys, pairs = P, 0
    for n, kv in lens:
        first = max(0, kv - n - window + 1) if window else 0
        keys += kv - max(first, P)
        if window:
            pairs += sum(min(window, i + 1) for i in range(kv - n, kv))
        else:
            pairs += n * kv - n * (n - 1) // 2
    by = 2 * e * keys * Hkv * D + 2 * e * tokens * H * D + (4 * tokens * H if case["lse"] else 0)
    return {"bytes": int(by), "flops": 4.0 * D * H * pairs}


# --------------------------------------------------------------------------------------------------------------------
# The 64-bit results
# --------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s, lens = _inputs(case, seed), _lens(case)
    return _exact_append(s, case, lens) if case["op"] == "append" else _exact_attention(s, case, lens)


def _exact_append(s, case, lens):
    D, page = case["D"], case["page"]
    half = D // 2
    inv = torch.tensor([case["theta"] ** (-2.0 * i / D) for i in range(half)], dtype=torch.float64, device="cuda")
    shape = s["q"].shape
    q, k, v = (_flat(s[name]).double() for name in ("q", "k", "v"))
    kp, vp = s["k_pages"].double(), s["v_pages"].double()
    q_out = torch.empty_like(q)
    t = 0
    for b, (n, kv) in enumerate(lens):
        pos = torch.arange(kv - n, kv, device="cuda")
        turn = torch.polar(torch.ones(n, half, dtype=torch.float64, device="cuda"), pos.double()[:, None] * inv)

        def rotate(x):
            z = torch.complex(x[..., :half].contiguous(), x[..., half:].contiguous()) * turn[:, None]
            return torch.cat([z.real, z.imag], dim=-1)

        q_out[t: t + n] = rotate(q[t: t + n])
        rows = (s["table"][b].long()[pos // page], pos % page)
        kp[rows] = rotate(k[t: t + n])
        vp[rows] = v[t: t + n]
        t += n
    return q_out.view(shape), kp, vp


def _exact_attention(s, case, lens):
    D, H, Hkv, page = case["D"], case["H"], case["Hkv"], case["page"]
    if sum(n * kv for n, kv in lens) * H * D > 4e12:
        return None
    q = _flat(s["q"])
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.zeros(q.shape[:2], dtype=torch.float64, device="cuda")
    t = 0
    for b, (n, kv) in enumerate(lens):
        at = torch.arange(kv, device="cuda")
        rows = (s["table"][b].long()[at // page], at % page)
        ks, vs = s["k_pages"][rows], s["v_pages"][rows]
        seen = at[None, :] <= (torch.arange(n, device="cuda") + kv - n)[:, None]
        if case["window"]:
            seen &= at[None, :] > (torch.arange(n, device="cuda") + kv - n - case["window"])[:, None]
        for hk in range(Hkv):
            kh, vh = ks[:, hk].double(), vs[:, hk].double()
            for h in range(hk * (H // Hkv), (hk + 1) * (H // Hkv)):
                x = torch.mm(q[t: t + n, h].double(), kh.t()) * D ** -0.5
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                x[~seen] = -math.inf
                out[t: t + n, h] = torch.mm(torch.softmax(x, dim=-1), vh)
                lse[t: t + n, h] = torch.logsumexp(x, dim=-1)
        t += n
    out = out.view(s["q"].shape)
    if not case["lse"]:
        return out
    return out, lse if _ragged(case) else lse.view(case["B"], case["q"], H).transpose(1, 2)
