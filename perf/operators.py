"""The paged-serving operators as a user's program runs them: the cases that stand for them, their plain forms in
elementary torch operations, and their values in 64 bits.

    append   a step's keys and values rotated, held in 4 bits (Q4_0) and put into the pages, its queries rotated beside
             them; the rows are then read back as the values they stand for
    read     cached rows gathered from the pages as dense keys and values (a shared prefix, ready for a prefill)
    decode   grouped-query attention of one or a few new tokens per sequence over the 4-bit pages
    prefill  causal (or sliding-window) attention over packed prompts of different lengths, with or without a prefix

A Q4_0 block is 32 elements: with m its element of the largest magnitude (the first of equals) the scale is
d = f16(m / -8), held within +-65504, and an element's code is floor(x / d + 8.5) held within 0..15 (8 where d is 0);
the element then stands for (code - 8) * d.  A page holds, for each KV head, page_size rows of Dh / 2 bytes.  Of the
32-bit words of a key row, word t * Dh/32 + b holds dimensions 32b + 8t .. + 7 of block b, the lowest in the lowest
four bits; of the 16-bit halfwords of a value row, halfword g * Dh/32 + b holds dimensions 32b + 4g .. + 3.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f32": 4, "bf16": 2, "f16": 2}


# ---- the cases -------------------------------------------------------------
def _text(lens):
    return ",".join(str(n) for n in lens)


def _lens(text):
    return [int(n) for n in text.split(",")]


def listed():
    r = random.Random(1)
    ragged = [r.randint(512, 8192) for _ in range(64)]
    return [
        # one user's next token: a short context, where latency counts (the 16 / 8 head layer of the single-sequence decode workload)
        dict(name="decode one 1k", op="decode", dtype="f32", H=16, KV=8, D=128, S=1, window=0, page=16, lens="1024"),
        # the batched decode workload: 64 sequences of 512 .. 8192 keys
        dict(name="decode batch 64", op="decode", dtype="bf16", H=32, KV=8, D=128, S=1, window=0, page=64, lens=_text(ragged)),
        # one long document being continued
        dict(name="decode one 128k", op="decode", dtype="bf16", H=32, KV=8, D=128, S=1, window=0, page=128, lens="131072"),
        # four drafted tokens of eight users checked at once, on the hybrid model's full-attention layer (16 / 2 heads of 256)
        dict(name="decode drafted dh256", op="decode", dtype="f32", H=16, KV=2, D=256, S=4, window=0, page=32,
             lens="4801,37,2500,1111,4096,733,3999,260"),
        # a chat turn of one user
        dict(name="prefill one 77", op="prefill", dtype="bf16", H=16, KV=8, D=128, window=0, new="77", prefix="0", fused=False),
        # the prompts that arrive together in a serving loop, packed, from one fused projection
        dict(name="prefill packed 8k", op="prefill", dtype="bf16", H=32, KV=8, D=128, window=0, new="3001,1,640,1777,129,2048,511,85",
             prefix="0,0,0,0,0,0,0,0", fused=True),
        # sliding-window layers over long packed prompts (16 / 4 heads, window 1024)
        dict(name="prefill window 32k", op="prefill", dtype="bf16", H=16, KV=4, D=128, window=1024,
             new="4096,5000,2222,4999,4096,3500,4500,4355", prefix="0,0,0,0,0,0,0,0", fused=False),
        # prompts whose beginnings are cached already: the new tokens attend the prefix too
        dict(name="prefill prefix f16", op="prefill", dtype="f16", H=32, KV=8, D=128, window=0, new="512,700,33,256",
             prefix="3500,1024,4000,2047", fused=False),
        # one decode step of 64 sequences
        dict(name="append step 64", op="append", dtype="bf16", H=32, KV=8, D=128, rotary=128, page=64, n=64, fused=False),
        # 8192 packed prompt tokens from one fused projection
        dict(name="append prompt 8k", op="append", dtype="bf16", H=32, KV=8, D=128, rotary=128, page=64, n=8192, fused=True),
        # a short shared prefix of the hybrid model's full-attention layer
        dict(name="read 300 dh256", op="read", dtype="f32", KV=2, D=256, page=16, n=300),
        # a long shared prefix, read for a bf16 prefill
        dict(name="read 16k", op="read", dtype="bf16", KV=8, D=128, page=64, n=16384),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["decode", "decode", "prefill", "prefill", "append", "read"])
    page = rng.choice([16, 32, 64, 128])
    H, KV, D = rng.choice([(16, 8, 128), (32, 8, 128), (16, 4, 128), (16, 2, 256), (6, 3, 128), (8, 1, 128)])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if op == "decode":
        S, longest, left = rng.choice([1, 1, 1, 2, 5]), 8192 if D == 128 else 4096, 100000
        lens = []
        for _ in range(_log(rng, 1, 48)):
            n = 0 if lens and rng.random() < 0.05 else _log(rng, 1, longest)
            if left - n < 0:
                break
            left -= n
            lens.append(n)
        return dict(op=op, dtype=dtype, H=H, KV=KV, D=D, S=S, window=rng.choice([0, 0, 0, 1024, 129]), page=page,
                    lens=_text(lens))
    if op == "prefill":
        H, KV = rng.choice([(16, 8), (16, 4), (6, 3), (8, 1), (32, 8)])
        new, prefix, left, some = [], [], 6000, rng.random() < 0.4
        for _ in range(_log(rng, 1, 24)):
            n = _log(rng, 1, 2000)
            if left - n < 0:
                break
            left -= n
            new.append(n)
            prefix.append(_log(rng, 1, 1000) if some and rng.random() < 0.7 else 0)
        return dict(op=op, dtype="bf16" if dtype == "f32" else dtype, H=H, KV=KV, D=128, window=rng.choice([0, 0, 1024, 129]),
                    new=_text(new), prefix=_text(prefix), fused=rng.random() < 0.4)
    if op == "append":
        return dict(op=op, dtype=dtype, H=H, KV=KV, D=D, rotary=rng.choice([D, D, D // 2, 64]), page=page,
                    n=_log(rng, 1, 4096 if D == 128 else 2048), fused=rng.random() < 0.4)
    return dict(op=op, dtype=dtype, KV=KV, D=D, page=page, n=_log(rng, 1, 8000))


# ---- inputs ----------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(1000003 * seed + 17)
    return g


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)


def _pack_k(code):
    """Codes [.., Dh] of key rows as their bytes [.., Dh / 2]."""
    x = code.to(torch.uint8).unflatten(-1, (-1, 4, 4, 2))
    return (x[..., 0] | (x[..., 1] << 4)).transpose(-3, -2).flatten(-3)


def _pack_v(code):
    """Codes [.., Dh] of value rows as their bytes [.., Dh / 2]."""
    x = code.to(torch.uint8).unflatten(-1, (-1, 8, 2, 2))
    return (x[..., 0] | (x[..., 1] << 4)).transpose(-3, -2).flatten(-3)


def _filled(g, KV, page, D, n_pages, pack):
    """Pages that other requests have filled before: every row holds something."""
    x = _normal(g, n_pages, KV, page, D // 32, 32)
    at = x.abs().argmax(-1, keepdim=True)
    d = (x.gather(-1, at) / -8).half()
    code = (x / d.float() + 8.5).floor().clamp(0, 15).flatten(-2)
    return pack(code).contiguous(), d.squeeze(-1).contiguous()


def _backend():
    global _be
    from hachiue_b200 import CudaBackend
    if _be is None:
        _be = CudaBackend(0)
    return _be


_be = None


def _handle(s):
    """The framework's view of the state, where its kernels run."""
    if own:
        from hachiue_b200 import PagedKVCache
        s["be"] = _backend()
        if "k_pages" in s:
            s["cache"] = PagedKVCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    return s


def _pages(s, g, case, n_pages):
    s["k_pages"], s["k_scale"] = _filled(g, case["KV"], case["page"], case["D"], n_pages, _pack_k)
    s["v_pages"], s["v_scale"] = _filled(g, case["KV"], case["page"], case["D"], n_pages, _pack_v)


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    op, dt, D = case["op"], DTYPES[case["dtype"]], case["D"]
    if op == "decode":
        lens = _lens(case["lens"])
        per = [-(-n // case["page"]) for n in lens]
        n_pages = sum(per) + 3
        _pages(s, g, case, n_pages)
        order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32).cpu()
        table = torch.zeros((len(lens), max(1, max(per))), dtype=torch.int32)
        at = 0
        for b, n in enumerate(per):
            table[b, :n] = order[at:at + n]
            at += n
        s["table"], s["context"] = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
        s["longest"] = max(1, max(lens))
        s["q"] = _normal(g, len(lens), case["S"], case["H"], D).to(dt)
        s["out"] = torch.empty_like(s["q"])
    elif op == "prefill":
        new, prefix = _lens(case["new"]), _lens(case["prefix"])
        nq, nk, H, KV = sum(new), sum(new) + sum(prefix), case["H"], case["KV"]
        if case["fused"] and nq == nk:  # views of one projection's output
            x = _normal(g, nq, H + 2 * KV, D).to(dt)
            s["q"], s["k"], s["v"] = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
        else:
            s["q"], s["k"], s["v"] = (_normal(g, n, h, D).to(dt) for n, h in ((nq, H), (nk, KV), (nk, KV)))
        s["cu_q"], s["cu_k"] = _cu(new), _cu([a + b for a, b in zip(new, prefix)])
        s["new_lens"], s["key_lens"] = new, [a + b for a, b in zip(new, prefix)]
        s["out"] = torch.empty((nq, H, D), dtype=dt, device="cuda")
    else:
        n, KV, page = case["n"], case["KV"], case["page"]
        n_pages = -(-n // page) * 2 + 2
        _pages(s, g, case, n_pages)
        s["k_read"], s["v_read"] = (torch.empty((n, KV, D), dtype=dt, device="cuda") for _ in range(2))
        if op == "append" and n <= 256:  # a decode step: every sequence has its own page and place
            first = torch.randperm(n_pages, generator=g, device="cuda")[:n] if n <= n_pages else None
            if first is None:
                s["slots"] = torch.randperm(n_pages * page, generator=g, device="cuda")[:n]
            else:
                s["slots"] = first * page + torch.randint(0, page, (n,), generator=g, device="cuda")
        else:  # whole prompts: pages in any order, filled from their beginning
            order = torch.randperm(n_pages, generator=g, device="cuda")
            i = torch.arange(n, device="cuda")
            s["slots"] = order[i // page] * page + i % page
        if op == "append":
            H, rot = case["H"], case["rotary"]
            if case["fused"]:
                x = _normal(g, n, H + 2 * KV, D).to(dt)
                s["q"], s["k"], s["v"] = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
            else:
                s["q"], s["k"], s["v"] = (_normal(g, n, h, D).to(dt) for h in (H, KV, KV))
            most = 8192
            s["positions"] = (torch.randint(0, most, (n,), generator=g, device="cuda") if n <= 256 else
                              torch.arange(n, device="cuda") % most).to(torch.int32)
            angle = (torch.arange(most, dtype=torch.float64, device="cuda")[:, None]
                     * torch.pow(torch.tensor(1e6, dtype=torch.float64, device="cuda"),
                                 -torch.arange(rot // 2, dtype=torch.float64, device="cuda") / (rot // 2))[None])
            s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
            s["q_out"] = torch.empty((n, H, D), dtype=dt, device="cuda")
            s["k_out"] = torch.empty((n, KV, D), dtype=dt, device="cuda")
    return _handle(s)


# ---- one pass --------------------------------------------------------------
def run(s):
    op = s["op"]
    if own:
        be = s["be"]
        if op == "decode":
            be.attention_paged(s["q"], s["cache"], s["out"], s["table"], s["context"], max_context=s["longest"],
                               window_size=s["window"])
            return s["out"]
        if op == "prefill":
            be.prefill_varlen(s["q"], s["k"], s["v"], s["out"], s["cu_q"], s["cu_k"], window=s["window"])
            return s["out"]
        if op == "append":
            be.rope_append_paged(s["k"], s["v"], s["cache"], s["slots"], cos=s["cos"], sin=s["sin"],
                                 positions=s["positions"], q=s["q"], q_out=s["q_out"], k_out=s["k_out"])
        be.read_paged(s["cache"], s["slots"], s["k_read"], s["v_read"])
    else:
        if op == "decode":
            return _plain_decode(s)
        if op == "prefill":
            return _plain_prefill(s)
        if op == "append":
            _plain_append(s)
        _plain_read(s)
    if op == "append":
        return s["q_out"], s["k_out"], s["k_read"], s["v_read"]
    return s["k_read"], s["v_read"]


def _values(packed, scale, groups, width):
    """Bytes [.., Dh / 2] and scales [.., Dh / 32] as f32 values [.., Dh]."""
    x = packed.unflatten(-1, (groups, -1, width)).transpose(-3, -2)
    code = torch.stack([x & 15, x >> 4], -1).flatten(-4).float()
    return ((code - 8).unflatten(-1, (-1, 32)) * scale.float()[..., None]).flatten(-2)


def _plain_decode(s):
    B, S, H, D = s["q"].shape
    KV, page = s["KV"], s["page"]
    T = s["table"].shape[1] * page
    rows = lambda x: x[s["table"].long()].transpose(1, 2).flatten(2, 3)  # noqa: E731  [B, KV, T, ..]
    k = _values(rows(s["k_pages"]), rows(s["k_scale"]), 4, 4)
    q = s["q"].float().view(B, S, KV, H // KV, D).permute(0, 2, 3, 1, 4)
    x = torch.matmul(q.flatten(2, 3), k.transpose(-1, -2)).view(B, KV, H // KV, S, T) / math.sqrt(D)
    del k
    at = torch.arange(T, device="cuda")[None, None]
    pos = s["context"].long()[:, None, None] - S + torch.arange(S, device="cuda")[None, :, None]
    keep = at <= pos
    if s["window"]:
        keep = keep & (at > pos - s["window"])
    x = x.masked_fill(~keep[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)  # a row without keys gives zeros
    v = _values(rows(s["v_pages"]), rows(s["v_scale"]), 8, 2)
    out = torch.matmul(p.flatten(2, 3), v).view(B, KV, H // KV, S, D).permute(0, 3, 1, 2, 4)
    s["out"].copy_(out.reshape(B, S, H, D))
    return s["out"]


def _padded(x, cu, most):
    """Packed rows [n, heads, D] as f32 [B, heads, most, D] and which of them exist."""
    first, n = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    at = torch.arange(most, device="cuda")
    there = at[None] < n[:, None]
    rows = torch.where(there, first[:, None] + at[None], 0)
    return torch.where(there[..., None, None], x[rows].float(), 0.0).transpose(1, 2), rows, there


def _plain_prefill(s):
    H, KV, D = s["H"], s["KV"], s["D"]
    Lq, Lk = max(s["new_lens"]), max(s["key_lens"])
    q, rows, there = _padded(s["q"], s["cu_q"], Lq)
    k = _padded(s["k"], s["cu_k"], Lk)[0]
    B = q.shape[0]
    x = torch.matmul(q.reshape(B, KV, H // KV * Lq, D), k.transpose(-1, -2)).view(B, KV, H // KV, Lq, Lk)
    x *= 1 / math.sqrt(D)
    nq, nk = (c[1:] - c[:-1] for c in (s["cu_q"], s["cu_k"]))
    pos = (nk - nq).long()[:, None, None] + torch.arange(Lq, device="cuda")[None, :, None]
    at = torch.arange(Lk, device="cuda")[None, None]
    keep = (at <= pos) & (at < nk[:, None, None])
    if s["window"]:
        keep = keep & (at > pos - s["window"])
    x.masked_fill_(~keep[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x -= torch.where(top == -math.inf, 0.0, top)
    x.exp_()
    x /= x.sum(-1, keepdim=True).clamp_min(1e-30)
    v = _padded(s["v"], s["cu_k"], Lk)[0]
    out = torch.matmul(x.view(B, KV, H // KV * Lq, Lk), v).view(B, H, Lq, D).transpose(1, 2)
    s["out"][rows[there]] = out[there].to(s["out"].dtype)
    return s["out"]


def _rotated(x, c, sn, half):
    a, b, rest = x[..., :half], x[..., half:2 * half], x[..., 2 * half:]
    return torch.cat([a * c - b * sn, b * c + a * sn, rest], -1)


def _quantised(x):
    """f32 rows [.., Dh] as codes [.., Dh] and f16 scales [.., Dh / 32]."""
    x = x.unflatten(-1, (-1, 32))
    m = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = (m / -8).clamp(-65504, 65504).half()
    code = (x.double() / torch.where(d == 0, 1, d).double() + 8.5).floor().clamp(0, 15)  # exact next to a border
    return torch.where(d == 0, 8.0, code).flatten(-2), d.squeeze(-1)


def _plain_append(s):
    half = s["rotary"] // 2
    at = s["positions"].long()
    c, sn = s["cos"][at][:, None], s["sin"][at][:, None]
    s["q_out"].copy_(_rotated(s["q"].float(), c, sn, half))
    k = _rotated(s["k"].double(), c.double(), sn.double(), half).float()
    s["k_out"].copy_(k)
    page, off = s["slots"] // s["page"], s["slots"] % s["page"]
    for x, pages, scale, pack in ((k, s["k_pages"], s["k_scale"], _pack_k), (s["v"].float(), s["v_pages"], s["v_scale"], _pack_v)):
        code, d = _quantised(x)
        pages[page, :, off] = pack(code)
        scale[page, :, off] = d


def _plain_read(s):
    page, off = s["slots"] // s["page"], s["slots"] % s["page"]
    s["k_read"].copy_(_values(s["k_pages"][page, :, off], s["k_scale"][page, :, off], 4, 4))
    s["v_read"].copy_(_values(s["v_pages"][page, :, off], s["v_scale"][page, :, off], 8, 2))


# ---- what a pass cannot do without ------------------------------------------
def _pairs(new, keys, window):
    """(query, key) pairs of a causal sequence, and the keys that any query sees."""
    pairs, first = 0, keys
    for i in range(new):
        pos = keys - new + i
        lo = max(0, pos + 1 - window) if window else 0
        pairs += max(0, pos + 1 - lo)
        first = min(first, lo)
    return pairs, keys - first


def work(case):
    D, KV, e = case["D"], case["KV"], BYTES[case["dtype"]]
    row = 2 * KV * (D // 2 + D // 32 * 2)  # a cached token's keys and values
    if case["op"] == "decode":
        got = [_pairs(case["S"], n, case["window"]) for n in _lens(case["lens"])]
        vec = len(got) * case["S"] * case["H"] * D
        return {"bytes": sum(n for _, n in got) * row + 2 * vec * e, "flops": 4 * D * case["H"] * sum(p for p, _ in got)}
    if case["op"] == "prefill":
        new, prefix = _lens(case["new"]), _lens(case["prefix"])
        got = [_pairs(a, a + b, case["window"]) for a, b in zip(new, prefix)]
        return {"bytes": (2 * sum(new) * case["H"] + 2 * sum(n for _, n in got) * KV) * D * e,
                "flops": 4 * D * case["H"] * sum(p for p, _ in got)}
    n = case["n"]
    if case["op"] == "read":
        return {"bytes": n * (row + 2 * KV * D * e), "flops": 2 * n * KV * D}
    tables = min(n, 8192) * case["rotary"] * 4
    return {"bytes": n * (2 * row + (2 * case["H"] + 3 * KV) * D * e + 2 * KV * D * e) + tables,
            "flops": n * (case["H"] + KV) * case["rotary"] * 3 + 6 * n * KV * D}


# ---- the definition in 64 bits ----------------------------------------------
def _nibbles(row, D, order):
    """One tensor of rows [.., D / 2] as 64-bit codes by an index table: dimension i is nibble order[i] of the row."""
    both = torch.stack([row.double() % 16, torch.div(row, 16, rounding_mode="floor").double()], -1).flatten(-2)
    return both[..., order] - 8


def _key_order(D):
    nb = D // 32
    return torch.tensor([((i % 32 // 8) * nb + i // 32) * 8 + i % 8 for i in range(D)], device="cuda")


def _value_order(D):
    nb = D // 32
    return torch.tensor([((i % 32 // 4) * nb + i // 32) * 4 + i % 4 for i in range(D)], device="cuda")


def _attend(q, k, v, first, window):
    """q [S, G, D] at positions first .. over k, v [T, D], in 64 bits."""
    S, G, D = q.shape
    out = torch.zeros((S, G, D), dtype=torch.float64, device="cuda")
    step = max(1, 200_000_000 // max(1, k.shape[0] * G))
    for lo in range(0, S, step):
        x = torch.einsum("sgd,td->sgt", q[lo:lo + step], k) / D ** 0.5
        pos = torch.arange(lo, min(S, lo + step), device="cuda")[:, None] + first
        t = torch.arange(k.shape[0], device="cuda")[None]
        hide = (t > pos) | ((t <= pos - window) if window else torch.zeros_like(t, dtype=torch.bool))
        w = torch.where(hide[:, None], torch.full_like(x, -math.inf), x)
        w = torch.nan_to_num(torch.softmax(w, -1), nan=0.0)
        out[lo:lo + step] = torch.einsum("sgt,td->sgd", w, v)
    return out


def exact(case, seed):
    s = prepare(case, seed)
    D, KV, op = case["D"], case["KV"], case["op"]
    if op == "decode":
        q = s["q"].double()
        out = torch.zeros_like(q)
        G = case["H"] // KV
        for b, n in enumerate(_lens(case["lens"])):
            if n == 0:
                continue
            t = torch.arange(n, device="cuda")
            page, off = s["table"][b].long()[t // case["page"]], t % case["page"]
            k = _nibbles(s["k_pages"][page, :, off], D, _key_order(D)) * s["k_scale"][page, :, off].double().repeat_interleave(32, -1)
            v = _nibbles(s["v_pages"][page, :, off], D, _value_order(D)) * s["v_scale"][page, :, off].double().repeat_interleave(32, -1)
            for h in range(KV):
                out[b, :, h * G:(h + 1) * G] = _attend(q[b, :, h * G:(h + 1) * G], k[:, h], v[:, h], n - case["S"], case["window"])
        return out
    if op == "prefill":
        q, k, v = (s[x].double() for x in "qkv")
        out = torch.zeros_like(q)
        G, i, j = case["H"] // KV, 0, 0
        for a, b in zip(_lens(case["new"]), _lens(case["prefix"])):
            for h in range(KV):
                out[i:i + a, h * G:(h + 1) * G] = _attend(q[i:i + a, h * G:(h + 1) * G], k[j:j + a + b, h], v[j:j + a + b, h], b, case["window"])
            i, j = i + a, j + a + b
        return out
    page, off = s["slots"] // case["page"], s["slots"] % case["page"]
    if op == "read":
        return tuple(_nibbles(s[p][page, :, off], D, order(D)) * s[c][page, :, off].double().repeat_interleave(32, -1)
                     for p, c, order in (("k_pages", "k_scale", _key_order), ("v_pages", "v_scale", _value_order)))
    half = case["rotary"] // 2
    c, sn = (s[x][s["positions"].long()].double()[:, None] for x in ("cos", "sin"))
    turned = []
    for x in (s["q"].double(), s["k"].double()):
        y = x.clone()
        y[..., :half] = x[..., :half] * c - x[..., half:2 * half] * sn
        y[..., half:2 * half] = x[..., half:2 * half] * c + x[..., :half] * sn
        turned.append(y)
    stands = []
    for x in (turned[1].float().double(), s["v"].double()):  # a cached key is rounded to f32 before it is held in 4 bits
        x = x.reshape(-1, 32)
        big = x.abs().max(-1, keepdim=True).values
        where = (x.abs() == big).to(torch.int8).argmax(-1, keepdim=True)  # the first of equals
        d = (x.gather(1, where) * -0.125).clamp(-65504, 65504).float().half().double()
        levels = torch.arange(16, dtype=torch.float64, device="cuda") - 8
        # the highest level whose lower border is not above the element
        code = (x / torch.where(d == 0, torch.ones_like(d), d))[..., None] >= (levels - 0.5)[None, None]
        code = (code.sum(-1) - 1).clamp_min(0)
        stands.append(torch.where(d == 0, torch.zeros_like(x), levels[code] * d).view(s["v"].shape))
    return turned[0], turned[1], stands[0], stands[1]
