"""The paged 4-bit cache on the GPU: the rotated append, the read and the decode attention against their definitions in
64 bits, and a run of them with the packed prefill as a serving loop uses them."""
import numpy as np
import pytest
import torch

from hachiue_b200 import HachiueError, PagedKVCache
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
dev = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def tables(half, rows=64, base=1e4):
    angle = torch.arange(rows, dtype=torch.float64)[:, None] * base ** (-torch.arange(half, dtype=torch.float64) / half)[None]
    return angle.cos().float().to(dev), angle.sin().float().to(dev)


def garbage_cache(g, n_pages, page, KV, Dh):
    """Pages that hold anything: random codes, and NaN and infinite scales."""
    c = PagedKVCache.allocate(n_pages, page, KV, Dh)
    for t in (c.k, c.v):
        t.copy_(torch.randint(0, 256, t.shape, generator=g, device=dev, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.where(torch.rand(t.shape, generator=g, device=dev) < 0.5, float("nan"), float("inf")))
    return c


def fill(g, c, slots, spread=1.0):
    """Random rows into the slots, through the reference's quantiser."""
    page, off = slots // c.page_size, slots % c.page_size
    for rows, scale, order in ((c.k, c.k_scale, ref.key_nibble), (c.v, c.v_scale, ref.value_nibble)):
        x = torch.randn((len(slots), c.kv_heads, c.head_dim), generator=g, device=dev) * spread
        code, d = ref.quantise(x)
        rows[page, :, off] = ref.pack(code, order(c.head_dim))
        scale[page, :, off] = d


def paged_batch(g, lens, page, KV, Dh, spread=1.0, spare=2):
    """A cache whose pages are handed out in random order; rows behind each sequence's end hold garbage."""
    per = [-(-n // page) for n in lens]
    c = garbage_cache(g, sum(per) + spare, page, KV, Dh)
    order = torch.randperm(c.n_pages, generator=g, device=dev)
    table = torch.full((len(lens), max(1, max(per))), -7, dtype=torch.int32, device=dev)  # unused entries are no pages
    at, slots = 0, []
    for b, n in enumerate(lens):
        mine = order[at:at + per[b]]
        table[b, :per[b]] = mine.int()
        at += per[b]
        t = torch.arange(n, device=dev)
        slots.append(mine[t // page] * page + t % page if n else t)
    every = torch.cat(slots)
    if len(every):
        fill(g, c, every, spread)
    return c, table, slots


# ---- append ------------------------------------------------------------------
def check_rows(c, before, slots, k, v):
    """Rows of the slots hold k and v's blocks bit for bit, every other row is as it was."""
    page, off = slots // c.page_size, slots % c.page_size
    for name, x, order in (("k", k, ref.key_nibble), ("v", v, ref.value_nibble)):
        code, d = ref.quantise(x)
        want, want_d = before[name].clone(), before[name + "_scale"].clone()
        want[page, :, off] = ref.pack(code, order(c.head_dim))
        want_d[page, :, off] = d
        assert torch.equal(getattr(c, name), want), name
        assert torch.equal(getattr(c, name + "_scale").view(torch.int16), want_d.view(torch.int16)), name


def snapshot(c):
    return {n: getattr(c, n).clone() for n in ("k", "v", "k_scale", "v_scale")}


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,KV,Dh,rotary,page,fused", [
    (1, 16, 8, 128, 128, 16, False), (5, 6, 3, 128, 64, 32, True), (37, 8, 1, 256, 64, 64, True),
    (200, 16, 2, 256, 256, 128, False), (63, 0, 2, 128, 128, 256, False), (9, 4, 4, 128, 0, 16, True),
    (17, 2, 1, 128, 8, 16, True), (33, 4, 2, 256, 200, 16, False)])
def test_append(backend, dtype, n, H, KV, Dh, rotary, page, fused):
    g = gen(n + H + Dh + rotary)
    c = garbage_cache(g, n // page + 4, page, KV, Dh)
    x = torch.randn((n, H + 2 * KV, Dh), generator=g, device=dev).to(dtype)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    slots = torch.randperm(c.n_pages * page, generator=g, device=dev)[:n].clone()
    if n > 4:
        slots[2] = -1  # padding
    pos = torch.randint(0, 64, (n,), generator=g, device=dev, dtype=torch.int32)
    cos, sin = tables(rotary // 2) if rotary else (None, None)
    q_out = torch.full((n, H, Dh), float("nan"), device=dev, dtype=dtype)
    k_out = torch.full((n, KV, Dh), float("nan"), device=dev, dtype=dtype)
    before = snapshot(c)
    backend.rope_append_paged(k, v, c, slots, cos, sin, pos if rotary else None, q if H else None, q_out if H else None, k_out)
    assert backend.device_status() == 0
    there = slots >= 0
    half = rotary // 2
    cr = cos.double()[pos.long()] if rotary else torch.zeros((n, 0), dtype=torch.float64, device=dev)
    sr = sin.double()[pos.long()] if rotary else cr
    turned = ref.rotate(k.double(), cr, sr).float()
    check_rows(c, before, slots[there], turned[there], v.float()[there])
    assert torch.equal(k_out[there], turned.to(dtype)[there])
    assert torch.isnan(k_out[~there].float()).all() and torch.isnan(q_out[~there].float()).all()
    if H:
        want = ref.rotate(q.double(), cr, sr)
        # two products and a sum in f32, then the rounding to dtype
        size = ref.rotate(q.double().abs(), cr.abs(), -sr.abs())
        size[..., half:] = ref.rotate(q.double().abs(), cr.abs(), sr.abs())[..., half:]
        err = (q_out.double() - want).abs()
        assert (err <= 3 * 2.0 ** -24 * size + ref.HALF_STEP[dtype] * 1.01 * want.abs() + 2.0 ** -25)[there].all()


def test_append_quantiser_at_its_borders(backend):
    """Elements on and next to a level's border, blocks whose largest magnitude occurs twice with both signs, zero blocks,
    blocks below the smallest scale and above the largest, and infinities."""
    rows = []
    for m in (1.0, -1.0, 3.0, -0.7, 65536.0, 2.0 ** -13, 2.0 ** -21, 2.0 ** -23, 1e-30, 0.0, 3e38, -5e5 - 3):
        d = float(np.float16(np.clip(np.float32(m) / -8, -65504, 65504)))
        for step in (0.0, 1.0, -1.0):
            x = np.array([(j - 8 + 0.5) * d for j in range(16)] + [(j - 8) * d for j in range(15)] + [m], dtype=np.float32)
            x[:31] = np.nextafter(x[:31], np.float32(np.inf) * step).astype(np.float32) if step else x[:31]
            rows.append(np.clip(x, -abs(m), abs(m)) if abs(m) < 5e5 else x)
    twice = np.zeros(32, np.float32)
    twice[[3, 9, 20]] = 2.0, -2.0, 2.0
    rows += [twice, -twice]
    rows = [r for r in rows if np.isfinite(r).all()]
    while len(rows) % 4:
        rows.append(np.full(32, 0.25, np.float32))
    x = torch.from_numpy(np.stack(rows)).view(-1, 1, 128).to(dev)
    c = PagedKVCache.allocate(8, 16, 1, 128)
    before = snapshot(c)
    slots = torch.arange(len(x), device=dev)
    backend.rope_append_paged(x, x, c, slots)
    check_rows(c, before, slots, x, x)
    inf = torch.zeros((1, 1, 128), device=dev)
    inf[0, 0, 5], inf[0, 0, 40] = float("inf"), float("-inf")
    backend.rope_append_paged(inf, inf, c, slots[:1])
    for w in "kv":  # an infinity is held as the largest value of its sign that a scale allows
        val = ref.cache_rows(c, slots[:1], w)
        assert val[0, 0, 5] == 8 * 65504 and val[0, 0, 40] == -8 * 65504 and val.abs().sum() == 16 * 65504


def test_append_in_place_and_twice(backend):
    """q_out and k_out may be q and k; the same call again over the slots gives the same rows."""
    g = gen(3)
    n, H, KV = 40, 8, 2
    c = PagedKVCache.allocate(4, 16, KV, 128)
    q, k, v = (torch.randn((n, h, 128), generator=g, device=dev).bfloat16() for h in (H, KV, KV))
    cos, sin = tables(64)
    pos = torch.arange(n, device=dev, dtype=torch.int32)
    slots = torch.arange(n, device=dev)
    q1, k1 = torch.empty_like(q), torch.empty_like(k)
    backend.rope_append_paged(k, v, c, slots, cos, sin, pos, q, q1, k1)
    first = snapshot(c)
    backend.rope_append_paged(k, v, c, slots, cos, sin, pos, q, q, k)
    assert torch.equal(q, q1) and torch.equal(k, k1)
    assert all(torch.equal(first[w], getattr(c, w)) for w in first)


def test_append_bad_slots_and_positions(backend):
    """A slot past the cache or a position outside the tables is reported and skipped; its row is written nowhere."""
    g = gen(4)
    c = garbage_cache(g, 2, 16, 2, 128)
    before = snapshot(c)
    k = torch.randn((5, 2, 128), generator=g, device=dev)
    cos, sin = tables(64, rows=8)
    slots = torch.tensor([0, 32, 2 ** 40, 3, 4], device=dev)
    pos = torch.tensor([0, 1, 2, 8, -1], device=dev, dtype=torch.int32)
    out = torch.full_like(k, 7.0)
    backend.rope_append_paged(k, k, c, slots, cos, sin, pos, k_out=out)
    assert backend.device_status() == 2
    want = ref.rotate(k.double(), cos.double()[[0] * 5], sin.double()[[0] * 5]).float()
    check_rows(c, before, slots[:1], want[:1], k[:1])
    assert (out[1:] == 7.0).all()
    assert backend.device_status() == 0


# ---- read --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,KV,Dh,page", [(1, 1, 128, 16), (100, 3, 128, 64), (77, 2, 256, 16), (300, 8, 256, 256)])
def test_read(backend, dtype, n, KV, Dh, page):
    g = gen(n + Dh)
    c = garbage_cache(g, n // page + 3, page, KV, Dh)
    every = torch.randperm(c.n_pages * page, generator=g, device=dev)
    fill(g, c, every[:n], 3.0)
    slots = every[torch.randint(0, n, (n,), generator=g, device=dev)]  # some more than once
    slots[0] = -5
    k, v = (torch.full((n, KV, Dh), 9.0, device=dev, dtype=dtype) for _ in range(2))
    backend.read_paged(c, slots, k, v)
    assert backend.device_status() == 0
    for got, w in ((k, "k"), (v, "v")):
        assert (got[0] == 9.0).all()
        assert torch.equal(got[1:], ref.cache_rows(c, slots[1:], w).float().to(dtype))  # (code - 8) d is exact in f32
    slots[-1] = c.n_pages * page
    k.fill_(9.0)
    backend.read_paged(c, slots, k, v)
    assert backend.device_status() == 2 and (k[-1] == 9.0).all()


# ---- decode attention ----------------------------------------------------------
def check_decode(backend, c, table, slots, q, lens, window, max_context=0, missing=None):
    out = torch.full_like(q, float("nan"))
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    backend.attention_paged(q, c, out, table, ctx, max_context, window)
    S, D = q.shape[1], q.shape[3]
    for b, n in enumerate(lens):
        k, v = (ref.cache_rows(c, slots[b], w) for w in "kv")
        want, spread, mag = ref.attend(q[b].double(), k, v, n - S, window, None if missing is None else missing[b])
        # a bf16 call with more than four rows per KV head rounds the weighted probabilities to f16
        rows = q.shape[1] * q.shape[2] // c.kv_heads
        p_step = 2.0 ** -11 if q.dtype == torch.bfloat16 and rows > 4 else 2.0 ** -22
        bound = ref.attention_bound(want, spread, mag, D, n, q.dtype, p_step)
        err = (out[b].double() - want).abs()
        assert (err <= bound).all(), (b, n, float((err / bound).max()), float(err.max()))
    return out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,Dh,S,window,page,lens", [
    (16, 8, 128, 1, 0, 16, [1024]),
    (2, 2, 128, 1, 0, 16, [1, 0, 15, 16, 17, 31, 33]),
    (8, 2, 128, 1, 0, 64, [700, 64, 1, 65, 0, 129]),
    (8, 1, 128, 1, 100, 32, [99, 100, 101, 1500, 7]),
    (6, 3, 128, 5, 0, 128, [300, 4, 5, 1, 0, 6]),
    (16, 2, 256, 4, 0, 32, [333, 3, 40]),
    (12, 2, 256, 1, 17, 16, [16, 17, 18, 900]),
    (32, 1, 128, 3, 40, 256, [257, 39, 2]),
    (5, 1, 128, 1, 1, 16, [1, 50])])
def test_decode(backend, dtype, H, KV, Dh, S, window, page, lens):
    g = gen(H * 7 + Dh + S + sum(lens))
    c, table, slots = paged_batch(g, lens, page, KV, Dh)
    q = torch.randn((len(lens), S, H, Dh), generator=g, device=dev).to(dtype)
    out = check_decode(backend, c, table, slots, q, lens, window)
    for b, n in enumerate(lens):  # queries without a token
        assert (out[b, :max(0, S - n)] == 0).all()
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,KV,Dh,S,lens", [(8, 2, 128, 1, [20000, 3]), (16, 1, 128, 1, [9000]), (2, 1, 256, 2, [12345, 4000, 1])])
def test_decode_long(backend, dtype, H, KV, Dh, S, lens):
    """The key axis is split over CTAs and joined."""
    g = gen(H + S + sum(lens))
    c, table, slots = paged_batch(g, lens, 64, KV, Dh)
    q = torch.randn((len(lens), S, H, Dh), generator=g, device=dev).to(dtype)
    check_decode(backend, c, table, slots, q, lens, 0, max(lens))
    check_decode(backend, c, table, slots, q, lens, 5000, max(lens))
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_decode_extreme_scores_and_scales(backend, dtype):
    """Scores far apart (one token takes all, at the beginning or the end of a long context), value scales from 2^-20 to
    2^12 in one sequence, and rows of zeros."""
    g = gen(9)
    lens = [600, 600, 600]
    c, table, slots = paged_batch(g, lens, 16, 2, 128)
    scale = torch.exp2(torch.randint(-20, 13, (600,), generator=g, device=dev).float())
    page, off = slots[0] // 16, slots[0] % 16
    c.v_scale[page, :, off] = (c.v_scale[page, :, off].float() * scale[:, None, None]).half()
    q = torch.randn((3, 1, 4, 128), generator=g, device=dev)
    k = ref.cache_rows(c, slots[1], "k")
    q[1, 0, :2] = 12 * k[0, 0].float()  # the first token of sequence 1 takes all, for KV head 0
    q[1, 0, 2:] = 12 * k[599, 1].float()  # the last one, for KV head 1
    page, off = slots[2] // 16, slots[2] % 16
    for t in (c.k_scale, c.v_scale):
        t[page, :, off] = 0
    out = check_decode(backend, c, table, slots, q.to(dtype), lens, 0)
    assert (out[2] == 0).all()
    q[:, :, 0] = 0
    q[:, :, 1] *= 1e-20 if dtype == torch.float32 else 1e-4
    check_decode(backend, c, table, slots, q.to(dtype), lens, 0)
    assert backend.device_status() == 0


def test_decode_bad_pages_and_contexts(backend):
    """A page outside the cache is left out and reported, a context above max_context gives zeros and is reported; pages
    that no visible token needs are not looked up."""
    g = gen(10)
    lens = [100, 90, 80]
    c, table, slots = paged_batch(g, lens, 16, 2, 128)
    q = torch.randn((3, 1, 4, 128), generator=g, device=dev)
    missing = [torch.zeros(n, dtype=torch.bool, device=dev) for n in lens]
    table[0, 2] = c.n_pages
    table[1, 0] = -1
    missing[0][32:48], missing[1][:16] = True, True
    check_decode(backend, c, table, slots, q, lens, 0, missing=missing)
    assert backend.device_status() == 2
    # the windows of sequences 0 and 1 lie behind the bad pages
    check_decode(backend, c, table, slots, q, lens, 40)
    assert backend.device_status() == 0
    out = torch.full_like(q, float("nan"))
    backend.attention_paged(q, c, out, table, torch.tensor([16, 3, 80], dtype=torch.int32, device=dev), max_context=48)
    assert backend.device_status() == 2
    assert (out[2] == 0).all() and torch.isfinite(out).all()


def test_decode_same_result_every_time(backend):
    """The same call gives the same bits, whatever ran between, and on another stream."""
    g = gen(11)
    lens = [5000, 1, 777]
    c, table, slots = paged_batch(g, lens, 64, 2, 128)
    q = torch.randn((3, 1, 8, 128), generator=g, device=dev).bfloat16()
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    outs = []
    for i in range(4):
        out = torch.empty_like(q)
        s = torch.cuda.Stream() if i % 2 else torch.cuda.current_stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            backend.attention_paged(q, c, out, table, ctx, 5000)
        torch.cuda.current_stream().wait_stream(s)
        outs.append(out)
    assert all(torch.equal(outs[0], o) for o in outs)


def test_decode_step_in_a_graph(backend):
    """Append and attention captured once and replayed while the lengths, slots and pages change on the device."""
    g = gen(12)
    B, H, KV, page, pages = 3, 8, 2, 16, 8
    c = garbage_cache(g, B * pages, page, KV, 128)
    table = torch.randperm(B * pages, generator=g, device=dev).int().view(B, pages)
    lens = [15, 40, 0]
    hist = []
    for b, n in enumerate(lens):
        t = torch.arange(n, device=dev)
        hist.append(table[b].long()[t // page] * page + t % page)
        if n:
            fill(g, c, hist[b])
    cos, sin = tables(64, rows=256)
    ctx = torch.tensor(lens, dtype=torch.int32, device=dev)
    q, k, v = (torch.zeros((B, h, 128), device=dev, dtype=torch.bfloat16) for h in (H, KV, KV))
    slots, pos = torch.zeros(B, dtype=torch.int64, device=dev), torch.zeros(B, dtype=torch.int32, device=dev)
    q_rot, out = torch.empty_like(q), torch.empty_like(q)

    def step():
        pos.copy_(ctx)
        slots.copy_(table.long()[torch.arange(B, device=dev), (ctx // page).long()] * page + ctx % page)
        backend.rope_append_paged(k, v, c, slots, cos, sin, pos, q, q_rot)
        ctx.add_(1)
        backend.attention_paged(q_rot[:, None], c, out[:, None], table, ctx, pages * page)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    saved = snapshot(c), ctx.clone()
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    for w, t in saved[0].items():
        getattr(c, w).copy_(t)
    ctx.copy_(saved[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(5):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g, device=dev))
        graph.replay()
        torch.cuda.synchronize()
        for b in range(B):
            n = lens[b] + i + 1
            t = torch.arange(n, device=dev)
            mine = table[b].long()[t // page] * page + t % page
            kk, vv = (ref.cache_rows(c, mine, w) for w in "kv")
            want, spread, mag = ref.attend(q_rot[b][None].double(), kk, vv, n - 1)
            err = (out[b][None].double() - want).abs()
            assert (err <= ref.attention_bound(want, spread, mag, 128, n, torch.bfloat16)).all()
    assert backend.device_status() == 0


# ---- as a serving loop uses them ------------------------------------------------
def test_serving_loop(backend):
    """Packed prompts are rotated, appended and prefilled; a later prompt shares a cached prefix, which is read back and
    attended in front of its own tokens; then every sequence decodes a few tokens.  Each step against 64 bits."""
    g = gen(13)
    H, KV, Dh, page, pages = 8, 2, 128, 16, 12
    dt = torch.bfloat16
    lens = [70, 1, 33]
    B = len(lens)
    c = garbage_cache(g, (B + 1) * pages, page, KV, Dh)
    table = torch.randperm((B + 1) * pages, generator=g, device=dev).int().view(B + 1, pages)
    cos, sin = tables(64, rows=256)

    def slots_of(b, lo, hi):
        t = torch.arange(lo, hi, device=dev)
        return table[b].long()[t // page] * page + t % page

    def bound(want, spread, mag, n, p_step):
        return ref.attention_bound(want, spread, mag, Dh, n, dt, p_step)

    n = sum(lens)
    x = torch.randn((n, H + 2 * KV, Dh), generator=g, device=dev).to(dt)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    pos = torch.cat([torch.arange(m, device=dev, dtype=torch.int32) for m in lens])
    q_rot, k_rot = torch.empty((n, H, Dh), device=dev, dtype=dt), torch.empty((n, KV, Dh), device=dev, dtype=dt)
    backend.rope_append_paged(k, v, c, torch.cat([slots_of(b, 0, m) for b, m in enumerate(lens)]), cos, sin, pos, q, q_rot, k_rot)
    cu = torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device=dev)
    out = torch.empty_like(q_rot)
    backend.prefill_varlen(q_rot, k_rot, v, out, cu)
    for b, m in enumerate(lens):
        sl = slice(int(cu[b]), int(cu[b + 1]))
        want, spread, mag = ref.attend(q_rot[sl].double(), k_rot[sl].double(), v[sl].double(), 0)
        assert ((out[sl].double() - want).abs() <= bound(want, spread, mag, m, 2.0 ** -8)).all()

    # sequence 3 shares the first 48 tokens (three whole pages) of sequence 0 and brings 20 of its own
    table[3, :3] = table[0, :3]
    pk, pv = (torch.empty((48, KV, Dh), device=dev, dtype=dt) for _ in range(2))
    backend.read_paged(c, slots_of(3, 0, 48), pk, pv)
    x = torch.randn((20, H + 2 * KV, Dh), generator=g, device=dev).to(dt)
    q2, k2 = torch.empty((20, H, Dh), device=dev, dtype=dt), torch.empty((20, KV, Dh), device=dev, dtype=dt)
    backend.rope_append_paged(x[:, H:H + KV], x[:, H + KV:], c, slots_of(3, 48, 68), cos, sin,
                              torch.arange(48, 68, device=dev, dtype=torch.int32), x[:, :H], q2, k2)
    keys, vals = torch.cat([pk, k2]), torch.cat([pv, x[:, H + KV:]])
    out2 = torch.empty_like(q2)
    backend.prefill_varlen(q2, keys, vals, out2, torch.tensor([0, 20], dtype=torch.int32, device=dev),
                           torch.tensor([0, 68], dtype=torch.int32, device=dev))
    want, spread, mag = ref.attend(q2.double(), keys.double(), vals.double(), 48)
    assert ((out2.double() - want).abs() <= bound(want, spread, mag, 68, 2.0 ** -8)).all()

    ctx = lens + [68]
    for _ in range(18):  # page borders are crossed
        x = torch.randn((4, H + 2 * KV, Dh), generator=g, device=dev).to(dt)
        q1 = torch.empty((4, H, Dh), device=dev, dtype=dt)
        backend.rope_append_paged(x[:, H:H + KV], x[:, H + KV:], c, torch.cat([slots_of(b, m, m + 1) for b, m in enumerate(ctx)]),
                                  cos, sin, torch.tensor(ctx, dtype=torch.int32, device=dev), x[:, :H], q1)
        ctx = [m + 1 for m in ctx]
        check_decode(backend, c, table, [slots_of(b, 0, m) for b, m in enumerate(ctx)], q1[:, None], ctx, 0, pages * page if _ % 2 else max(ctx))
    assert backend.device_status() == 0


# ---- refusals --------------------------------------------------------------------
def test_c_refusals(backend):
    """What the C entry points refuse, each with its status and nothing launched."""
    import ctypes

    from hachiue_b200 import _lib
    L, h = backend.lib, backend._h
    c = PagedKVCache.allocate(4, 16, 2, 128)
    q = torch.zeros((1, 1, 4, 128), device=dev)
    table, ctx = torch.zeros((1, 4), dtype=torch.int32, device=dev), torch.ones(1, dtype=torch.int32, device=dev)
    kv = c.c_struct()

    def attn(status, kvs=None, qp=q.data_ptr(), **over):
        p = _lib.hcu_attention_paged_params(1, 1, 4, 0, _lib.DT_F32, 64, 4, table.data_ptr(), ctx.data_ptr())
        for name, value in over.items():
            setattr(p, name, value)
        st = _lib.hcu_paged_kv.from_buffer_copy(kv)
        for name, value in (kvs or {}).items():
            setattr(st, name, value)
        assert L.hcu_attention_paged(h, ctypes.byref(p), qp, ctypes.byref(st), q.data_ptr()) == status, (over, kvs)

    attn(0)
    attn(0, batch=0)
    for over in (dict(S=0), dict(H=0), dict(H=3), dict(dtype=7), dict(max_context=65), dict(block_table=None),
                 dict(context=None), dict(batch=70000), dict(windowSize=2 ** 31)):
        attn(1, **over)
    for over in (dict(page_size=24), dict(page_size=8), dict(page_size=512), dict(n_pages=0), dict(KV=0), dict(k=None),
                 dict(v_scale=None), dict(k=c.k.data_ptr() + 8)):
        attn(1, over)
    attn(6, dict(format=_lib.KV_Q8_0))
    attn(6, dict(Dh=64))
    attn(1, qp=None)
    attn(1, qp=q.data_ptr() + 4)

    x = torch.zeros((2, 2, 128), device=dev)
    slots, pos = torch.zeros(2, dtype=torch.int64, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    cos, sin = tables(64)

    def append(status, kp=x.data_ptr(), qo=None, ko=None, pp=pos.data_ptr(), **over):
        p = _lib.hcu_rope_append_params(2, 0, _lib.DT_F32, 128, 64, 0, 0, 0)
        for name, value in over.items():
            setattr(p, name, value)
        got = L.hcu_rope_append_paged(h, ctypes.byref(p), None, kp, x.data_ptr(), cos.data_ptr(), sin.data_ptr(), pp,
                                      slots.data_ptr(), qo, ko, ctypes.byref(kv))
        assert got == status, over

    append(0, n=0)
    for over in (dict(rotaryDim=12), dict(rotaryDim=136), dict(dtype=9), dict(H=2), dict(k_row_stride=258),
                 dict(v_row_stride=128), dict(kp=None), dict(pp=None), dict(kp=x.data_ptr() + 4),
                 dict(ko=x.data_ptr(), k_row_stride=512)):
        append(1, **over)
    assert L.hcu_read_paged(h, 2, _lib.DT_F32, slots.data_ptr(), ctypes.byref(kv), x.data_ptr(), None) == 1
    assert L.hcu_read_paged(h, 2, 5, slots.data_ptr(), ctypes.byref(kv), x.data_ptr(), x.data_ptr()) == 1
    assert L.hcu_read_paged(h, 0, _lib.DT_F32, None, ctypes.byref(kv), None, None) == 0
    backend.inject_failure(2)
    with pytest.raises(HachiueError):
        backend.attention_paged(q, c, q.clone(), table, ctx)
    assert backend.device_status() == 0
