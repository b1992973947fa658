"""The paged-serving operators where a call is unusual: buffers past 2^32 bytes, little workspace, options, nothing to do,
pages held twice, queries and rows that are not finite, many rows or sequences, and two handles at once."""
import numpy as np
import pytest
import torch

from hachiue_b200 import CudaBackend, HachiueError, PagedKVCache
from tests import paged_reference as ref
from tests.test_paged_gpu import check_decode, check_rows, fill, gen, garbage_cache, paged_batch, tables
from tests.test_prefill_varlen_gpu import check, offsets

pytestmark = pytest.mark.gpu
dev = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def test_pages_past_4_gib(backend):
    """A sequence whose pages lie all over a cache of 5 GiB of key codes (and as much of values)."""
    g = gen(1)
    n_pages, page, KV, n = 40960, 256, 8, 900
    c = PagedKVCache.allocate(n_pages, page, KV, 128)
    assert c.k.numel() > 2 ** 32
    table = i32([[n_pages - 1, 3, 33000, n_pages - 2]])
    t = torch.arange(n, device=dev)
    slots = table[0].long()[t // page] * page + t % page
    k, v = (torch.randn((n, KV, 128), generator=g, device=dev).bfloat16() for _ in range(2))
    backend.rope_append_paged(k, v, c, slots)
    code, d = ref.quantise(k.float())
    p, off = slots // page, slots % page
    assert torch.equal(c.k[p, :, off], ref.pack(code, ref.key_nibble(128))) and torch.equal(c.k_scale[p, :, off], d)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    backend.read_paged(c, slots, ko, vo)
    assert torch.equal(vo, ref.cache_rows(c, slots, "v").bfloat16())
    q = torch.randn((1, 1, 16, 128), generator=g, device=dev).bfloat16()
    check_decode(backend, c, table, [slots], q, [n], 0)
    assert backend.device_status() == 0


def test_token_rows_past_4_gib(backend):
    """A batch padded to 270000 rows of a fused projection, of which the last 700 are tokens: their append, and the packed
    attention of two sequences behind 2^31 elements."""
    g = gen(2)
    n, m, H, KV = 270000, 700, 64, 8
    x = torch.zeros((n, H + 2 * KV, 128), device=dev, dtype=torch.bfloat16)
    assert (n - m) * H * 128 > 2 ** 31
    x[n - m:] = torch.randn((m, H + 2 * KV, 128), generator=g, device=dev).bfloat16()
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    c = garbage_cache(g, 50, 16, KV, 128)
    before = {w: getattr(c, w).clone() for w in ("k", "v", "k_scale", "v_scale")}
    slots = torch.full((n,), -1, dtype=torch.int64, device=dev)
    slots[n - m:] = torch.randperm(800, generator=g, device=dev)[:m]
    pos = torch.full((n,), 10 ** 9, dtype=torch.int32, device=dev)  # of padding: not looked at
    pos[n - m:] = torch.arange(m, device=dev) % 64
    cos, sin = tables(64)
    q_out = torch.empty((n, H, 128), device=dev, dtype=torch.bfloat16)
    k_out = torch.empty((n, KV, 128), device=dev, dtype=torch.bfloat16)
    backend.rope_append_paged(k, v, c, slots, cos, sin, pos, q, q_out, k_out)
    assert backend.device_status() == 0
    at = pos[n - m:].long()
    cr, sr = cos.double()[at], sin.double()[at]
    turned = ref.rotate(k[n - m:].double(), cr, sr).float()
    check_rows(c, before, slots[n - m:], turned, v[n - m:].float())
    assert torch.equal(k_out[n - m:], turned.bfloat16())
    size = ref.rotate(q[n - m:].double().abs(), cr.abs(), -sr.abs())
    size[..., 64:] = ref.rotate(q[n - m:].double().abs(), cr.abs(), sr.abs())[..., 64:]
    want = ref.rotate(q[n - m:].double(), cr, sr)
    assert ((q_out[n - m:].double() - want).abs() <= 3 * 2.0 ** -24 * size + 2.0 ** -8 * 1.01 * want.abs() + 2.0 ** -25).all()
    out = torch.full_like(q_out, 7.0)
    cu = i32([n - m, n - 300, n])
    backend.prefill_varlen(q, k, v, out, cu)
    assert backend.device_status() == 0
    assert (out[:n - m] == 7.0).all()
    check(out, q, k, v, cu, cu, 0, torch.bfloat16)


def test_little_workspace():
    """Without room for partial sums every unit is one warp's; a list of blocks that does not fit is refused."""
    be = CudaBackend(0, workspace_bytes=(1 << 18) + 4096)
    try:
        g = gen(3)
        for dtype, H, KV, S, window, lens in ((torch.bfloat16, 8, 2, 1, 0, [700, 64, 1, 0, 129] * 20), (torch.float32, 12, 2, 2, 50, [900, 3]),
                                              (torch.float16, 16, 1, 3, 0, [333])):
            c, table, slots = paged_batch(g, lens, 32, KV, 128)
            q = torch.randn((len(lens), S, H, 128), generator=g, device=dev).to(dtype)
            check_decode(be, c, table, slots, q, lens, window)
        q, k, v = (torch.randn((500, h, 128), generator=g, device=dev).bfloat16() for h in (4, 2, 2))
        out, cu = torch.empty_like(q), offsets([200, 300])
        be.prefill_varlen(q, k, v, out, cu)
        check(out, q, k, v, cu, cu, 0, torch.bfloat16)
        q = torch.zeros((50000, 4, 128), device=dev, dtype=torch.bfloat16)
        with pytest.raises(HachiueError, match="workspace"):
            be.prefill_varlen(q, q[:, :1], q[:, :1], torch.empty_like(q), offsets([50000]))
        assert be.device_status() == 0
    finally:
        be.close()


@pytest.mark.parametrize("H,KV,Dh", [(8, 8, 128), (16, 2, 128), (4, 2, 256), (16, 2, 256)])
def test_long_sums_have_no_bias(H, KV, Dh):
    """f32 sums over 16384 tokens by one warp.  1024 additions that round to nearest are off by u / sqrt(3) of the sum each
    (u = 2^-24), sqrt(1024 / 3) u / sqrt(3) = 11 u together for values of one sign; three times that, and a few steps for
    scores of 0.1.  Additions that truncate would be off by some 500 u."""
    be = CudaBackend(0, workspace_bytes=(1 << 18) + 4096)
    try:
        g = gen(H + Dh)
        n = 16384
        c = PagedKVCache.allocate(n // 64, 64, KV, Dh)
        for t in (c.k, c.v):
            t.copy_(torch.randint(0, 256, t.shape, generator=g, device=dev, dtype=torch.uint8))
        c.v.bitwise_or_(0x88)  # codes from 8 to 15
        for t in (c.k_scale, c.v_scale):
            t.copy_(torch.rand(t.shape, generator=g, device=dev) * 0.2 + 0.05)
        q = torch.randn((1, 1, H, Dh), generator=g, device=dev) * 0.01
        out = torch.empty_like(q)
        table = torch.randperm(n // 64, generator=g, device=dev).int()[None]
        be.attention_paged(q, c, out, table, i32([n]))
        t = torch.arange(n, device=dev)
        slots = table[0].long()[t // 64] * 64 + t % 64
        k, v = (ref.cache_rows(c, slots, w) for w in "kv")
        want = ref.attend(q[0].double(), k, v, n - 1)[0]
        assert float((out[0].double() - want).norm() / want.norm()) < (33 + 8) * 2.0 ** -24
    finally:
        be.close()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,KV,Dh,S", [(4, 2, 128, 1), (16, 1, 128, 1), (12, 2, 256, 2)])
@pytest.mark.parametrize("lens", [[32], [33, 1], [256, 255, 0], [290, 512], [513, 40, 1000], [1024], [1025], [2047], [2048, 5, 31, 32],
                                  [2049], [1024] * 40 + [0, 7]])
def test_short_contexts(backend, dtype, H, KV, Dh, S, lens):
    """Around the lengths at which a unit's cluster grows, and where the work goes over to equal pieces."""
    g = gen(H + Dh + sum(lens))
    c, table, slots = paged_batch(g, lens, 32, KV, Dh)
    q = torch.randn((len(lens), S, H, Dh), generator=g, device=dev).to(dtype)
    check_decode(backend, c, table, slots, q, lens, 0)
    check_decode(backend, c, table, slots, q, lens, 77)
    assert backend.device_status() == 0


@pytest.fixture(scope="module")
def little():
    """A handle without room for partial sums."""
    be = CudaBackend(0, workspace_bytes=(1 << 18) + 4096)
    yield be
    be.close()


@pytest.mark.parametrize("pieces", ["line", "warps"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
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
def test_short_contexts_in_other_pieces(backend, little, pieces, dtype, H, KV, Dh, S, window, page, lens):
    """Short contexts by equal pieces of a line (as long ones are), and with whole units for warps."""
    be = backend if pieces == "line" else little
    g = gen(H * 5 + Dh + S + sum(lens))
    c, table, slots = paged_batch(g, lens, page, KV, Dh)
    q = torch.randn((len(lens), S, H, Dh), generator=g, device=dev).to(dtype)
    be.set_option("attn_chunk", 64)  # a set one keeps the call from taking clusters
    try:
        out = check_decode(be, c, table, slots, q, lens, window)
    finally:
        be.set_option("attn_chunk", 0)
    for b, n in enumerate(lens):
        assert (out[b, :max(0, S - n)] == 0).all()
    assert be.device_status() == 0


@pytest.mark.parametrize("chunk", [1, 32, 100, 4096, 2 ** 40])
def test_chunk_option(backend, chunk):
    g = gen(4)
    lens = [3000, 17, 0, 650]
    c, table, slots = paged_batch(g, lens, 16, 2, 128)
    q = torch.randn((4, 1, 8, 128), generator=g, device=dev)
    backend.set_option("attn_chunk", chunk)
    try:
        check_decode(backend, c, table, slots, q, lens, 0)
        check_decode(backend, c, table, slots, q.bfloat16(), lens, 200)
    finally:
        backend.set_option("attn_chunk", 0)
    assert backend.device_status() == 0


@pytest.mark.parametrize("H,KV,ctas", [(6, 2, 1), (5, 1, 3), (8, 2, 2), (7, 7, 5)])
def test_long_chains_of_items(backend, H, KV, ctas):
    """Few CTAs, each with a long list of items of all sizes; groups that divide a tile and that do not."""
    g = gen(H)
    lens = [int(n) for n in np.random.default_rng(H).integers(0, 300, 40)] + [900]
    keys = [n + int(p) for n, p in zip(lens, np.random.default_rng(1).integers(-20, 200, 41))]
    keys = [max(0, n) for n in keys]
    q, k, v = (torch.randn((n, h, 128), generator=g, device=dev).half() for n, h in ((sum(lens), H), (sum(keys), KV), (sum(keys), KV)))
    cu_q, cu_k = offsets(lens), offsets(keys)
    backend.set_option("swa_ctas", ctas)
    try:
        for window in (0, 150):
            out = torch.full_like(q, float("nan"))
            backend.prefill_varlen(q, k, v, out, cu_q, cu_k, window)
            assert backend.device_status() == 0
            check(out, q, k, v, cu_q, cu_k, window, torch.float16)
    finally:
        backend.set_option("swa_ctas", 0)


@pytest.mark.parametrize("H,KV", [(130, 1), (256, 1), (400, 2), (128, 1), (64, 1)])
def test_groups_as_large_as_a_tile(backend, H, KV):
    """More query heads per KV head than a tile has rows, and as many."""
    g = gen(H)
    lens, keys = [3, 1, 0, 9], [200, 1, 5, 9]
    q, k, v = (torch.randn((n, h, 128), generator=g, device=dev).bfloat16() for n, h in ((13, H), (215, KV), (215, KV)))
    out = torch.full_like(q, float("nan"))
    for window in (0, 4):
        backend.prefill_varlen(q, k, v, out, offsets(lens), offsets(keys), window)
        check(out, q, k, v, offsets(lens), offsets(keys), window, torch.bfloat16)
    c, table, slots = paged_batch(g, keys, 16, KV, 128)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        check_decode(backend, c, table, slots, torch.randn((4, 1, H, 128), generator=g, device=dev).to(dtype), keys, 0)
    assert backend.device_status() == 0


def test_many_prompts(backend):
    """A batch of 20000 prompts, most of them empty or a single token."""
    g = gen(11)
    lens = np.random.default_rng(5).choice([0, 1, 1, 2, 5], 20000).tolist()
    lens[7777] = 600
    q, k, v = (torch.randn((sum(lens), h, 128), generator=g, device=dev).half() for h in (2, 1, 1))
    cu = offsets(lens)
    out = torch.full_like(q, float("nan"))
    backend.prefill_varlen(q, k, v, out, cu)
    assert backend.device_status() == 0 and torch.isfinite(out).all()
    ones = torch.tensor([n == 1 for n in lens], device=dev)
    at = cu[:-1][ones].long()
    assert torch.equal(out[at], v[at].expand(-1, 2, -1))  # one key: its value
    lo, hi = int(cu[7770]), int(cu[7785])
    some = cu[7770:7786] - lo
    check(out[lo:hi], q[lo:hi], k[lo:hi], v[lo:hi], some, some, 0, torch.float16)


def test_offsets_that_begin_again(backend):
    """Offsets that go back to 0 time and again name the same rows more often than the tensors have rows: all but the first
    such sequence are skipped, in the first thousand as behind it."""
    g = gen(12)
    q, k, v = (torch.randn((300, h, 128), generator=g, device=dev).bfloat16() for h in (4, 2, 2))
    for cu in ([0, 200] + [0, 0, 200] * 700 + [200, 300], [0] * 1030 + [200, 0, 0, 200, 200, 300]):
        cu = i32(cu)
        out = torch.full_like(q, 7.0)
        backend.prefill_varlen(q, k, v, out, cu)
        assert backend.device_status() == 2
        check(out, q, k, v, i32([0, 200, 300]), i32([0, 200, 300]), 0, torch.bfloat16)
    out = torch.full_like(q, 7.0)
    backend.prefill_varlen(q, k, v, out, i32([-3, -2, 0, 300]), i32([0, 0, 0, 300]))  # negative ones are out of range
    assert backend.device_status() == 2
    check(out, q, k, v, i32([0, 300]), i32([0, 300]), 0, torch.bfloat16)


def test_nothing_to_do(backend):
    c = PagedKVCache.allocate(2, 16, 1, 128)
    q = torch.ones((2, 1, 2, 128), device=dev)
    out = torch.full_like(q, 7.0)
    backend.attention_paged(q, c, out, i32([[], []]), i32([0, 0]))  # a table without pages: empty sequences
    assert (out == 0).all() and backend.device_status() == 0
    backend.attention_paged(q, c, out.fill_(7.0), i32([[], []]), i32([0, 3]))
    assert (out == 0).all() and backend.device_status() == 2
    backend.attention_paged(q[:0], c, out[:0], i32([[0]])[:0], i32([0])[:0])
    x = torch.ones((3, 2, 128), device=dev).half()
    o = torch.full_like(x, 7.0)
    none = x[:0, :1]
    backend.prefill_varlen(x, none, none, o, i32([0, 1, 3]), i32([0, 0, 0]))  # no key at all
    assert (o == 0).all() and backend.device_status() == 0
    backend.prefill_varlen(x, x[:, :1], x[:, :1], o.fill_(7.0), i32([1, 1, 1]))
    backend.prefill_varlen(x, x[:, :1], x[:, :1], o, i32([0]))
    assert (o == 7.0).all() and backend.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_pages_held_twice(backend, dtype):
    """Two sequences over the same pages, and a sequence that holds a page twice."""
    g = gen(5)
    c = garbage_cache(g, 6, 16, 2, 128)
    fill(g, c, torch.arange(4 * 16, device=dev))
    table = i32([[0, 1, 2, 3], [0, 1, 2, 9], [3, 3, 0, 3]])
    lens = [64, 40, 60]
    t = torch.arange(64, device=dev)
    slots = [table[b].long()[t[:n] // 16] * 16 + t[:n] % 16 for b, n in enumerate(lens)]
    q = torch.randn((3, 2, 4, 128), generator=g, device=dev).to(dtype)
    check_decode(backend, c, table, slots, q, lens, 0)
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H", [4, 12])
def test_rows_that_are_not_finite(backend, dtype, H):
    """A query or a visible row that is not finite spoils the results that take it in and no other."""
    g = gen(6)
    lens = [300, 300, 300]
    c, table, slots = paged_batch(g, lens, 16, 2, 128)
    q = torch.randn((3, 1, H, 128), generator=g, device=dev).to(dtype)
    q[0, 0, 1, 5], q[1, 0, H - 1, 7] = float("nan"), float("inf")
    page, off = int(slots[2][77]) // 16, int(slots[2][77]) % 16
    c.k_scale[page, 0, off] = float("nan")
    out = torch.empty_like(q)
    backend.attention_paged(q, c, out, table, i32(lens))
    bad = torch.zeros((3, H), dtype=torch.bool, device=dev)
    bad[0, 1] = bad[1, H - 1] = True
    bad[2, :H // 2] = True
    assert torch.isnan(out[:, 0].float()).all(-1)[bad].all()
    for b, n in enumerate(lens):
        k, v = (torch.nan_to_num(ref.cache_rows(c, slots[b], w)) for w in "kv")
        want, spread, mag = ref.attend(torch.nan_to_num(q[b].double(), posinf=0.0), k, v, n - 1)
        p_step = 2.0 ** -11 if dtype == torch.bfloat16 and H > 8 else 2.0 ** -22
        err = (out[b].double() - want).abs() <= ref.attention_bound(want, spread, mag, 128, n, dtype, p_step)
        assert err[0][~bad[b]].all()
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype,big,small", [(torch.float32, 1e30, 1e-35), (torch.bfloat16, 1e30, 1e-35), (torch.float16, 5e3, 1e-7)])
def test_exponents_of_queries(backend, dtype, big, small):
    """Queries near the ends of their type's range: huge ones pick one token, tiny ones weigh all alike."""
    g = gen(7)
    c, table, slots = paged_batch(g, [200], 16, 2, 128)
    page, off = slots[0] // 16, slots[0] % 16
    c.k_scale[page[50], :, off[50]] *= 8
    k, v = (ref.cache_rows(c, slots[0], w) for w in "kv")
    q = torch.empty((1, 1, 4, 128), device=dev)
    q[0, 0, :2], q[0, 0, 2:] = k[50, 0].sign().float() * big, torch.randn((2, 128), generator=g, device=dev) * small
    q = q.to(dtype)
    out = torch.empty_like(q)
    backend.attention_paged(q, c, out, table, i32([200]))
    half = ref.HALF_STEP[dtype]
    assert ((out[0, 0, :2].double() - v[50, 0]).abs() <= (1.01 * half + 2.0 ** -20) * v[50, 0].abs()).all()
    want = v[:, 1].mean(0)
    # the weights and the sum of 200 tokens: see attention_bound
    assert ((out[0, 0, 2:].double() - want).abs() <= 2.0 ** -18 * v[:, 1].abs().mean(0) + 1.01 * half * want.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_query_rows(backend, dtype):
    """Sixty-four tokens of drafts, 2048 rows per KV head."""
    g = gen(8)
    lens = [130, 64, 63, 1]
    c, table, slots = paged_batch(g, lens, 64, 1, 128)
    q = torch.randn((4, 64, 32, 128), generator=g, device=dev).to(dtype)
    out = check_decode(backend, c, table, slots, q, lens, 0)
    assert (out[3, :63] == 0).all()
    check_decode(backend, c, table, slots, q, lens, 9)
    assert backend.device_status() == 0


def test_many_sequences(backend):
    g = gen(9)
    lens = [int(n) for n in np.random.default_rng(3).integers(0, 20, 3000)]
    lens[1234] = 2000
    c, table, slots = paged_batch(g, lens, 16, 1, 128)
    q = torch.randn((3000, 1, 2, 128), generator=g, device=dev)
    out = torch.full_like(q, float("nan"))
    backend.attention_paged(q, c, out, table, i32(lens))
    assert backend.device_status() == 0
    assert torch.isfinite(out).all()
    pick = [0, 1, 2, 1233, 1234, 1235, 2998, 2999] + list(range(100, 130))
    for b in pick:
        k, v = (ref.cache_rows(c, slots[b], w) for w in "kv")
        want, spread, mag = ref.attend(q[b].double(), k, v, lens[b] - 1)
        assert ((out[b].double() - want).abs() <= ref.attention_bound(want, spread, mag, 128, lens[b], torch.float32)).all(), b
    alone = torch.empty_like(q[pick])
    backend.attention_paged(q[pick], c, alone, table[pick].contiguous(), i32([lens[b] for b in pick]))
    assert float((alone - out[pick]).abs().max()) < 1e-5


def test_two_handles_at_once(backend):
    """Graphs of a handle each, replayed on two streams together, give what each gives alone."""
    g = gen(10)
    other = CudaBackend(0)
    try:
        lens = [4000, 300, 77]
        c, table, slots = paged_batch(g, lens, 64, 2, 128)
        ctx = i32(lens)
        runs = []
        for be in (backend, other):
            q = torch.randn((3, 1, 16, 128), generator=g, device=dev).bfloat16()
            x = [torch.randn((600, h, 128), generator=g, device=dev).bfloat16() for h in (4, 2, 2)]
            cu = offsets([100, 500])
            out, o2 = torch.empty_like(q), torch.empty_like(x[0])

            def step(be=be, q=q, x=x, cu=cu, out=out, o2=o2):
                for _ in range(4):
                    be.attention_paged(q, c, out, table, ctx, 4000)
                    be.prefill_varlen(*x, o2, cu)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                step()
            side.synchronize()
            want = out.clone(), o2.clone()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                step()
            runs.append((graph, side, out, o2, want, step))  # step holds the graph's inputs
        for _ in range(5):
            torch.cuda.synchronize()
            for graph, side, out, o2, *_ in runs:
                out.fill_(7.0), o2.fill_(7.0)
                side.wait_stream(torch.cuda.current_stream())
            for graph, side, *_ in runs:
                with torch.cuda.stream(side):
                    graph.replay()
            torch.cuda.synchronize()
            for _, _, out, o2, want, _ in runs:
                assert torch.equal(out, want[0]) and torch.equal(o2, want[1])
        assert backend.device_status() == 0 and other.device_status() == 0
        del runs, graph
    finally:
        other.close()
