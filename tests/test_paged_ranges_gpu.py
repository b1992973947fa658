"""The decode over the 4-bit pages where its numbers are far apart: scores and queries near the ends of f32, value scales that
differ between the blocks of a row and between tokens."""
import pytest
import torch

from hachiue_b200 import CudaBackend
from tests import paged_reference as ref
from tests.test_paged_gpu import DTYPES, check_decode, dev, gen, paged_batch

pytestmark = pytest.mark.gpu


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.fixture(scope="module")
def little():
    """A handle without room for partial sums: whole units for warps."""
    be = CudaBackend(0, workspace_bytes=(1 << 18) + 4096)
    yield be
    be.close()


def runs(backend, little):
    """The three ways in which a call is cut: clusters (or the line, where it is long), the line, whole units for warps."""
    yield backend
    backend.set_option("attn_chunk", 64)
    try:
        yield backend
    finally:
        backend.set_option("attn_chunk", 0)
    yield little


def check(be, c, table, slots, q, lens, window=0, without=None, blocks=False):
    """As check_decode, with the step of f16's smallest numbers; token `without` has no weight, so that its own score's
    error says nothing about the others'.

    `blocks`: an element is held to the size of its block, sum_j p_j 8 |d_j|, not to its own, sum_j p_j |v_j|.  Where the
    token that takes nearly all has code 8 (a zero) the second one is the sum of the others alone, which the arithmetic does
    not resolve to 22 bits: a weight w is two f16 numbers, off by 2^-22 w or, below 2^-2, by up to 2^-24, and the largest
    weight W of the row and block is at least 2^8: T weights are off by at most T 2^-32 W (times 8, their largest code),
    below the T / 16 steps of 2^-24 of the bound.  16-bit calls add codes and their offset inside the tensor cores, of which
    each sum of 16 tokens truncates twice, by 2^-23 of at most 15 / 8 of the block's size: T / 16 * 7.5 steps, below the
    2 (D + 8) mag steps of a bound whose scores reach 40."""
    out = torch.full_like(q, float("nan"))
    be.attention_paged(q, c, out, table, i32(lens), window_size=window)
    S, D = q.shape[1], q.shape[3]
    for b, n in enumerate(lens):
        k, v = (ref.cache_rows(c, slots[b], w) for w in "kv")
        want, spread, mag = ref.attend(q[b].double(), k, v, n - S, window)
        if blocks:
            page, off = slots[b] // c.page_size, slots[b] % c.page_size
            size = 8 * c.v_scale[page, :, off].double().abs().repeat_interleave(32, -1)
            spread = ref.attend(q[b].double(), k, size, n - S, window)[0]
            assert n / 16 * 7.5 < 2 * (D + 8) * float(mag.min())
        if without is not None:
            k[without] = 0
            mag = ref.attend(q[b].double(), k, v, n - S, window)[2]
        rows = S * q.shape[2] // c.kv_heads
        p_step = 2.0 ** -11 if q.dtype == torch.bfloat16 and rows > 4 else 2.0 ** -22
        bound = ref.attention_bound(want, spread, mag, D, n, q.dtype, p_step) + (2.0 ** -25 if q.dtype == torch.float16 else 0)
        err = (out[b].double() - want).abs()
        assert (err <= bound).all(), (b, n, float((err / bound).max()), float(err.max()))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H,Dh,S", [(2, 128, 1), (8, 128, 1), (12, 128, 1), (2, 256, 2), (8, 256, 1)])
def test_scores_far_below_zero(backend, little, dtype, H, Dh, S):
    """Rows whose every score is finite and hugely negative: the one nearest to zero takes all, in a context of one token as
    in one that is joined from many parts."""
    g = gen(H + Dh)
    lens = [S, 1, 200, 3000]
    c, table, slots = paged_batch(g, lens, 16, 1, Dh)
    c.k.bitwise_or_(0x88)  # codes from 8 on, under positive scales: no key element is negative
    c.k_scale.copy_(c.k_scale.abs())
    for b in range(len(lens)):
        page, off = int(slots[b][0]) // 16, int(slots[b][0]) % 16
        c.k_scale[page, :, off] *= 0.25  # the first token's scores are the nearest to zero
    for be in runs(backend, little):
        for big in (1e3, 1e20, 1e30, 1e33):
            q = torch.full((4, S, H, Dh), -big, device=dev).to(dtype)
            out = torch.full_like(q, float("nan"))
            be.attention_paged(q, c, out, table, i32(lens))
            for b, n in enumerate(lens):
                k, v = (ref.cache_rows(c, slots[b], w)[:, 0] for w in "kv")
                x = k @ q[b, 0, 0].double() / Dh ** 0.5
                assert x.abs().max() < 3e38 and x[0] < 0 and (x[1:] < x[0] - 100).all()
                for s in range(S):
                    want = v[0] if n - S + s >= 0 else torch.zeros_like(v[0])
                    err = (out[b, s].double() - want).abs()
                    assert (err <= (1.01 * ref.HALF_STEP[dtype] + 2.0 ** -20) * want.abs()).all(), (big, b, s)
    assert backend.device_status() == 0 and little.device_status() == 0


@pytest.mark.parametrize("H,Dh,S", [(2, 128, 1), (8, 128, 1), (12, 128, 1), (2, 256, 2), (8, 256, 1)])
def test_negative_scores_alone(backend, little, H, Dh, S):
    """All tokens of a long context have the same key and a score of -1e31: every one weighs the same."""
    g = gen(H)
    lens = [700, 37]
    c, table, slots = paged_batch(g, lens, 16, 1, Dh)
    for b in range(2):
        page, off = slots[b] // 16, slots[b] % 16
        c.k[page, :, off] = c.k[page[0], :, off[0]].clone()
        c.k_scale[page, :, off] = c.k_scale[page[0], :, off[0]].clone()
    for dtype in (torch.float32, torch.bfloat16):
        q = torch.empty((2, S, H, Dh), device=dev)
        for b in range(2):
            q[b] = -1e30 * ref.cache_rows(c, slots[b][:1], "k")[0, 0].sign().float()
        q = q.to(dtype)
        for be in runs(backend, little):
            out = torch.empty_like(q)
            be.attention_paged(q, c, out, table, i32(lens))
            for b, n in enumerate(lens):
                v = ref.cache_rows(c, slots[b], "v")[:, 0]
                for s in range(S):
                    mean, size = v[:n - S + s + 1].mean(0), v[:n - S + s + 1].abs().mean(0)
                    # weights of 2^-11 (bf16, more than four rows) or 2^-22, the sum of n tokens and the division
                    step = 2.0 ** -11 if dtype == torch.bfloat16 and S * H > 4 else 2.0 ** -18
                    assert ((out[b, s].double() - mean).abs() <= step * size + 1.01 * ref.HALF_STEP[dtype] * mean.abs()).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("H", [2, 8, 12])
def test_largest_queries(backend, dtype, H):
    """Queries of 2^126 over the smallest scales that f16 holds: finite scores, the largest take all."""
    g = gen(H + 1)
    c, table, slots = paged_batch(g, [90], 16, 1, 128)
    page, off = slots[0] // 16, slots[0] % 16
    c.k_scale[page, :, off] = torch.randint(1, 6, (90, 1, 4), generator=g, device=dev).half() * 2.0 ** -24
    q = torch.zeros((1, 1, H, 128), device=dev)
    q[..., 3] = 2.0 ** 126
    q = q.to(dtype)
    out = torch.empty_like(q)
    backend.attention_paged(q, c, out, table, i32([90]))
    x = ref.cache_rows(c, slots[0], "k")[:, 0, 3]
    v = ref.cache_rows(c, slots[0], "v")[:, 0][x == x.max()]
    bound = ref.HALF_STEP[dtype] * 1.01 * v.mean(0).abs() + (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -20) * v.abs().mean(0)
    assert ((out[0, 0].double() - v.mean(0)).abs() <= bound).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,Dh,S", [(4, 2, 128, 1), (16, 2, 128, 1), (24, 2, 128, 1), (6, 2, 256, 1), (16, 2, 256, 2)])
@pytest.mark.parametrize("apart", [10, 18, 24])
def test_value_scales_of_blocks(backend, little, dtype, H, KV, Dh, S, apart):
    """One block of every value row is 2^apart times as large as the others, another 2^-8 of those: each block's results
    keep the accuracy of their own size."""
    g = gen(H + Dh + apart)
    lens = [900, 33, 1]
    c, table, slots = paged_batch(g, lens, 32, KV, Dh)
    every = torch.cat(slots)
    page, off = every // 32, every % 32
    size = torch.full((Dh // 32,), 2.0 ** (8 - apart), device=dev)
    size[1], size[2] = 2.0 ** 8, 2.0 ** -apart
    c.v_scale[page, :, off] = ((torch.rand((len(every), KV, Dh // 32), generator=g, device=dev) + 0.5) * size).half()
    q = torch.randn((3, S, H, Dh), generator=g, device=dev).to(dtype)
    for be in runs(backend, little):
        check(be, c, table, slots, q, lens)
        check(be, c, table, slots, q, lens, 100)
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,Dh", [(4, 2, 128), (16, 2, 128), (24, 2, 128), (6, 2, 256), (16, 2, 256)])
@pytest.mark.parametrize("at", [0, 17, 450, 899])
@pytest.mark.parametrize("blocks", [slice(None), 1], ids=["all", "one"])
def test_a_large_token_of_no_weight(backend, little, dtype, H, KV, Dh, at, blocks):
    """A token whose values (all, or those of one block) are 2^27 times the others' has a probability near 2^-50: it adds
    nothing, wherever it lies, and takes nothing from the accuracy of the rest."""
    g = gen(H + Dh + at)
    lens = [900]
    c, table, slots = paged_batch(g, lens, 32, KV, Dh)
    page, off = slots[0] // 32, slots[0] % 32
    c.v_scale[page, :, off] = ((torch.rand((900, KV, Dh // 32), generator=g, device=dev) + 0.5) * 2.0 ** -12).half()
    c.v_scale[page[at], :, off[at], blocks] = 2.0 ** 15
    k = ref.cache_rows(c, slots[0], "k")
    G = H // KV
    q = torch.empty((1, 1, H, Dh), device=dev)
    for h in range(H):  # a score near -35 with that token, and a random one with the others
        u = k[at, h // G].float()
        q[0, 0, h] = torch.randn(Dh, generator=g, device=dev) * 0.3 - 35 * Dh ** 0.5 * u / (u * u).sum()
    for be in runs(backend, little):
        check(be, c, table, slots, q.to(dtype), lens, without=at)
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,Dh", [(4, 2, 128), (16, 2, 128), (24, 2, 128), (16, 2, 256)])
def test_scales_and_scores_that_grow(backend, little, dtype, H, KV, Dh):
    """Scores and value scales that grow along the context, each block's at its own pace, so that references move often."""
    g = gen(H + Dh + 5)
    n = 1500
    c, table, slots = paged_batch(g, [n], 32, KV, Dh)
    page, off = slots[0] // 32, slots[0] % 32
    t = torch.arange(n, device=dev)[:, None, None] / n
    pace = torch.linspace(-20, 20, Dh // 32, device=dev)
    c.v_scale[page, :, off] = torch.exp2(pace * t - 10 - pace.clamp_min(0) / 2).expand(-1, KV, -1).half()
    c.k_scale[page, :, off] = (c.k_scale[page, :, off].float() * (0.1 + 4 * t)).half()
    q = torch.randn((1, 1, H, Dh), generator=g, device=dev)
    q[0, 0, 1:] += ref.cache_rows(c, slots[0], "k")[n - 1, 0].float() * 0.3
    for be in runs(backend, little):
        check(be, c, table, slots, q.to(dtype), [n], blocks=True)
    assert backend.device_status() == 0


@pytest.mark.parametrize("bad", [-1, -2, -3, -(2 ** 31), 2 ** 31 - 1])
@pytest.mark.parametrize("page", [16, 64])
def test_every_bad_page_is_reported(backend, bad, page):
    g = gen(page)
    c, table, slots = paged_batch(g, [200], page, 2, 128)
    q = torch.randn((1, 1, 4, 128), generator=g, device=dev)
    table[0, 1] = bad
    missing = torch.zeros(200, dtype=torch.bool, device=dev)
    missing[page:2 * page] = True
    check_decode(backend, c, table, slots, q, [200], 0, missing=[missing])
    assert backend.device_status() == 2


@pytest.mark.parametrize("window", [0, 2 ** 31 - 500, 2 ** 31 - 257, 2 ** 31 - 1])
def test_windows_near_the_largest_context(backend, window):
    """A table of 2^31 - 256 tokens a row (its one page again and again), whose sequences hold fewer tokens than the call has
    queries: a window near 2^31 hides nothing, and what there is is seen."""
    g = gen(window % 97)
    S, page = 700, 256
    c, table, slots = paged_batch(g, [200, 256], page, 1, 128, spare=0)
    wide = table[:, :1].expand(2, 2 ** 31 // page - 1).contiguous()
    q = torch.randn((2, S, 2, 128), generator=g, device=dev)
    out = torch.full_like(q, float("nan"))
    backend.attention_paged(q, c, out, wide, i32([200, 256]), 2 ** 31 - 256, window)
    plain = torch.full_like(q, float("nan"))
    backend.attention_paged(q, c, plain, table, i32([200, 256]))
    assert backend.device_status() == 0
    for b, n in enumerate((200, 256)):
        assert (out[b, :S - n] == 0).all()
        k, v = (ref.cache_rows(c, slots[b], w) for w in "kv")
        want, spread, mag = ref.attend(q[b].double(), k, v, n - S)
        for got in (out, plain):
            assert ((got[b].double() - want).abs() <= ref.attention_bound(want, spread, mag, 128, n, torch.float32)).all()
