"""The decode over the 4-bit pages where its numbers are far apart."""
import pytest
import torch

from hachiue_b200 import CudaBackend
from tests import paged_reference as ref
from tests.test_paged_gpu import dev, gen, paged_batch

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
