"""The append of whole prompts, whose blocks walk from token to token: bit for bit, as the append of a few tokens is tested."""
import pytest
import torch

from hachiue_b200 import PagedKVCache
from tests import paged_reference as ref
from tests.test_paged_gpu import DTYPES, check_rows, dev, garbage_cache, gen, snapshot, tables

pytestmark = pytest.mark.gpu


def check(backend, dtype, n, H, KV, Dh, rotary, page, fused, in_place, holes):
    g = gen(n + H + Dh + rotary)
    c = garbage_cache(g, -(-n // page) + 3, page, KV, Dh)
    total = c.n_pages * page
    x = torch.randn((n, H + 2 * KV, Dh), generator=g, device=dev).to(dtype)
    q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    if not fused:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    slots = torch.randperm(total, generator=g, device=dev)[:n].clone()
    pos = torch.randint(0, 64, (n,), generator=g, device=dev, dtype=torch.int32)
    written, reported = torch.ones(n, dtype=torch.bool, device=dev), False
    if holes:  # padding, slots past the cache, positions outside of the tables, in any order among the rest
        kind = torch.randint(0, 12, (n,), generator=g, device=dev)
        slots[kind == 0], slots[kind == 1] = -1, total
        slots[kind == 2] = 2 ** 62
        pos[kind == 0] = 2 ** 31 - 1  # of padding: not looked at
        written &= kind > 2
        if rotary:
            pos[kind == 3], pos[kind == 4] = 64, -1
            written &= kind > 4
        reported = True
    cos, sin = tables(rotary // 2) if rotary else (None, None)
    k0, q0 = k.clone(), q.clone()
    if in_place:
        q_out, k_out = q, k
    else:
        q_out, k_out = torch.full((n, H, Dh), 7.0, device=dev, dtype=dtype), torch.full((n, KV, Dh), 7.0, device=dev, dtype=dtype)
    before = snapshot(c)
    backend.rope_append_paged(k, v, c, slots, cos, sin, pos if rotary else None, q if H else None, q_out if H else None, k_out)
    assert backend.device_status() == (2 if reported else 0)
    half = rotary // 2
    cr = cos.double()[pos.long().clamp(0, 63)] if rotary else torch.zeros((n, 0), dtype=torch.float64, device=dev)
    sr = sin.double()[pos.long().clamp(0, 63)] if rotary else cr
    turned = ref.rotate(k0.double(), cr, sr).float()
    check_rows(c, before, slots[written], turned[written], v.float()[written])
    assert torch.equal(k_out[written], turned.to(dtype)[written])
    left_q, left_k = (q0, k0) if in_place else (torch.full_like(q_out, 7.0), torch.full_like(k_out, 7.0))
    assert torch.equal(k_out[~written], left_k[~written]) and torch.equal(q_out[~written], left_q[~written])
    if H:
        want = ref.rotate(q0.double(), cr, sr)
        # two products and a sum in f32, then the rounding to dtype
        size = ref.rotate(q0.double().abs(), cr.abs(), -sr.abs())
        size[..., half:] = ref.rotate(q0.double().abs(), cr.abs(), sr.abs())[..., half:]
        err = (q_out.double() - want).abs()
        assert (err <= 3 * 2.0 ** -24 * size + ref.HALF_STEP[dtype] * 1.01 * want.abs() + 2.0 ** -25)[written].all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,H,KV,Dh,rotary,page,fused,in_place", [
    (4000, 8, 2, 128, 128, 64, True, False), (3001, 6, 3, 128, 64, 16, False, True), (5000, 4, 1, 256, 256, 256, False, False),
    (3000, 4, 2, 256, 200, 32, True, False), (4099, 0, 1, 128, 128, 128, False, False), (3500, 2, 2, 128, 0, 16, True, False),
    (3333, 34, 8, 128, 8, 64, False, True), (700, 16, 2, 256, 64, 16, False, False), (592, 4, 2, 128, 128, 16, False, False),
    (593, 4, 2, 128, 64, 16, True, False), (591, 4, 2, 128, 128, 16, False, True)])
@pytest.mark.parametrize("holes", [False, True])
def test_prompts(backend, dtype, n, H, KV, Dh, rotary, page, fused, in_place, holes):
    check(backend, dtype, n, H, KV, Dh, rotary, page, fused, in_place, holes)


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_of_values_on_borders(backend, dtype):
    """Elements on the borders between levels and next to them, a prompt of them in keys and values."""
    g = gen(6)
    n = 3000
    m = torch.exp2(torch.randint(-6, 7, (n, 2, 4, 1), generator=g, device=dev).float()) * (1 + torch.randint(0, 100, (n, 2, 4, 1), generator=g, device=dev) / 128)
    m = m.to(dtype).float()
    d = (m / -8).half().float()
    level = torch.randint(0, 16, (n, 2, 4, 32), generator=g, device=dev) - 7.5
    x = (level * d).to(dtype).float()
    away = torch.randint(-1, 2, x.shape, generator=g, device=dev)  # in steps of the type
    step = torch.where(away == 0, torch.zeros_like(x), torch.finfo(dtype).eps * x.abs() * away)
    x = (x + step).to(dtype).float()
    x = torch.minimum(torch.maximum(x, -m), m)
    x[..., 5:6] = m
    x = x.flatten(-2).to(dtype)
    c = PagedKVCache.allocate(200, 16, 2, 128)
    before = snapshot(c)
    slots = torch.randperm(3200, generator=g, device=dev)[:n].clone()
    backend.rope_append_paged(x, x, c, slots)
    check_rows(c, before, slots, x.float(), x.float())
    assert backend.device_status() == 0
