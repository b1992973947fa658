"""NaN in what the paged 4-bit cache is given and holds: it stays visible in the results that take it in, and reaches no other."""
import pytest
import torch

from hachiue_b200 import PagedKVCache
from tests import paged_reference as ref
from tests.test_paged_gpu import DTYPES, check_rows, dev, gen, snapshot, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Dh,rotary,n", [(128, 0, 3), (128, 64, 3), (256, 256, 3), (128, 128, 2000)])
def test_append_keeps_nan(backend, dtype, Dh, rotary, n):
    """The block of a NaN element reads back as NaN, in keys (both partners' blocks of a rotated one) and in values; every
    other block is held as ever, and a decode that sees the row gives NaN where the definition does."""
    g = gen(Dh + rotary + n)
    c = PagedKVCache.allocate(-(-n // 16) + 1, 16, 2, Dh)
    before = snapshot(c)
    k, v = (torch.randn((n, 2, Dh), generator=g, device=dev).to(dtype) for _ in range(2))
    clean_k, clean_v = k.clone(), v.clone()
    k[1, 0, 5] = float("nan")
    v[n - 1, 1, Dh - 1], v[0, 1, 40] = float("nan"), -float("nan")
    slots = torch.arange(n, device=dev)
    pos = (slots % 64).int()
    cos, sin = tables(rotary // 2) if rotary else (None, None)
    backend.rope_append_paged(k, v, c, slots, cos, sin, pos if rotary else None)
    ko, vo = (torch.empty((n, 2, Dh), device=dev, dtype=dtype) for _ in range(2))
    backend.read_paged(c, slots, ko, vo)
    bad_k = torch.zeros((n, 2, Dh // 32), dtype=torch.bool, device=dev)
    bad_v = bad_k.clone()
    bad_k[1, 0, 0] = True
    if rotary:
        bad_k[1, 0, (5 + rotary // 2) // 32] = True  # the partner's
    bad_v[n - 1, 1, -1] = bad_v[0, 1, 1] = True
    assert torch.equal(torch.isnan(ko), bad_k.repeat_interleave(32, -1))
    assert torch.equal(torch.isnan(vo), bad_v.repeat_interleave(32, -1))
    assert torch.isnan(c.k_scale[slots // 16, :, slots % 16][bad_k]).all()

    # without those blocks the rows are those of the clean call
    turned = clean_k.double()
    if rotary:
        at = pos.long()
        turned = ref.rotate(turned, cos.double()[at], sin.double()[at])
    got = snapshot(c)
    other = PagedKVCache.allocate(c.n_pages, 16, 2, Dh)
    backend.rope_append_paged(clean_k, clean_v, other, slots, cos, sin, pos if rotary else None)
    check_rows(other, before, slots, turned.float(), clean_v.float())
    for w, bad in (("k", bad_k), ("v", bad_v)):
        rows = lambda t: t[slots // 16, :, slots % 16]  # noqa: E731
        assert torch.equal(rows(got[w + "_scale"])[~bad], rows(getattr(other, w + "_scale"))[~bad])
    for mine, theirs, bad in ((ko, clean_k, bad_k), (vo, clean_v, bad_v)):
        assert torch.isfinite(mine[~bad.repeat_interleave(32, -1)]).all()

    q = torch.randn((1, 1, 4, Dh), generator=g, device=dev).to(dtype)
    out = torch.empty_like(q)
    backend.attention_paged(q, c, out, torch.arange(c.n_pages, device=dev, dtype=torch.int32)[None],
                            torch.tensor([n], dtype=torch.int32, device=dev))
    nan = torch.isnan(out[0, 0])
    assert nan[:2].all()  # a NaN key of their head
    assert torch.equal(nan[2:], (bad_v[0, 1] | bad_v[n - 1, 1]).repeat_interleave(32, -1).expand(2, -1))
    assert backend.device_status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,Dh,S,n", [(2, 2, 128, 2, 40), (8, 2, 128, 2, 300), (8, 1, 128, 4, 100), (2, 2, 128, 8, 70), (6, 2, 128, 3, 50), (16, 2, 256, 4, 333),
                                         (3, 1, 256, 5, 2500)])
@pytest.mark.parametrize("window", [0, 20])
def test_a_draft_that_is_nan(backend, dtype, H, KV, Dh, S, n, window):
    """The last drafted token's key or value row is NaN: the drafts before it do not see it, and with a window the ones
    behind a NaN row do not either."""
    g = gen(H + Dh + S + n + window)
    pages = -(-n // 16)
    c = PagedKVCache.allocate(pages, 16, KV, Dh)
    k, v = (torch.randn((n, KV, Dh), generator=g, device=dev) for _ in range(2))
    slots = torch.arange(n, device=dev)
    q = torch.randn((1, S, H, Dh), generator=g, device=dev).to(dtype)
    table, ctx = torch.arange(pages, device=dev, dtype=torch.int32)[None], torch.tensor([n], dtype=torch.int32, device=dev)
    clean, out = torch.empty_like(q), torch.empty_like(q)
    backend.rope_append_paged(k, v, c, slots)
    backend.attention_paged(q, c, clean, table, ctx, window_size=window)
    at = [n - 1] if not window else [n - 1, n - window - 1]  # the first query's window begins at n - S + 1 - window
    saved = snapshot(c)
    for scales in ("v_scale", "k_scale"):
        rows = getattr(c, scales)
        for i in at:
            rows[i // 16, :, i % 16, 1 if scales == "v_scale" else 0] = float("nan")
        backend.attention_paged(q, c, out, table, ctx, window_size=window)
        for s in range(S):
            pos = n - S + s
            sees = [i for i in at if i <= pos and (not window or i > pos - window)]
            nan = torch.isnan(out[0, s])
            if not sees:
                assert torch.equal(out[0, s], clean[0, s]), (scales, s)
            elif scales == "v_scale":
                assert nan[:, 32:64].all() and not nan[:, :32].any() and not nan[:, 64:].any(), s
            else:
                assert nan.all(), s
        rows.copy_(saved[scales])
    assert backend.device_status() == 0
