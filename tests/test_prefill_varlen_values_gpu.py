"""The packed prefill over values that are not finite or nearly overflow: rows keep what they see, and only that."""
import math

import pytest
import torch

from tests import paged_reference as ref
from tests.test_prefill_varlen_gpu import DTYPES, check, dev, gen, offsets

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def expect(q, k, v, window=0):
    """The definition in 64 bits where values may be anything: a key that a query does not see is left out, not weighted by
    zero.  q [S, H, D], k and v [T, KV, D]."""
    S, H, D = q.shape
    T, KV, _ = k.shape
    out = torch.zeros((S, H, D), dtype=torch.float64, device=q.device)
    for s in range(S):
        pos = T - S + s
        lo = max(0, pos + 1 - window) if window else 0
        if pos < lo:
            continue
        kk, vv = (x[lo:pos + 1].double().repeat_interleave(H // KV, 1) for x in (k, v))
        x = torch.einsum("hd,thd->ht", q[s].double(), kk) / math.sqrt(D)
        p = torch.softmax(x, -1)
        out[s] = (p.t()[..., None] * vv).sum(0)
    return out


def compare(out, want, dtype):
    """Not finite in the same places, and elsewhere within the roundings of P and of the result (32 steps of f32 beside)."""
    got = out.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    ok = torch.isfinite(want)
    size = want[ok].abs().max() if ok.any() else 0.0
    assert ((got - want)[ok].abs() <= 4 * ref.HALF_STEP[dtype] * size).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,window", [(4, 2, 0), (3, 1, 0), (4, 2, 60), (6, 3, 200), (2, 2, 1)])
def test_values_that_are_not_finite(backend, dtype, H, KV, window):
    """Single elements and whole rows of v, before, in the middle of and behind what a query sees: a query takes in those of
    its own keys in their own dimensions, and no other."""
    g = gen(H + window)
    n = 400
    q, k, v = (torch.randn((n, h, 128), generator=g, device=dev).to(dtype) for h in (H, KV, KV))
    v[3, 0, 7], v[130, 0, 8], v[131, KV - 1, 9], v[300, 0] = NAN, INF, -INF, NAN
    out = torch.empty_like(q)
    backend.prefill_varlen(q, k, v, out, offsets([n]), window=window)
    assert backend.device_status() == 0
    compare(out, expect(q, k, v, window), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 40])
def test_scores_that_are_not_finite(backend, dtype, window):
    """Keys and queries that are not finite: a score of -infinity weighs nothing beside finite ones, whichever comes first and
    with a later value that is not finite in the same tile; rows of nothing but -infinity, of +infinity and of NaN are NaN."""
    g = gen(window)
    n = 300
    q, k, v = (torch.randn((n, h, 128), generator=g, device=dev).to(dtype) for h in (2, 1, 1))
    q[:, :, 0] = q[:, :, 0].abs() + 0.1
    k[0, 0, 0], k[90, 0, 0] = -INF, -INF
    k[200, 0, 0] = INF
    q[150, 1] = NAN
    v[60, 0, 5], v[100, 0] = NAN, INF
    out = torch.empty_like(q)
    backend.prefill_varlen(q, k, v, out, offsets([n]), window=window)
    assert backend.device_status() == 0
    compare(out, expect(q, k, v, window), dtype)


@pytest.mark.parametrize("window", [0, 100])
def test_values_near_the_end_of_bf16(backend, window):
    """Finite values whose weighted sums would pass the largest f32 before they are divided."""
    g = gen(3)
    n = 300
    q, k = (torch.randn((n, h, 128), generator=g, device=dev).bfloat16() * 3 for h in (2, 1))
    v = (torch.rand((n, 1, 128), generator=g, device=dev) * 0.9 + 0.05).mul(3.3e38).bfloat16()
    out = torch.empty_like(q)
    backend.prefill_varlen(q, k, v, out, offsets([n]), window=window)
    assert backend.device_status() == 0
    compare(out, expect(q, k, v, window), torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_to_mend_in_long_chains_of_items(backend, dtype):
    """Values that are not finite in prompts between clean ones, a CTA working through many of both."""
    g = gen(4)
    lens = [300, 5, 700, 129, 64, 400, 1, 200]
    q, k, v = (torch.randn((sum(lens), h, 128), generator=g, device=dev).to(dtype) for h in (6, 2, 2))
    cu = offsets(lens)
    clean = torch.empty_like(q)
    backend.prefill_varlen(q, k, v, clean, cu)
    at = cu.tolist()
    v[at[0] + 250, 0, 3], v[at[2] + 400, 1], v[at[5] + 10, 0, 100] = NAN, INF, NAN
    for ctas in (0, 1, 3):
        out = torch.full_like(q, 7.0)
        backend.set_option("swa_ctas", ctas)
        try:
            backend.prefill_varlen(q, k, v, out, cu)
        finally:
            backend.set_option("swa_ctas", 0)
        for b, n in enumerate(lens):
            sl = slice(at[b], at[b + 1])
            if b in (0, 2, 5):
                compare(out[sl], expect(q[sl], k[sl], v[sl]), dtype)
            else:
                assert torch.equal(out[sl], clean[sl])
    assert backend.device_status() == 0


@pytest.mark.parametrize("what", ["k", "v", "element"])
def test_an_early_nan_costs_its_own_rows_alone(backend, what):
    """A NaN near the front of a long prompt: the prompts packed beside it come out as without it, no wait runs out, and the
    call stays within a few times of the clean one's time."""
    g = gen(5)
    lens = [100, 2048, 500]
    q, k, v = (torch.randn((sum(lens), h, 128), generator=g, device=dev).bfloat16() for h in (16, 4, 4))
    cu = offsets(lens)

    def timed(out):
        for _ in range(2):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            backend.prefill_varlen(q, k, v, out, cu)
            b.record()
            b.synchronize()
        return a.elapsed_time(b)

    clean, out = torch.empty_like(q), torch.empty_like(q)
    t0 = timed(clean)
    if what == "k":
        k[103] = NAN
    elif what == "v":
        v[103] = NAN
    else:
        v[103, :, 77] = NAN
    t1 = timed(out)
    assert backend.device_status() == 0
    assert torch.equal(out[:100], clean[:100]) and torch.equal(out[2148:], clean[2148:])
    hit = torch.zeros(128, dtype=torch.bool, device=dev)
    hit[77 if what == "element" else slice(None)] = True
    assert torch.isnan(out[103:2148]).eq(hit).all()
    check(out[100:103], q[100:103], k[100:103], v[100:103], offsets([3]), offsets([3]), 0, torch.bfloat16)
    if what == "element":
        keep = ~hit
        want = clean[103:2148][..., keep].double()
        assert torch.equal(out[103:2148][..., keep].double(), want)
    assert t1 < 20 * t0 + 0.2, (t0, t1)  # ms; row by row on its own it would be hundreds of times


@pytest.mark.parametrize("window", [2 ** 31 - 1, 2 ** 31 - 200, 1000])
@pytest.mark.parametrize("new,keys", [([300, 500], [100, 40]), ([700], [700]), ([5, 2], [0, 900])])
def test_windows_longer_than_any_sequence(backend, window, new, keys):
    """They hide nothing, with more queries than keys and the reverse."""
    g = gen(sum(new))
    q, k, v = (torch.randn((m, h, 128), generator=g, device=dev).bfloat16() for m, h in ((sum(new), 4), (sum(keys), 2), (sum(keys), 2)))
    out, plain = torch.empty_like(q), torch.empty_like(q)
    backend.prefill_varlen(q, k, v, plain, offsets(new), offsets(keys))
    backend.prefill_varlen(q, k, v, out, offsets(new), offsets(keys), window=window)
    assert backend.device_status() == 0
    assert torch.equal(out, plain)
    check(out, q, k, v, offsets(new), offsets(keys), 0, torch.bfloat16)
