"""Packed causal attention (prefill_varlen) on the GPU against its definition in 64 bits."""
import numpy as np
import pytest
import torch

from hachiue_b200 import HachiueError
from tests import paged_reference as ref

pytestmark = pytest.mark.gpu
dev = "cuda"
DTYPES = [torch.bfloat16, torch.float16]


def gen(seed):
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    return g


def offsets(lens, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(lens)]), dtype=torch.int32, device=dev)


def check(out, q, k, v, cu_q, cu_k, window, dtype):
    cq, ck = cu_q.tolist(), cu_k.tolist()
    for b in range(len(cq) - 1):
        nq, nk = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        if nq == 0:
            continue
        want, spread, mag = ref.attend(q[cq[b]:cq[b + 1]].double(), k[ck[b]:ck[b + 1]].double(), v[ck[b]:ck[b + 1]].double(),
                                       nk - nq, window)
        # the probabilities are rounded to dtype for their product with the values
        bound = ref.attention_bound(want, spread, mag, 128, nk, dtype, ref.HALF_STEP[dtype])
        got = out[cq[b]:cq[b + 1]].double()
        err = (got - want).abs()
        assert (err <= bound).all(), (b, nq, nk, float((err / bound).max()), float(err.max()))
        # a bound on each element is far above what many roundings add up to: their mean square stays near one rounding's
        if nq * nk > 100:
            assert float((got - want).norm() / want.norm()) < 2 * ref.HALF_STEP[dtype]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("H,KV,window,new,prefix", [
    (2, 1, 0, [1], [0]),
    (2, 2, 0, [128], [0]),
    (16, 8, 0, [77], [0]),
    (4, 2, 0, [1, 127, 129, 0, 256, 3, 64], None),
    (6, 3, 0, [300, 1, 515], None),
    (5, 1, 33, [200, 32, 33, 34, 700], None),
    (8, 2, 1024, [1500, 10], None),
    (2, 1, 1, [140, 2], None),
    (4, 1, 0, [5, 200, 1, 130, 0], [300, 128, 1000, 0, 77]),
    (3, 3, 129, [5, 200, 1, 130], [300, 128, 1000, 0]),
    (4, 4, 0, [40, 300, 7, 129], [-10, -300, 5, -128]),
    (8, 1, 0, list(range(1, 40)), None)])
@pytest.mark.parametrize("fused", [False, True])
def test_packed(backend, dtype, H, KV, window, new, prefix, fused):
    """Lengths from nothing to several tiles, prefixes, windows, odd groups; negative prefixes leave the first queries
    without a key; out rows behind the last sequence and before the first stay as they were."""
    g = gen(sum(new) + H + window)
    first, tail = 3, 5
    keys = new if prefix is None else [a + b for a, b in zip(new, prefix)]
    nq, nk = sum(new) + first + tail, sum(keys) + first + tail
    if fused and prefix is None:
        x = torch.randn((nq, H + 2 * KV, 128), generator=g, device=dev).to(dtype)
        q, k, v = x[:, :H], x[:, H:H + KV], x[:, H + KV:]
    else:
        q, k, v = (torch.randn((n, h, 128), generator=g, device=dev).to(dtype) for n, h in ((nq, H), (nk, KV), (nk, KV)))
    k[:first], v[:first], k[nk - tail:], v[nk - tail:] = (float("nan"),) * 4
    cu_q, cu_k = offsets(new, first), offsets(keys, first)
    out = torch.full((nq, H, 128), 7.0, device=dev, dtype=dtype)
    backend.prefill_varlen(q, k, v, out, cu_q, None if prefix is None else cu_k, window)
    assert backend.device_status() == 0
    assert (out[:first] == 7.0).all() and (out[nq - tail:] == 7.0).all()
    check(out, q, k, v, cu_q, cu_k, window, dtype)
    for b, (a, n) in enumerate(zip(new, keys)):
        empty = max(0, a - n)
        assert (out[int(cu_q[b]):int(cu_q[b]) + empty] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_neighbours_do_not_leak(backend, dtype):
    """Sequences between others whose keys and values are NaN and infinite."""
    g = gen(5)
    lens = [100, 131, 5, 260, 1]
    q, k, v = (torch.randn((sum(lens), h, 128), generator=g, device=dev).to(dtype) for h in (4, 2, 2))
    cu = offsets(lens)
    for b, bad in ((0, float("nan")), (2, float("inf")), (4, float("nan"))):
        sl = slice(int(cu[b]), int(cu[b + 1]))
        k[sl], v[sl] = bad, bad
    out = torch.empty_like(q)
    backend.prefill_varlen(q, k, v, out, cu)
    for b in (1, 3):
        sl = slice(int(cu[b]), int(cu[b + 1]))
        one = torch.empty_like(q[sl])
        backend.prefill_varlen(q[sl], k[sl], v[sl], one, offsets([lens[b]]))
        assert torch.isfinite(out[sl].float()).all() and torch.equal(out[sl], one)


def test_later_tokens_do_not_reach_back(backend):
    """NaN and infinite keys and values of later tokens leave every earlier query as it was."""
    g = gen(6)
    n, bad = 300, 170
    q, k, v = (torch.randn((n, h, 128), generator=g, device=dev).bfloat16() for h in (4, 2, 2))
    cu = offsets([n])
    clean, out = torch.empty_like(q), torch.empty_like(q)
    backend.prefill_varlen(q, k, v, clean, cu)
    k[bad:bad + 40], v[bad:bad + 20], v[bad + 20:bad + 40] = float("nan"), float("nan"), float("inf")
    backend.prefill_varlen(q, k, v, out, cu)
    assert torch.isfinite(out[:bad].float()).all()
    want, spread, mag = ref.attend(q[:bad].double(), k[:bad].double(), v[:bad].double(), 0)
    bound = ref.attention_bound(want, spread, mag, 128, bad, torch.bfloat16, 2.0 ** -8)
    assert ((out[:bad].double() - want).abs() <= bound).all()
    assert torch.isnan(out[bad:].float()).any(-1).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_scores(backend, dtype):
    """Scores up to some hundreds, so that a row's maximum moves from tile to tile and one key takes all."""
    g = gen(7)
    lens = [700, 390]
    q, k, v = (torch.randn((sum(lens), h, 128), generator=g, device=dev).to(dtype) for h in (4, 1, 1))
    k *= torch.linspace(0.2, 8, sum(lens), device=dev)[:, None, None].to(dtype)
    cu = offsets(lens)
    out = torch.empty_like(q)
    backend.prefill_varlen(q, k, v, out, cu)
    check(out, q, k, v, cu, cu, 0, dtype)


def test_bad_offsets_are_skipped(backend):
    """Offsets that decrease or leave the tensors: that sequence is skipped and reported, the others are right."""
    g = gen(8)
    q, k, v = (torch.randn((100, h, 128), generator=g, device=dev).bfloat16() for h in (2, 1, 1))
    cu_q = torch.tensor([0, 40, 30, 101, 100], dtype=torch.int32, device=dev)
    cu_k = torch.tensor([0, 40, 40, 60, 100], dtype=torch.int32, device=dev)
    out = torch.full_like(q, 7.0)
    backend.prefill_varlen(q, k, v, out, cu_q, cu_k)
    assert backend.device_status() == 2
    assert (out[40:] == 7.0).all()
    check(out, q, k, v, cu_q[:2], cu_k[:2], 0, torch.bfloat16)
    out.fill_(7.0)
    backend.prefill_varlen(q, k, v, out, torch.tensor([-5, 20, 100], dtype=torch.int32, device=dev),
                           torch.tensor([0, 20, 100], dtype=torch.int32, device=dev))
    assert backend.device_status() == 2
    assert (out[:20] == 7.0).all()
    check(out[20:], q[20:], k[20:], v[20:], offsets([80]), offsets([80]), 0, torch.bfloat16)


def test_many_sequences_long_and_short(backend):
    g = gen(9)
    lens = [int(n) for n in np.random.default_rng(0).integers(0, 40, 600)] + [2500, 1000]
    q, k, v = (torch.randn((sum(lens), h, 128), generator=g, device=dev).bfloat16() for h in (4, 2, 2))
    cu = offsets(lens)
    out = torch.full_like(q, float("nan"))
    backend.prefill_varlen(q, k, v, out, cu, window=300)
    check(out, q, k, v, cu, cu, 300, torch.bfloat16)
    assert backend.device_status() == 0


def test_graph_and_streams(backend):
    """Captured and replayed with other lengths; the same call on another stream gives the same bits."""
    g = gen(10)
    q, k, v = (torch.randn((500, h, 128), generator=g, device=dev).bfloat16() for h in (4, 2, 2))
    cu = offsets([500, 0, 0])
    out = torch.empty_like(q)
    backend.prefill_varlen(q, k, v, out, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        backend.prefill_varlen(q, k, v, out, cu)
    for lens in ([500, 0, 0], [1, 250, 249], [130, 140, 230]):
        cu.copy_(offsets(lens))
        graph.replay()
        torch.cuda.synchronize()
        check(out, q, k, v, cu, cu, 0, torch.bfloat16)
        again = torch.empty_like(out)
        with torch.cuda.stream(side):
            backend.prefill_varlen(q, k, v, again, cu)
        side.synchronize()
        assert torch.equal(again, out)


def test_c_refusals(backend):
    import ctypes

    from hachiue_b200 import _lib
    q = torch.zeros((8, 4, 128), device=dev, dtype=torch.bfloat16)
    cu = offsets([8])

    def call(status, qp=q.data_ptr(), out=q.data_ptr(), **over):
        p = _lib.hcu_prefill_varlen_params(1, 4, 4, 128, 0, _lib.DT_BF16, 8, 8, cu.data_ptr(), None, 0, 0, 0)
        for name, value in over.items():
            setattr(p, name, value)
        got = backend.lib.hcu_prefill_varlen(backend._h, ctypes.byref(p), qp, q.data_ptr(), q.data_ptr(), out)
        assert got == status, over

    call(0, batch=0)
    call(0, total_q=0, total_k=0)
    for over in (dict(dtype=_lib.DT_F32), dict(H=6), dict(KV=0), dict(total_k=9), dict(q_row_stride=516),
                 dict(k_row_stride=256), dict(window=2 ** 31), dict(cu_q=None), dict(qp=None), dict(qp=q.data_ptr() + 2),
                 dict(batch=70000)):
        call(1, **over)
    call(6, D=64)
    with pytest.raises(HachiueError):
        backend.prefill_varlen(q.float(), q, q, q, cu)
    assert backend.device_status() == 0
