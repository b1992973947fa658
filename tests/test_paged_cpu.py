"""The paged operators' host side and number tricks, on the CPU: what the Python methods refuse and what they hand to the
library, the layout of the pages, and the arithmetic that the kernels use in place of divisions and conversions."""
import types
from fractions import Fraction

import numpy as np
import pytest
import torch

from hachiue_b200 import CudaBackend, HachiueError, PagedKVCache, _lib
from hachiue_b200 import backend as module
from tests import paged_reference as ref


# ---- refusals of the Python methods, and the parameters behind them ------------
class FakeLib:
    """Records the last call, its structures copied."""

    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        if not name.startswith("hcu_"):
            raise AttributeError(name)

        def call(*args):
            self.calls.append((name, [type(a._obj).from_buffer_copy(a._obj) if hasattr(a, "_obj") else a for a in args]))
            return 0
        return call


@pytest.fixture
def be(monkeypatch):
    monkeypatch.setattr(module, "_ptr", lambda t: None if t is None else t.data_ptr())
    b = CudaBackend.__new__(CudaBackend)
    b.lib, b._h, b.device = FakeLib(), 1, types.SimpleNamespace(index=-1)
    b._paged_params, b._varlen_params = _lib.hcu_attention_paged_params(), _lib.hcu_prefill_varlen_params()
    b._append_params = _lib.hcu_rope_append_params()
    b._bind_stream = lambda: None
    yield b
    b._h = None


def cache(n_pages=4, page=16, KV=2, Dh=128):
    return PagedKVCache.allocate(n_pages, page, KV, Dh, device="cpu")


def refused(f, *args, **kw):
    with pytest.raises(HachiueError):
        f(*args, **kw)


def test_append_parameters_and_refusals(be):
    c = cache()
    x = torch.zeros((5, 8, 128))
    q, k, v = x[:, :4], x[:, 4:6], x[:, 6:]
    slots, pos = torch.zeros(5, dtype=torch.int64), torch.zeros(5, dtype=torch.int32)
    cos = torch.zeros((7, 32))
    q_out, k_out = torch.zeros((5, 4, 128)), torch.zeros((5, 2, 128))
    good = dict(cos=cos, sin=cos, positions=pos, q=q, q_out=q_out, k_out=k_out)
    be.rope_append_paged(k, v, c, slots, **good)
    name, args = be.lib.calls.pop()
    p = args[1]
    assert name == "hcu_rope_append_paged"
    assert (p.n, p.H, p.dtype, p.rotaryDim, p.table_rows) == (5, 4, _lib.DT_F32, 64, 7)
    assert (p.q_row_stride, p.k_row_stride, p.v_row_stride) == (1024, 1024, 1024)
    assert args[2:5] == [q.data_ptr(), k.data_ptr(), v.data_ptr()]
    st = args[-1]
    assert (st.format, st.page_size, st.n_pages, st.KV, st.Dh) == (_lib.KV_Q4_0, 16, 4, 2, 128)
    be.rope_append_paged(k[:1], v[:1], c, slots[:1])  # one row: its stride says nothing
    p = be.lib.calls.pop()[1][1]
    assert (p.H, p.rotaryDim, p.table_rows, p.q_row_stride, p.k_row_stride) == (0, 0, 0, 0, 0)
    be.rope_append_paged(k[:0], v[:0], c, slots[:0])
    assert not be.lib.calls
    bad = lambda **kw: refused(be.rope_append_paged, **{**dict(k=k, v=v, cache=c, slots=slots, **good), **kw})
    bad(k=k[0])
    bad(k=k[..., :64])
    bad(k=x[:, :4])
    bad(v=v.half())
    bad(v=v[:4])
    bad(k=k.double(), v=v.double())
    bad(slots=slots.int())
    bad(slots=slots[:4])
    bad(slots=torch.zeros((5, 2), dtype=torch.int64)[:, 0])
    bad(sin=None)
    bad(cos=None)
    bad(positions=None)
    bad(positions=pos.long())
    bad(cos=cos.double(), sin=cos.double())
    bad(sin=cos[:6])
    bad(q_out=None)
    bad(q=None)
    bad(q=q[:, 0])
    bad(q=q.half())
    bad(q_out=q)  # a view of wider rows
    bad(k_out=k)
    bad(k_out=k_out.bfloat16())
    bad(k=k[:1].expand(5, 2, 128))  # one row for five tokens
    bad(k=torch.zeros((5, 2, 256))[..., ::2])
    bad(k=torch.zeros((5, 2, 256))[..., :128])
    bad(k=torch.zeros((2, 5, 128)).transpose(0, 1))
    assert not be.lib.calls


def test_read_parameters_and_refusals(be):
    c = cache(Dh=256)
    slots, k, v = torch.zeros(3, dtype=torch.int64), torch.zeros((3, 2, 256)).half(), torch.zeros((3, 2, 256)).half()
    be.read_paged(c, slots, k, v)
    name, args = be.lib.calls.pop()
    assert name == "hcu_read_paged" and args[1:3] == [3, _lib.DT_F16] and args[4].Dh == 256
    be.read_paged(c, slots[:0], k[:0], v[:0])
    for bad in ((slots.int(), k, v), (slots[:2], k, v), (slots[0], k[0], v[0]), (slots, k.float(), v), (slots, k, v[:, :1]),
                (slots, k.double(), v.double()), (slots, torch.zeros((3, 2, 512)).half()[..., :256], v)):
        refused(be.read_paged, c, *bad)
    assert not be.lib.calls


def test_decode_parameters_and_refusals(be):
    c = cache()
    q, table, ctx = torch.zeros((3, 2, 4, 128)).bfloat16(), torch.zeros((3, 9), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    out = torch.zeros_like(q)
    be.attention_paged(q, c, out, table, ctx, window_size=7)
    name, args = be.lib.calls.pop()
    p = args[1]
    assert name == "hcu_attention_paged"
    assert (p.batch, p.S, p.H, p.windowSize, p.dtype, p.max_context, p.table_stride) == (3, 2, 4, 7, _lib.DT_BF16, 144, 9)
    assert (p.block_table, p.context) == (table.data_ptr(), ctx.data_ptr())
    be.attention_paged(q, c, out, table, ctx, max_context=20)
    assert be.lib.calls.pop()[1][1].max_context == 20
    be.attention_paged(q[:0], c, out[:0], table[:0], ctx[:0])
    be.attention_paged(q[:, :0], c, out[:, :0], table, ctx)
    for bad in ((q[0], out[0], table, ctx), (q[..., :64], out[..., :64], table, ctx), (q, out.half(), table, ctx),
                (q.double(), out.double(), table, ctx), (q, out[:, :1], table, ctx), (q.transpose(1, 2), out.transpose(1, 2), table, ctx),
                (q, out, table.long(), ctx), (q, out, table[:2], ctx), (q, out, table[:, :4], ctx), (q, out, table[0], ctx),
                (q, out, table, ctx.long()), (q, out, table, ctx[:2])):
        refused(be.attention_paged, bad[0], c, *bad[1:])
    assert not be.lib.calls


def test_prefill_parameters_and_refusals(be):
    x = torch.zeros((6, 8, 128)).half()
    q, k, v, out = x[:, :4], x[:, 4:6], x[:, 6:], torch.zeros((6, 4, 128)).half()
    cu = torch.tensor([0, 2, 6], dtype=torch.int32)
    be.prefill_varlen(q, k, v, out, cu, window=5)
    name, args = be.lib.calls.pop()
    p = args[1]
    assert name == "hcu_prefill_varlen"
    assert (p.batch, p.H, p.KV, p.D, p.window, p.dtype, p.total_q, p.total_k) == (2, 4, 2, 128, 5, _lib.DT_F16, 6, 6)
    assert (p.q_row_stride, p.cu_q, p.cu_k) == (1024, cu.data_ptr(), None)
    be.prefill_varlen(q, k, v, out, cu, cu.clone())
    assert be.lib.calls.pop()[1][1].cu_k
    be.prefill_varlen(q[:0], k[:0], v[:0], out[:0], cu)
    be.prefill_varlen(q, k, v, out, cu[:1])
    for bad in ((q.float(), k.float(), v.float(), out.float(), cu), (q, k.bfloat16(), v, out, cu), (q, k, v[:5], out, cu),
                (q, k, v, x[:, :4], cu), (q, k, v, out[:, :2], cu), (q[0], k, v, out, cu), (q, k[0], v, out, cu),
                (q, k, v, out, cu.long()), (q, k, v, out, cu[:0]), (q, k, v, out, cu[None]), (q, k, v, out, cu, cu[:2]),
                (q, k, v, out, cu, cu.long()), (q, k[:1].expand(6, 2, 128), v, out, cu)):
        refused(be.prefill_varlen, *bad)
    assert not be.lib.calls


def test_other_devices_are_refused(be):
    be.device = types.SimpleNamespace(index=0)
    c, x = cache(), torch.zeros((1, 2, 128))
    one, off = torch.zeros(1, dtype=torch.int64), torch.zeros(2, dtype=torch.int32)
    refused(be.rope_append_paged, x, x, c, one)
    refused(be.read_paged, c, one, x, x)
    refused(be.attention_paged, x[None], c, x[None], off[None], off[:1])
    refused(be.prefill_varlen, x.half(), x.half(), x.half(), x.half(), off)


def test_cache_geometry(be):
    c = cache(3, 32, 5, 256)
    assert (c.n_pages, c.page_size, c.kv_heads, c.head_dim) == (3, 32, 5, 256)
    st = c.c_struct()
    assert st.k == c.k.data_ptr() and c.c_struct() is st
    c.v = c.v.clone()
    assert c.c_struct().v == c.v.data_ptr()
    c.k.resize_(2, 5, 32, 128)
    refused(c.c_struct)
    for name, t in (("k", torch.zeros((3, 5, 32, 128))), ("v", torch.zeros((3, 5, 32, 64), dtype=torch.uint8)),
                    ("k_scale", torch.zeros((3, 5, 32, 8))), ("v_scale", torch.zeros((3, 5, 32, 16), dtype=torch.float16)[..., :8])):
        c = cache(3, 32, 5, 256)
        setattr(c, name, t)
        refused(c.c_struct)


# ---- layouts and the quantiser, from scalar definitions --------------------------
@pytest.mark.parametrize("Dh", [128, 256])
def test_layout(Dh):
    nb = Dh // 32
    code = torch.randint(0, 16, (3, Dh), dtype=torch.uint8)
    k = ref.pack(code, ref.key_nibble(Dh)).numpy().view("<u4")
    v = ref.pack(code, ref.value_nibble(Dh)).numpy().view("<u2")
    for r in range(3):
        for b in range(nb):
            for t in range(4):
                assert k[r, t * nb + b] == sum(int(code[r, 32 * b + 8 * t + c]) << (4 * c) for c in range(8))
            for g in range(8):
                assert v[r, g * nb + b] == sum(int(code[r, 32 * b + 4 * g + c]) << (4 * c) for c in range(4))
    scale = torch.ones((3, nb), dtype=torch.float16)
    assert torch.equal(ref.unpack(ref.pack(code, ref.key_nibble(Dh)), scale, ref.key_nibble(Dh)), code.double() - 8)
    assert torch.equal(ref.unpack(ref.pack(code, ref.value_nibble(Dh)), scale, ref.value_nibble(Dh)), code.double() - 8)


def test_quantiser_by_fractions():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((40, 32)) * 10.0 ** rng.integers(-6, 5, (40, 1))).astype(np.float32)
    x[7] = 0
    code, d = ref.quantise(torch.from_numpy(x))
    for r in range(40):
        m = max(range(32), key=lambda j: (abs(x[r, j]), -j))
        want = np.float16(np.clip(x[r, m] / np.float32(-8), -65504, 65504))
        assert d[r, 0].numpy() == want
        for j in range(32):
            level = 8
            if want != 0:
                level = min(15, max(0, (Fraction(float(x[r, j])) / Fraction(float(want)) + Fraction(17, 2)).__floor__()))
            assert code[r, j] == level


# ---- arithmetic that stands in for divisions and conversions ----------------------
def f32(x):
    return np.asarray(x, dtype=np.float64).astype(np.float32)


def test_levels_without_a_division():
    """paged_cache.cu, q4_code: a rounded product that two compares put right, at and next to every border of every f16
    scale.  (An fma is the f64 result rounded: its product has 48 bits, and a last bit more or less before the compares is
    what they are there for.)"""
    a = np.arange(1, 0x7c00, dtype=np.uint16).view(np.float16).astype(np.float32)  # every positive finite one
    inv = f32(1.0) / a
    for j in range(-2, 18):
        for step in (-1, 0, 1):
            y = f32((j - 8.5) * a.astype(np.float64))
            assert np.array_equal(y.astype(np.float64), (j - 8.5) * a.astype(np.float64))  # a border is exact in f32
            if step:
                y = np.nextafter(y, np.float32(step * np.inf))
            y64, a64 = y.astype(np.float64), a.astype(np.float64)
            c = np.clip(f32(y64 * inv + 12582920.0) - np.float32(12582912.0), 0, 15).astype(np.float32)
            lower = f32(c * a64 - 8.5 * a64)
            c = np.where(lower > y, c - 1, c)
            c = np.where(lower + a <= y, c + 1, c)
            got = (np.clip(c, 0, 15).astype(np.float32) + np.float32(8388608.0)).view(np.uint32) & 15
            want = sum((y64 >= (n - 8.5) * a64).astype(np.int64) for n in range(1, 16))
            assert np.array_equal(got, want), (j, step)


@pytest.mark.parametrize("ulp", [-1, 0, 1])
def test_levels_by_a_biased_rounding(ulp):
    """paged_cache.cu, q4_codes: x * inv + 8 + 2^-18 rounded, with a reciprocal that is off by an ulp either way.  Right for
    every 16-bit input next to a border; an f32 input that it takes for the level above is one that it looks for."""
    a = np.arange(1, 0x7c00, dtype=np.uint16).view(np.float16).astype(np.float32)
    inv = f32(1.0) / a
    inv = inv if ulp == 0 else np.nextafter(inv, np.float32(ulp * np.inf))
    bias = np.float32(8 + 2.0 ** -18)
    assert float(bias) == 8 + 2.0 ** -18
    a64 = a.astype(np.float64)

    def levels(y):
        v = np.clip(f32(y.astype(np.float64) * inv + float(bias)), 0, 15).astype(np.float32)
        c = (v + np.float32(12582912.0)) - np.float32(12582912.0)
        return c, v - c

    def exact(y):
        return sum((y.astype(np.float64) >= (n - 8.5) * a64).astype(np.int64) for n in range(1, 16))

    for j in range(1, 16):
        border = (j - 8.5) * a64
        for bits in (8, 11):  # bf16 and f16 inputs: the multiples of an 8- or 11-bit number's last place around the border
            last = 2.0 ** (np.floor(np.log2(np.abs(border))) - bits + 1)
            for k in (-2, -1, 0, 1, 2, 3):
                y = f32((np.floor(border / last) + k) * last)
                c, _ = levels(y)
                assert np.array_equal(c.astype(np.int64), exact(y)), (j, bits, k)
        for k in range(-40, 41, 5):  # f32 inputs within some steps of the border
            y = (f32(border).view(np.int32) + k).view(np.float32)
            c, rest = levels(y)
            wrong = c.astype(np.int64) != exact(y)
            assert (rest[wrong] < -0.49999).all()


def test_codes_as_f16_bits():
    """attention_paged.cu: a code's bits in place are a subnormal f16, and with the exponent of 1024 an integer whose offset
    one subtraction takes off."""
    c = np.arange(16, dtype=np.uint16)
    f = lambda bits: np.asarray(bits, dtype=np.uint16).view(np.float16)
    assert np.array_equal(f(c).astype(np.float64), c * 2.0 ** -24)
    assert np.array_equal(f(c << 4).astype(np.float64), c * 2.0 ** -20)
    assert np.array_equal((f(c | 0x6400) - f(0x6408)).astype(np.float64), c - 8.0)
    assert np.array_equal((f((c << 4) | 0x6400) - f(0x6480)).astype(np.float64), 16 * (c - 8.0))


def test_quotients_by_a_reciprocal():
    """prefill_varlen.cu, quot: the high half of a product, put right by two compares, in 32 bits."""
    rng = np.random.default_rng(1)
    for d in [1, 2, 3, 4, 5, 6, 7, 8, 12, 15, 16, 100, 127, 128, 129, 1000, 32768, 65535]:
        recip = min(2 ** 32 - 1, 2 ** 32 // d + 1)
        n = rng.integers(0, 2 ** 30, 4000)
        n = np.unique(np.concatenate([n, n // d * d, np.maximum(n // d * d - 1, 0), [0, 1, d - 1, d, d + 1, 2 ** 30 - 1]]))
        q = (n * recip) >> 32
        assert (np.abs(q - n // d) <= 1).all() and (q * d < 2 ** 31).all()
        q = np.where(q * d > n, q - 1, q)
        q = np.where(n - q * d >= d, q + 1, q)
        assert np.array_equal(q, n // d), d


@pytest.mark.parametrize("total,ctas", [(1, 1), (7, 7), (296, 296), (1000, 296), (12345, 148), (2 ** 31 - 2, 296)])
def test_pieces_of_the_line(total, ctas):
    """attention_paged.cu, PagedPlan: the pieces of the line lie end to end, and cta_of finds the one that holds a position."""
    share, more = total // ctas, total % ctas
    start = [i * share + min(i, more) for i in range(ctas + 1)]
    assert start[0] == 0 and start[-1] == total and all(b - a in (share, share + 1) for a, b in zip(start, start[1:]))
    edge = more * (share + 1)
    rng = np.random.default_rng(2)
    for x in sorted({0, total - 1, max(0, edge - 1), min(total - 1, edge), *(int(n) for n in rng.integers(0, total, 200))}):
        i = x // (share + 1) if x < edge else more + (x - edge) // share
        assert start[i] <= x < start[i + 1]
