"""The packed prefill at the ends of its arguments' ranges."""
import pytest
import torch

from tests.test_prefill_varlen_gpu import check, dev, gen, offsets

pytestmark = pytest.mark.gpu


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
