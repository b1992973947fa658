"""Numbers that the 32-bit fields of the C structures cannot hold: refused, or held within what the library takes, before they
wrap."""
import pytest
import torch

from tests.test_paged_cpu import be, cache, refused  # noqa: F401  (be: a backend over a recording library)


@pytest.mark.parametrize("bad", [-1, 2 ** 31, 2 ** 32, 2 ** 32 + 5, -2 ** 32 + 7])
def test_out_of_range(be, bad):  # noqa: F811
    c = cache()
    q, table, ctx = torch.zeros((3, 2, 4, 128)), torch.zeros((3, 9), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    refused(be.attention_paged, q, c, torch.zeros_like(q), table, ctx, window_size=bad)
    refused(be.attention_paged, q, c, torch.zeros_like(q), table, ctx, max_context=bad)
    x, cu = torch.zeros((6, 2, 128)).half(), torch.tensor([0, 6], dtype=torch.int32)
    refused(be.prefill_varlen, x, x, x, torch.zeros_like(x), cu, window=bad)
    assert not be.lib.calls


def test_the_largest_that_are_taken(be):  # noqa: F811
    c = cache()
    q, table, ctx = torch.zeros((1, 2, 4, 128)), torch.zeros((1, 9), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    be.attention_paged(q, c, torch.zeros_like(q), table, ctx, max_context=2 ** 31 - 1, window_size=2 ** 31 - 1)
    p = be.lib.calls.pop()[1][1]
    assert (p.max_context, p.windowSize) == (2 ** 31 - 1, 2 ** 31 - 1)  # the library says what it takes of these


@pytest.mark.parametrize("pages", [2 ** 23 - 1, 2 ** 23, 2 ** 24, 2 ** 24 + 3])
def test_a_table_of_more_tokens_than_a_context_has(be, pages):  # noqa: F811
    """256 tokens a page: without a max_context the bound is the library's, not the table's 2^31 or 2^32 tokens wrapped."""
    c = cache(page=256)
    q, ctx = torch.zeros((1, 1, 4, 128)), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros((1, pages), dtype=torch.int32)
    be.attention_paged(q, c, torch.zeros_like(q), table, ctx)
    p = be.lib.calls.pop()[1][1]
    assert p.max_context == 0x7fffff00 and p.table_stride == pages
