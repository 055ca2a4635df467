"""CPU tests of the paged cache's own bookkeeping, on tables in host memory, and of a
frequency scaling at its end."""
from types import SimpleNamespace

import pytest
import torch

from edgeexpert_b200._lib import TFError
from edgeexpert_b200.paged import PagedKVCache


def cache_of(lens, page=4, max_pages=5):
    cache = PagedKVCache(1, 1, 8, len(lens), 32, max_pages, 8, page_size=page, device="cpu",
                         context=SimpleNamespace(handle=None, device=0))
    at = 0
    for b, n in enumerate(lens):
        held = -(-n // page)
        cache.page_table[b, :held] = torch.arange(at, at + held)
        at += held
    cache.seq_lens[:] = torch.tensor(lens)
    cache.free_state[:] = torch.tensor([at, 32 - at, 0, 0])
    return cache


@pytest.mark.parametrize("lens,request_,length", [
    ([9, 0, 0], 0, 8),    # the request holds a page more: nobody would have it any longer
    ([9, 0, 0], 0, 12),   # positions that were never written
    ([9, 0, 0], 0, 13),   # a page that it does not hold
    ([9, 0, 2], 0, 9),    # the others' positions would move behind the prefix
    ([9, 0, 0], 1, 9), ([9, 0, 0], 3, 9), ([9, 0, 0], -1, 9), ([9, 0, 0], 0, 0), ([9, 0, 0], 0, 21)])
def test_a_prefix_that_the_tables_do_not_hold_is_refused(lens, request_, length):
    cache = cache_of(lens)
    with pytest.raises(TFError):
        cache.share(request_, length)
    assert cache.prefix_len == 0 and cache.prefix_pages is None and cache.seq_lens.tolist() == lens


@pytest.mark.parametrize("length", [1, 4, 9, 20])
def test_a_request_becomes_the_prefix_once(length):
    cache = cache_of([0, length, 0])
    pages = cache.page_table[1, :-(-length // 4)].tolist()
    cache.share(1, length)
    assert cache.prefix_len == length and cache.prefix_pages.tolist() == pages and cache.seq_lens.tolist() == [0, 0, 0]
    cache.page_table[1, 0] = 31  # the prefix keeps its own list
    assert cache.prefix_pages.tolist() == pages
    with pytest.raises(TFError):
        cache.share(1, length)


@pytest.mark.parametrize("factor", [1e-6, 0.25, 0.5, 1.0])
def test_a_context_that_is_not_extended_keeps_its_attention(factor):
    """The ramp's attention factor makes up for a longer context; factors up to 1 leave it at 1
    (0.1 ln(factor) + 1 would fall, below e^-10 to negative values)."""
    from edgeexpert_b200.paged import rope_frequencies
    _, mul = rope_frequencies(64, scaling="ramp", factor=factor, original_context=8192, device="cpu")
    assert mul == 1.0
