"""CPU checks of PagedKVCache's bookkeeping."""
import pytest
import torch

import fully_custom_cuda_inference_lamma2_b200 as pkg


def bare_cache(batch=2, num_pages=6, page_size=16, max_pages=4):
    """The bookkeeping alone, on the CPU (a whole cache makes its workspace on a GPU)."""
    c = pkg.PagedKVCache.__new__(pkg.PagedKVCache)
    c.page_size, c.num_pages, c.max_pages, c.device = page_size, num_pages, max_pages, torch.device("cpu")
    c.page_table = torch.full((batch, max_pages), -1, dtype=torch.int32)
    c.seq_lens = torch.zeros(batch, dtype=torch.int32)
    c._free = list(range(num_pages - 1, -1, -1))
    c._pages = [[] for _ in range(batch)]
    return c


class FailingTable:
    def __setitem__(self, at, value):
        raise RuntimeError("out of memory")


def test_reserve_that_fails_changes_nothing():
    c = bare_cache()
    c.reserve(0, 20)
    held, free, table = c.pages_of(0), list(c._free), c.page_table
    assert table[0].tolist() == held + [-1, -1]
    c.page_table = FailingTable()
    with pytest.raises(RuntimeError, match="out of memory"):
        c.reserve(0, 40)
    assert c.pages_of(0) == held and c._free == free
    c.page_table = table
    c.reserve(0, 40)
    c.reserve(1, 48)
    assert c.free_pages() == 0 and sorted(c.pages_of(0) + c.pages_of(1)) == list(range(6))
    assert table[0].tolist() == c.pages_of(0) + [-1] and table[1].tolist() == c.pages_of(1) + [-1]
    c.seq_lens[1] = 48
    c.release(1)
    assert c.free_pages() == 3 and (table[1] == -1).all() and c.seq_lens.tolist() == [0, 0]
