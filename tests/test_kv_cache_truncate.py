"""KvCache.truncate: the host side of an eviction (no GPU needed)."""
import pytest
import torch

from aoakv.utils import KvCache


@pytest.mark.parametrize("page", [1, 7, 16])
def test_truncate_gives_pages_back(page):
    c = KvCache(1, 1, 64, 200, page, torch.float16, "cpu")
    c.append_seq(100)
    ids = list(c.indicies)
    for n in (100, 99, 97, 50, 49, 33, 32, 1, 0):
        had = len(c.indicies)
        assert c.truncate(n) == had - len(c.indicies)
        assert c.seqlen == n and c.indicies == ids[:-(-n // page)]
        assert c.pool.num_free_blocks == c.pool.capacity - len(c.indicies)
    c.append_seq(100)
    assert len(c.indicies) == -(-100 // page) and len(set(c.indicies)) == len(c.indicies)
    for bad in (101, -1):
        with pytest.raises(ValueError, match="cannot be kept"):
            c.truncate(bad)
