"""The paged cache's allocator on the CPU."""
from __future__ import annotations

import pytest

from llama1b_megakernel_b200.config import TINY
from llama1b_megakernel_b200.kv_cache import PagedKVCache, QuantizedPagedKVCache


@pytest.mark.parametrize("kind", [PagedKVCache, QuantizedPagedKVCache])
def test_refused_reservation_takes_no_pages(kind):
    """A reservation that the pool cannot meet leaves the sequence and the pool as they were, and
    a smaller one after it reaches the device's table."""
    kv = kind(TINY, max_batch=2, max_seq_len=64, page_size=8, num_pages=5, device="cpu")
    kv.reserve(1, 9)
    with pytest.raises(RuntimeError):
        kv.reserve(0, 33)
    assert kv.pages_of(0) == [] and len(kv._free) == 3 and (kv.block_tables[0] == -1).all()
    kv.reserve(0, 24)
    assert kv.block_tables[0, :3].tolist() == kv.pages_of(0) and (kv.block_tables[0, 3:] == -1).all()
    assert not set(kv.pages_of(0)) & set(kv.pages_of(1))
