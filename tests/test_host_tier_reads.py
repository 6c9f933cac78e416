"""CPU: blocks that one prefetch returns together stay what they are while it
loads the rest."""
import threading
from collections import OrderedDict

import torch

from tidegs_b200.host_tier import PinnedBlockCache

B, D = 4, 59


class _Store:
    """Blocks in memory; writes wait for `gate`."""

    def __init__(self, n):
        self.blocks = {b: torch.full((B, D), float(b)) for b in range(n)}
        self.gate = threading.Event()

    def read_blocks_into(self, block_ids, dest):
        for b in block_ids:
            dest[b].copy_(self.blocks[b])
        return OrderedDict((b, B) for b in block_ids)

    def write_patch(self, blocks):
        assert self.gate.wait(30)
        for b, t in blocks.items():
            self.blocks[b] = t.clone()


def _cache(store, capacity):
    return PinnedBlockCache(store, max_ram_gb=1.0, block_size=B, point_dim=D, verbose=False,
                            capacity_blocks=capacity, pin_memory=False)


def test_a_block_found_in_the_flushing_buffer_is_not_overwritten_by_the_next_load():
    store = _Store(4)
    cache = _cache(store, 6)
    try:
        cache.upsert_dirty_blocks({0: torch.full((B, D), 100.0)})
        cache.evict_and_flush(1)  # block 0 waits in the flushing buffer
        reserve = cache._reserve_inflight_read

        def reserve_after_the_flush(block_id):
            store.gate.set()
            cache.flush_queue.join()  # its entry goes back before block 1 is loaded
            return reserve(block_id)

        cache._reserve_inflight_read = reserve_after_the_flush
        got = cache.prefetch([0, 1])
        assert torch.equal(got[0], torch.full((B, D), 100.0))
        assert torch.equal(got[1], torch.full((B, D), 1.0))
        assert cache.get_stats()["free_entries"] == 5  # block 1's is in use
    finally:
        store.gate.set()
        cache.shutdown()
