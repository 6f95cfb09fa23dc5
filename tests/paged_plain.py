"""A KV cache in pages, restated in numpy for the tests: sequences' slots scattered over a pool in a random
order, and every slot that no sequence holds NaN, so that what reads one shows."""
import numpy as np

import bchip

DTYPE = {bchip.F32: np.float32, bchip.F16: np.float16}


class Batch:
    """Sequences of `lens` slots, the last `rows` of each new; `pad` rows behind the last sequence's. Slots'
    K and V are drawn into a pool of shuffled pages; the table's entries past a list are no page."""

    def __init__(self, rng, rows, lens, nkv, hd, kv_type, page_slots=16, pad=0, spare=3, stride=None, scale=1.0):
        self.rows, self.lens, self.nkv, self.hd, self.kv_type, self.page_slots = list(rows), list(lens), nkv, hd, kv_type, page_slots
        self.starts = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.uint32)
        self.total = int(self.starts[-1]) + pad
        held = [-(-n // page_slots) for n in self.lens]
        self.npages = sum(held) + spare
        order = rng.permutation(self.npages).astype(np.uint32)
        self.stride = max(held + [1]) if stride is None else stride
        self.table = np.full((len(self.lens), self.stride), 0xFFFFFFFF, np.uint32)
        for i, (a, n) in enumerate(zip(np.cumsum([0] + held), held)):
            self.table[i, :n] = order[a:a + n]
        self.k, self.v = (np.full((self.npages, page_slots, nkv, hd), np.nan, DTYPE[kv_type]) for _ in range(2))
        self.draw(rng, scale)

    def draw(self, rng, scale=1.0):
        for i, n in enumerate(self.lens):
            p, o = self.places(i)
            for pool in (self.k, self.v):
                pool[p, o] = (rng.standard_normal((n, self.nkv, self.hd)) * scale).astype(pool.dtype)

    def places(self, i):
        """Pages and slots in them of sequence i."""
        t = np.arange(self.lens[i])
        return self.table[i, t // self.page_slots], t % self.page_slots

    def of(self, pool, i):
        """Sequence i's slots of a pool."""
        return pool[self.places(i)]

    def args(self, ctx):
        """What the calls take between their data and their heads."""
        return self.starts, np.array(self.lens, np.uint32), ctx.upload(self.table), self.stride, self.page_slots, self.npages
