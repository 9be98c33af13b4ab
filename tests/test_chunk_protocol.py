"""Model check of the barrier protocol of the cached attention's tcgen05 kernel (csrc/kv4_chunk.cu,
`kv4_chunk`), on the CPU.

As test_bwd_protocol.py does for the backward: each role of one CTA is a generator that follows the
kernel's loops and waits, barriers count arrivals per phase and are waited for by parity, the MMAs of
the one issuing thread run in order and a commit arrives once all before it have run, and a
scheduler with random speeds interleaves everything.  Checked: no parity wait sees its barrier
outside the phase meant or the next; no unpacked tile, score buffer, query buffer or accumulator is
written while something may still read it, nor read before it is written; nothing deadlocks.
"""
import random

import pytest

from test_bwd_protocol import Bar, Wait


class Cta:
    def __init__(self, items, ring, rng, warps=2, unpackers=2, skip=()):
        self.items, self.ring, self.rng, self.W, self.U = items, ring, rng, warps, unpackers  # tiles of each item
        self.skip = set(skip)
        self.q_full, self.q_free = ([Bar(n) for _ in range(2)] for n in (1, 2 * warps + 1))
        self.kv_full, self.kv_free = ([Bar(n) for _ in range(ring)] for n in (unpackers, 1))
        self.s_full, self.p_full, self.pv_done = ({(h, b): Bar(n) for h in (0, 1) for b in (0, 1)} for n in (1, warps, 1))
        self.queue = []
        self.unpacked, self.read_table, self.read_s, self.wrote_p = {}, {}, {}, {}
        self.s_done, self.pv = set(), set()
        self.q_loaded, self.left_q = set(), {}  # items whose queries are there; warps done with an item's buffer
        self.rescaling = {0: 0, 1: 0}           # warps at work on an accumulator
        self.read_o = {}

    def wait(self, bar, k, what):
        if what not in self.skip:
            yield Wait(bar, k, what)

    # ------------------------------------------------------------ roles
    def accumulate(self, m, first):
        for h in (0, 1):
            yield from self.wait(self.p_full[h, m & 1], m >> 1, "mma: p_full")
            self.queue += [("pv", m, h, first), ("commit", self.pv_done[h, m & 1])]
        self.queue.append(("commit", self.kv_free[m % self.ring]))

    def mma(self):
        n = 0
        for k, tiles in enumerate(self.items):
            yield from self.wait(self.q_full[k & 1], k >> 1, "mma: q_full")
            if "mma: q_free" not in self.skip:
                self.q_free[k & 1].arrive()
            for i in range(tiles):
                yield from self.wait(self.kv_full[n % self.ring], n // self.ring, "mma: kv_full")
                for h in (0, 1):
                    self.queue += [("s", n, h, k), ("commit", self.s_full[h, n & 1])]
                if i > 0:
                    yield from self.accumulate(n - 1, i == 1)
                n += 1
            if tiles > 0:
                yield from self.accumulate(n - 1, tiles == 1)

    def unpack(self, w):
        n = 0
        for tiles in self.items:
            for _ in range(tiles):
                if n >= self.ring:
                    yield from self.wait(self.kv_free[n % self.ring], n // self.ring - 1, "unpack: kv_free")
                    old = n - self.ring
                    assert all((old, h) in self.pv and (old, h) in self.s_done for h in (0, 1)), "tile replaced while read"
                    assert len(self.read_table.get(old, ())) == 2 * self.W, "table replaced while read"
                self.unpacked.setdefault(n, set()).add(w)
                self.kv_full[n % self.ring].arrive()
                n += 1

    def query(self):
        for k in range(len(self.items) + 1):  # the last one says that there are no more
            if k >= 2:
                yield from self.wait(self.q_free[k & 1], (k >> 1) - 1, "query: q_free")
                assert len(self.left_q.get(k - 2, ())) == 2 * self.W, "query buffer replaced while in use"
            yield None  # the copies take their time
            self.q_loaded.add(k)
            self.q_full[k & 1].arrive()

    def softmax(self, h, w):
        n = 0
        for k, tiles in enumerate(self.items):
            yield from self.wait(self.q_full[k & 1], k >> 1, "softmax: q_full")
            assert k in self.q_loaded, "query row read before it is there"
            for i in range(tiles):
                yield from self.wait(self.kv_full[n % self.ring], n // self.ring, "softmax: kv_full")
                yield from self.wait(self.s_full[h, n & 1], n >> 1, "softmax: s_full")
                assert (n, h) in self.s_done, "scores read before they are there"
                assert len(self.unpacked[n]) == self.U, "table read before it is there"
                self.read_s.setdefault((n, h), set()).add(w)
                if i > 0 and self.rng.random() < 0.4:
                    yield from self.wait(self.pv_done[h, (n - 1) & 1], (n - 1) >> 1, "softmax: pv_done (rescale)")
                    assert (n - 1, h) in self.pv, "accumulator rescaled under a product"
                    self.rescaling[h] += 1
                    yield None
                    self.rescaling[h] -= 1
                self.read_table.setdefault(n, set()).add((h, w))
                self.wrote_p.setdefault((n, h), set()).add(w)
                self.p_full[h, n & 1].arrive()
                n += 1
            if tiles > 0:
                yield from self.wait(self.pv_done[h, (n - 1) & 1], (n - 1) >> 1, "softmax: pv_done (output)")
                assert (n - 1, h) in self.pv, "output read before the last product"
            yield None
            self.read_o.setdefault((k, h), set()).add(w)  # rows staged in the item's own query buffer
            self.left_q.setdefault(k, set()).add((h, w))
            self.q_free[k & 1].arrive()
        k = len(self.items)
        yield from self.wait(self.q_full[k & 1], k >> 1, "softmax: q_full")
        assert k in self.q_loaded, "end read before it is there"

    # ------------------------------------------------------------ products
    def run_mma(self):
        op = self.queue.pop(0)
        if op[0] == "commit":
            op[1].arrive()
        elif op[0] == "s":
            _, n, h, k = op
            assert len(self.unpacked.get(n, ())) == self.U and k in self.q_loaded, "scores of operands that are not there"
            if n >= 2:
                assert (n - 2, h) in self.pv and len(self.read_s[n - 2, h]) == self.W, "score buffer overwritten while in use"
            self.s_done.add((n, h))
        else:
            _, m, h, first = op
            assert len(self.wrote_p.get((m, h), ())) == self.W, "product before the weights are there"
            assert self.rescaling[h] == 0, "product while the accumulator is rescaled"
            if first:
                k = self.item_of(m)
                assert k == 0 or len(self.read_o.get((k - 1, h), ())) == self.W, "accumulator overwritten before it is read"
            self.pv.add((m, h))

    def item_of(self, m):
        k = 0
        while m >= self.items[k]:
            m -= self.items[k]
            k += 1
        return k

    def simulate(self):
        agents = [self.mma(), self.query()] + [self.unpack(w) for w in range(self.U)]
        agents += [self.softmax(h, w) for h in (0, 1) for w in range(self.W)]
        waits, live = [None] * len(agents), list(range(len(agents)))
        speeds = [0.01, 0.1, 1.0, 1.0, 10.0]
        weight, w_mma = [self.rng.choice(speeds) for _ in agents], self.rng.choice(speeds)
        while live or self.queue:
            ready = [i for i in live if waits[i] is None or waits[i].ready()]
            choices = ready + (["mma"] if self.queue else [])
            assert choices, "deadlock: " + ", ".join(waits[i].what for i in live if waits[i] is not None)
            pick = self.rng.choices(choices, [weight[i] for i in ready] + ([w_mma] if self.queue else []))[0]
            if pick == "mma":
                self.run_mma()
                continue
            try:
                waits[pick] = next(agents[pick])
            except StopIteration:
                live.remove(pick)
        assert len(self.pv) == 2 * sum(self.items)


def _items(rng, least=1):
    return [rng.choice([0, 0, 1, 1, 2, 3, 5, 11]) for _ in range(rng.randint(least, 6))]


@pytest.mark.parametrize("ring", [2, 3])
def test_chunk_barrier_protocol(ring):
    rng = random.Random(ring)
    for _ in range(150):
        Cta(_items(rng), ring, rng).simulate()


def test_items_without_tiles_need_the_products_to_keep_up():
    """Without the MMA warp's arrival at q_free, a query buffer could pass two phases while it waits for one."""
    rng, caught = random.Random(5), 0
    for _ in range(300):
        cta = Cta([0] * 6 + [1, 0, 0, 2], 2, rng, skip={"mma: q_free"})
        for bar in cta.q_free:
            bar.count -= 1
        try:
            cta.simulate()
        except AssertionError:
            caught += 1
    assert caught > 0


# The softmax's wait for kv_full follows from its wait for the scores, whose operand that is;
# it is there so that the reading threads have themselves seen the writes.
@pytest.mark.parametrize("what", ["mma: p_full", "mma: q_full", "mma: kv_full", "unpack: kv_free", "query: q_free",
                                  "softmax: q_full", "softmax: s_full", "softmax: pv_done (rescale)", "softmax: pv_done (output)"])
def test_the_model_notices_a_missing_wait(what):
    rng = random.Random(sum(map(ord, what)))
    caught = 0
    for _ in range(80):
        try:
            Cta(_items(rng, 4), 2, rng, skip={what}).simulate()
        except AssertionError:
            caught += 1
    assert caught > 0
