"""Host model of the span tile kernel's pipeline (vllm_b200/csrc/tvp_span_tiles.cu):
its warps, barriers and parities, stepped in random orders with copies and MMAs
that finish any time after they were issued (those of one thread in order).
Every order ends, no buffer is overwritten before its last reader, and every
chunk of keys is added once, by its side, in order."""
import random
import re
from pathlib import Path

import pytest

SOURCE = (Path(__file__).resolve().parents[1] / "vllm_b200/csrc/tvp_span_tiles.cu").read_text()
STAGES = int(re.search(r"constexpr int kStages = (\d+);", SOURCE).group(1))


class Barrier:
    """An mbarrier: `count` arrivals complete a phase; wait(parity) passes once the
    phase of that parity is complete (a fresh barrier passes parity 1)."""

    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count

    def passed(self, parity):
        return (self.phase & 1) != parity


class Tile:
    def __init__(self, chunks, quarters):
        self.chunks, self.quarters = chunks, quarters
        self.q_full, self.o_full = Barrier(4), Barrier(1)
        side = lambda n: [Barrier(n), Barrier(n)]  # noqa: E731
        self.s_full, self.s_read, self.p_full, self.pv_done = side(1), side(quarters), side(quarters), side(1)
        self.kv_full = [Barrier(2) for _ in range(STAGES)]
        self.kv_empty = [Barrier(1) for _ in range(STAGES)]
        self.ring = [{"K": None, "V": None} for _ in range(STAGES)]
        self.s, self.s_readers = None, 0  # chunk whose scores S holds, warps that still read it
        self.p = [[None] * quarters, [None] * quarters]
        self.o = [[], []]
        self.s_done, self.finished = [], 0
        self.queues = []  # one per issuing thread: functions that run in order, later

    def producer(self, which):
        queue = []
        self.queues.append(queue)
        stage, parity = 0, 1
        for c in range(self.chunks):
            if c >= STAGES:
                yield lambda: self.kv_empty[stage].passed(parity)

            def land(c=c, stage=stage):
                old = self.ring[stage][which]
                if old is not None:
                    assert old in self.s_done and old in self.o[old & 1], f"chunk {old} overwritten by {c}"
                self.ring[stage][which] = c
                self.kv_full[stage].arrive()
            queue.append(land)
            stage += 1
            if stage == STAGES:
                stage, parity = 0, parity ^ 1

    def s_issuer(self):
        queue = []
        self.queues.append(queue)
        stage, parity = 0, 0
        yield lambda: self.q_full.passed(0)
        for c in range(self.chunks):
            yield lambda: self.kv_full[stage].passed(parity)
            if c > 0:
                yield lambda: self.s_read[(c - 1) & 1].passed(((c - 1) >> 1) & 1)

            def mma(c=c, stage=stage):
                assert self.ring[stage]["K"] == c
                assert self.s_readers == 0, f"scores of chunk {self.s} overwritten by {c}"
                self.s, self.s_readers = c, self.quarters
                self.s_done.append(c)
                self.s_full[c & 1].arrive()
            queue.append(mma)
            stage += 1
            if stage == STAGES:
                stage, parity = 0, parity ^ 1

    def pv_issuer(self):
        queue = []
        self.queues.append(queue)
        stage = 0
        for c in range(self.chunks):
            side = c & 1
            yield lambda: self.p_full[side].passed((c >> 1) & 1)

            def mma(c=c, stage=stage, side=side):
                assert self.ring[stage]["V"] == c and self.p[side] == [c] * self.quarters
                self.o[side].append(c)
                self.pv_done[side].arrive()
                self.kv_empty[stage].arrive()
            queue.append(mma)
            stage = (stage + 1) % STAGES
        queue.append(self.o_full.arrive)

    def softmax(self, side, quarter):
        if side == 0:
            self.q_full.arrive()
        if quarter < self.quarters:
            parity = 0
            for c in range(side, self.chunks, 2):
                yield lambda: self.s_full[side].passed(parity)
                assert self.s == c
                yield lambda: True  # the scores are on their way into registers
                assert self.s == c
                self.s_readers -= 1
                self.s_read[side].arrive()
                if c >= 2:
                    yield lambda: self.pv_done[side].passed(parity ^ 1)
                    assert c - 2 in self.o[side]
                parity ^= 1
                yield lambda: True  # exponentials
                self.p[side][quarter] = c
                self.p_full[side].arrive()
            yield lambda: self.o_full.passed(0)
            assert self.o == [list(range(0, self.chunks, 2)), list(range(1, self.chunks, 2))]
        self.finished += 1

    def run(self, rng):
        agents = [self.producer("K"), self.producer("V"), self.s_issuer(), self.pv_issuer()]
        agents += [self.softmax(s, q) for s in (0, 1) for q in range(4)]
        waits = {a: (lambda: True) for a in agents}
        while waits or any(self.queues):
            ready = [a for a, ok in waits.items() if ok()]
            queued = [q for q in self.queues if q]
            assert ready or queued, "no warp can go on"
            pick = rng.randrange(len(ready) + len(queued))
            if pick >= len(ready):
                queued[pick - len(ready)].pop(0)()
                continue
            try:
                waits[ready[pick]] = next(ready[pick])
            except StopIteration:
                del waits[ready[pick]]
        assert self.finished == 8


@pytest.mark.parametrize("quarters", [1, 2, 3, 4])
@pytest.mark.parametrize("chunks", list(range(1, 4 * STAGES)))
def test_every_order_of_the_tile_pipeline_ends(chunks, quarters):
    for seed in range(25):
        Tile(chunks, quarters).run(random.Random(1000 * chunks + 10 * quarters + seed))


def test_the_model_sees_a_missing_wait():
    """Without the wait for P V of two chunks before, P is overwritten in some order."""
    class Hasty(Tile):
        def softmax(self, side, quarter):
            for ok in super().softmax(side, quarter):
                cells = dict(zip(ok.__code__.co_freevars, ok.__closure__ or ()))
                pv = "parity" in cells and "pv_done" in ok.__code__.co_names
                yield (lambda: True) if pv else ok
    with pytest.raises(AssertionError):
        for seed in range(200):
            Hasty(9, 4).run(random.Random(seed))
