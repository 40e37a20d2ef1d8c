"""CPU restatement of the expert kernels' ring (csrc/moe.cu): a producer fills S
stages in turn, slab i belongs to split i % 3, four warps of a split read a slab
and release it, and a warp follows a stage's phase from its own slabs only.
Random interleavings; a barrier wait is by phase parity, as mbarriers have it.
With a number of stages that is not a multiple of the splits a warp can take a
phase for one that is two behind, which the simulation shows."""

import random

import pytest

STAGES, SPLITS, TILES = 9, 3, 4  # MOE_S, MOE_KS, MOE_RT


class Bar:
    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0

    def arrive(self):
        assert self.pending > 0
        self.pending -= 1
        if self.pending == 0:
            self.phase += 1
            self.pending = self.count

    def done(self, parity):  # the wait for the phase of this parity passes
        return (self.phase & 1) != parity


def simulate(seed, units, slabs, stages=STAGES):
    rng = random.Random(seed)
    full = [Bar(1) for _ in range(stages)]
    empty = [Bar(TILES) for _ in range(stages)]
    slot, flying, got = [None] * stages, [], []
    total = units * slabs

    def producer():
        for i in range(total):
            s = i % stages
            while i >= stages and not empty[s].done((i // stages - 1) & 1):
                yield
            flying.append((s, i))
            yield

    def warp(split, tile):
        first, slab, s, phase, shift = split, split, split, 0, slabs % SPLITS
        for unit in range(units):
            while slab < slabs:
                while not full[s].done(phase):
                    yield
                assert slot[s] == unit * slabs + slab
                got.append((tile, slot[s]))
                yield
                empty[s].arrive()
                s += SPLITS
                if s >= stages:
                    s, phase = s - stages, phase ^ 1
                slab += SPLITS
            first = first - shift if first >= shift else first - shift + SPLITS
            slab = first

    todo = [producer()] + [warp(k, t) for k in range(SPLITS) for t in range(TILES)]
    while todo or flying:
        if flying and rng.random() < 0.2:
            s, i = flying.pop(rng.randrange(len(flying)))
            slot[s] = i
            full[s].arrive()
        elif todo:
            k = min(int(rng.expovariate(0.3)), len(todo) - 1)  # some run far ahead of others
            try:
                next(todo[k])
            except StopIteration:
                todo.pop(k)
            if rng.random() < 0.05:
                rng.shuffle(todo)
    assert sorted(got) == sorted((t, i) for t in range(TILES) for i in range(total))


@pytest.mark.parametrize("block", range(4))
def test_every_slab_is_read_once_by_its_split(block):
    for seed in range(50 * block, 50 * block + 50):
        r = random.Random(seed)
        simulate(seed, units=r.randint(1, 8), slabs=r.randint(1, 11))


def test_stages_that_change_hands_between_splits_would_be_misread():
    with pytest.raises(AssertionError):
        for seed in range(200):
            simulate(seed, units=6, slabs=7, stages=8)
