"""The ring of shared memory buffers between the copying and the issuing warps of the gated block's kernel,
restated on the CPU: barriers with phases and parities as mbarrier has them, arrivals that land at any later
time. What is checked is that a block which has made its waits has nothing on its way to it any more."""

import random

import pytest


class Barrier:
    """Counts arrivals; a phase ends with the count. wait(parity) passes once the phase of that parity is over."""

    def __init__(self, count=1):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def passes(self, parity):
        return (self.phase & 1) != parity


def run(stages, fills, seed, drained):
    """Fills a ring `fills` times in one block; releases land in order after random delays. Returns the number of
    releases that are still on their way when the block's last wait has passed."""
    r = random.Random(seed)
    full, empty = [Barrier() for _ in range(stages)], [Barrier() for _ in range(stages)]
    flying = []          # releases on their way: buffers, in order
    taken = 0            # fills that the products have read

    def land():          # the next event elsewhere: a product is done, or a release lands
        nonlocal taken
        stage = taken % stages
        if taken < fills and full[stage].passes(taken // stages & 1) and (not flying or r.random() < 0.5):
            flying.append(stage)
            taken += 1
        elif flying:
            empty[flying.pop(0)].arrive()

    def wait(barrier, parity):
        for _ in range(10 * (fills + stages) + 100):
            if barrier.passes(parity):
                return
            land()
        raise AssertionError("a wait that nothing ends")

    stage = phase = used = 0
    for _ in range(fills):
        wait(empty[stage], phase ^ 1)
        full[stage].arrive()
        used |= 1 << stage
        stage += 1
        if stage == stages:
            stage, phase = 0, phase ^ 1
    if drained:
        for i in range(stages):
            if used >> i & 1:
                wait(empty[i], phase if i < stage else phase ^ 1)
    return fills - taken + len(flying)


@pytest.mark.parametrize("stages", [5, 6])
def test_no_release_is_on_its_way_to_a_block_that_has_ended(stages):
    for fills in range(4 * stages + 1):
        for seed in range(20):
            assert run(stages, fills, seed, drained=True) == 0
    assert run(stages, 3, 0, drained=False) > 0  # what the waits at the end are for


class Copies(Barrier):
    """A barrier that also counts bytes, expected minus come: a phase ends when both counts are zero."""

    def __init__(self):
        super().__init__()
        self.bytes = 0

    def settle(self):
        if self.pending == 0 and self.bytes == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def expect(self, n):
        self.bytes += n
        self.pending -= 1
        self.settle()

    def come(self, n):
        self.bytes -= n
        self.settle()


def give_up(stages, own, other, read, seed, mended):
    """The first block has filled `own` buffers, the second `other`, the products have read `read` of them, and all
    warps have given up. Returns the copies that are still on their way after the waits at the end, or None where
    such a wait has nothing to end it."""
    r = random.Random(seed)
    full = [Copies() for _ in range(stages)]
    flying = []
    for i in range(max(own, other)):
        if i < own:
            full[i % stages].expect(2)
            flying.append(i)
        if i < other:
            flying.append(i)
        while i < read and i in flying:  # a buffer is filled again only after its products
            flying.remove(i)
            full[i % stages].come(1)
    if mended:
        for i in range(own, other):
            full[i % stages].expect(1)
        for i in range(other, own):
            full[i % stages].come(1)
    fills = max(own, other) if mended else own
    for i in range(stages):
        if fills > i:
            rounds = (fills - i + stages - 1) // stages
            while not full[i].passes((rounds - 1) & 1):
                if not flying:
                    return None
                full[flying.pop(r.randrange(len(flying))) % stages].come(1)
    return len(flying)


@pytest.mark.parametrize("stages", [5, 6])
def test_copies_have_landed_after_waits_that_ran_out(stages):
    """For all that two blocks can have filled, the second ahead or behind by up to the buffers that are free."""
    plain = []
    for read in range(2 * stages + 2):
        for own in range(read, read + stages + 1):
            for other in range(read, read + stages + 1):
                for seed in range(3):
                    assert give_up(stages, own, other, read, seed, mended=True) == 0
                plain.append(give_up(stages, own, other, read, 0, mended=False))
    assert None in plain and any(plain)  # what the first block's own count alone leaves behind
