"""The list of alternatives that a warp's lanes share while they look through a row's groups again
(csrc/log_probs.cu: Best, look_at), restated on the CPU: lanes that run in any order between the warp's barriers. What is
checked is that all lanes take the same decision to shorten the list, that its room holds, and that the best are left."""

import random

import pytest

LANES, MANY, EACH = 4, 4, 2        # EACH: keys a lane adds in a step at most
ROOM = MANY + LANES * EACH


class Apart(Exception):
    """Lanes wait at different barriers, or the list has run out of its room."""


class List:
    def __init__(self):
        self.keys, self.count, self.least = [0] * ROOM, 0, 0


def lane(me, best, steps, top, mended):
    """One lane, as a generator: it yields before what it does to the list, and a barrier's name at a barrier."""
    least = 0
    for step in steps:
        for key in step[me]:
            if key > least:
                yield None
                if best.count == ROOM:
                    raise Apart
                best.keys[best.count] = key
                best.count += 1
        yield "added"
        count = best.count
        if mended:
            yield "read"
        else:
            yield None
        if count > MANY:
            yield "keep"
            n = best.count
            yield "counted"
            if me == 0:
                best.keys[:top] = sorted(best.keys[:n], reverse=True)[:top]
                best.count, best.least = min(n, top), best.keys[top - 1] if n >= top else 0
            yield "kept"
            least = best.least or least
            yield "known"


def run(steps, top, seed, mended):
    """The best `top` keys of all steps, or Apart."""
    r, best = random.Random(seed), List()
    lanes = [lane(i, best, steps, top, mended) for i in range(LANES)]
    waiting = [None] * LANES
    while lanes.count(None) < LANES:
        ready = [i for i in range(LANES) if lanes[i] and waiting[i] is None]
        if not ready:
            at = {waiting[i] for i in range(LANES) if lanes[i]}
            if len(at) != 1 or None in lanes:
                raise Apart
            waiting = [None] * LANES
            continue
        i = r.choice(ready)
        try:
            waiting[i] = next(lanes[i])
        except StopIteration:
            lanes[i] = None
    return sorted(best.keys[:best.count], reverse=True)[:top]


@pytest.mark.parametrize("top", [1, 3, 4])
def test_lanes_shorten_the_list_together(top):
    unmended = 0
    for seed in range(200):
        r = random.Random(1000 + seed)
        keys = list(range(1, 6 * LANES * EACH + 1))
        if seed % 2:
            r.shuffle(keys)  # else rising: every key reaches the list
        steps = [[[keys.pop(0) for _ in range(EACH)] for _ in range(LANES)] for _ in range(6)]
        want = sorted((k for step in steps for lane in step for k in lane), reverse=True)[:top]
        assert run(steps, top, seed, mended=True) == want
        try:
            unmended += run(steps, top, seed, mended=False) != want
        except Apart:
            unmended += 1
    assert unmended > 0  # what the second barrier is for
