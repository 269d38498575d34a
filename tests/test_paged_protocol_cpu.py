"""CPU model of the page ring of the few-row attention kernel (csrc/pattn.cu): 4 warps take the pages of a split in turn
from 6 slots, each slot with one full barrier (phases, parity waits) and a count of its fills; the warp that consumed a slot
refills it with the page 6 further on, which another warp will read. Random interleavings of warps and copies: no warp reads
a slot that does not hold its page, no copy lands in a slot that is being read or behind the kernel's end, and the kernel
ends. Without looking at the fill count a warp a lap ahead passes on the parity of the phase before the last; the model
shows it."""
import random

import pytest

WARPS, SLOTS = 4, 6


def run(n, rng, look_at_fills):
    """None, or what went wrong."""
    phase, pending, holds, fills, reading = [0] * SLOTS, [0] * SLOTS, [None] * SLOTS, [0] * SLOTS, [None] * SLOTS
    flights = []                                       # (slot, page) of copies under way

    def issue(page):
        s = page % SLOTS
        if pending[s]:
            return "a second copy into a slot whose first is under way"
        pending[s] = 1
        flights.append((s, page))
        fills[s] = page // SLOTS + 1
        return None

    for page in range(min(n, SLOTS)):
        issue(page)
    at = list(range(WARPS))                            # page each warp is at
    stage = ["wait"] * WARPS
    slow = rng.randrange(WARPS)                        # one warp that is scheduled seldom
    for _ in range(100000):
        if all(p >= n for p in at):
            return "a copy lands after the end" if flights else None
        if flights and rng.random() < 0.3:
            s, page = flights.pop(rng.randrange(len(flights)))
            if reading[s] is not None:
                return "a copy lands in a slot that is being read"
            holds[s], pending[s] = page, 0
            phase[s] += 1
            continue
        w = rng.randrange(WARPS)
        if (w == slow and rng.random() < 0.95) or at[w] >= n:
            continue
        page = at[w]
        s, lap = page % SLOTS, page // SLOTS
        if stage[w] == "wait":
            if look_at_fills and fills[s] < lap + 1:
                continue
            # parity wait: passes when the phase of this parity is complete, that is when the current one has the other
            if phase[s] % 2 == lap % 2:
                continue
            if holds[s] != page:
                return "a warp reads another page than its own"
            reading[s], stage[w] = w, "read"
        else:
            reading[s], stage[w] = None, "wait"
            at[w] += WARPS
            if page + SLOTS < n:
                bad = issue(page + SLOTS)
                if bad:
                    return bad
    return "no end"


@pytest.mark.parametrize("n", [0, 1, 5, 6, 7, 20, 64])
def test_ring_hands_every_page_to_its_warp(n):
    for seed in range(60):
        assert run(n, random.Random(seed), True) is None


def test_parity_alone_is_not_enough():
    assert any(run(40, random.Random(seed), False) for seed in range(200))
