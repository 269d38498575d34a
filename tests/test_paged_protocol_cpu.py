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


# ------------------------------------------------------------------------------------------------ many query rows
class Bar:
    """An mbarrier: `count` arrivals complete a phase."""

    def __init__(self, count):
        self.count = self.pending = count
        self.phase = 0                                   # phases completed

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0, "too many arrivals in a phase"
        if self.pending == 0:
            self.phase, self.pending = self.phase + 1, self.count


class ManyRows:
    """The many-row attention CTA (csrc/prows.cu): 4 widening warps, the MMA issuer, 4 softmax warps for each of two row tiles;
    a warp's 32 arrivals are one here. MMAs on one accumulator complete in the order of issue, on different ones in any;
    a commit arrives when all that was issued before it has completed. `broken` leaves one wait out."""
    STAGES = 4

    def __init__(self, n, seed, broken=None):
        self.n, self.rng, self.broken = n, random.Random(seed), broken
        self.q_full, self.drain = Bar(8), Bar(1)
        self.k_full, self.v_full = ([Bar(4) for _ in range(self.STAGES)] for _ in range(2))
        self.k_empty, self.v_empty = ([Bar(1) for _ in range(self.STAGES)] for _ in range(2))
        self.s_full, self.o_done = ([[Bar(1), Bar(1)] for _ in range(2)] for _ in range(2))
        self.p_full = [[Bar(4), Bar(4)] for _ in range(2)]
        self.k_holds, self.v_holds = ([[None] * 4 for _ in range(self.STAGES)] for _ in range(2))     # page a warp's part is of
        self.s_holds = [[None, None], [None, None]]      # [tile][buffer]: ("scores", u), or {warp: u} of weights
        self.o_pages = [0, 0]                            # products complete on O
        self.flight = []                                 # MMAs under way: (number, accumulator, what it reads, callback)
        self.issued, self.commits = 0, []

    def wait(self, bar, k, name=None):
        """The parity wait for phase k of a barrier (phase -1: the fresh barrier's)."""
        if name is not None and name == self.broken:
            return
        while bar.phase <= k:
            yield
        assert bar.phase <= k + 1, "a wait two phases late: its parity would be wrong"

    def issue(self, accumulator, reads, done):
        self.flight.append((self.issued, accumulator, reads, done))
        self.issued += 1

    def commit(self, bar):
        self.commits.append((self.issued, bar))
        self.settle()

    def settle(self):
        first = min((f[0] for f in self.flight), default=self.issued)
        ready = [bar for upto, bar in self.commits if upto <= first]
        self.commits = [c for c in self.commits if c[0] > first]
        for bar in ready:
            bar.arrive()

    def complete_one(self):
        heads = {}
        for f in self.flight:
            heads.setdefault(f[1], f)
        f = self.rng.choice(list(heads.values()))
        self.flight.remove(f)
        f[3]()
        self.settle()

    def read_by_mma(self, what):
        return any(what in f[2] or what == f[1] for f in self.flight)

    # -- roles
    def widen(self, w):
        for u in range(self.n):
            s = u % self.STAGES
            for holds, full, empty, kind in ((self.k_holds, self.k_full, self.k_empty, "k"),
                                             (self.v_holds, self.v_full, self.v_empty, "v")):
                yield from self.wait(empty[s], u // self.STAGES - 1, kind + "_empty")
                assert not self.read_by_mma((kind, s)), f"{kind} stage written under an MMA"
                holds[s][w] = u
                yield
                full[s].arrive()

    def scores(self, t, u):
        e, s = u & 1, u % self.STAGES
        assert self.k_holds[s] == [u] * 4, "scores of another page"
        assert not self.read_by_mma(("s", t, e)), "scores over weights that a product reads"
        held = self.s_holds[t][e]
        assert held is None or held == {w: u - 2 for w in range(4)}, "scores over scores that were not read"
        self.s_holds[t][e] = "under way"

        def done():
            self.s_holds[t][e] = ("scores", u)
        self.issue(("s", t, e), {("k", s)}, done)
        self.commit(self.s_full[t][e])

    def issuer(self):
        n = self.n
        yield from self.wait(self.q_full, 0)
        for u in range(min(n, 2)):
            yield from self.wait(self.k_full[u], 0)
            self.scores(0, u)
            yield
            self.scores(1, u)
            self.commit(self.k_empty[u])
        for u in range(n):
            s, e = u % self.STAGES, u & 1
            yield from self.wait(self.v_full[s], u // self.STAGES)
            for t in range(2):
                yield from self.wait(self.p_full[t][e], u >> 1)
                assert self.s_holds[t][e] == {w: u for w in range(4)} and self.v_holds[s] == [u] * 4

                def done(t=t):
                    self.o_pages[t] += 1
                self.issue(("o", t), {("v", s), ("s", t, e)}, done)
                self.commit(self.o_done[t][e])
                yield
            self.commit(self.v_empty[s])
            if u + 2 < n:
                yield from self.wait(self.k_full[(u + 2) % self.STAGES], (u + 2) // self.STAGES)
                for t in range(2):
                    yield from self.wait(self.o_done[t][e], u >> 1, "o_done before scores")
                    self.scores(t, u + 2)
                    yield
                self.commit(self.k_empty[(u + 2) % self.STAGES])
        self.commit(self.drain)
        yield from self.wait(self.drain, 0)
        assert not self.flight

    def softmax(self, t, w):
        self.q_full.arrive()
        yield
        for u in range(self.n):
            e = u & 1
            yield from self.wait(self.s_full[t][e], u >> 1)
            held = self.s_holds[t][e]
            assert held == ("scores", u) or (type(held) is dict and w not in held and set(held.values()) == {u}), "wrong scores"
            yield
            if u and self.rng.random() < 0.4:            # the maximum moved: O is rescaled
                yield from self.wait(self.o_done[t][(u - 1) & 1], (u - 1) >> 1, "o_done before rescale")
                assert not self.read_by_mma(("o", t)), "O rescaled under a product"
                assert self.o_pages[t] == u, "O rescaled before the last page's product"
                yield
            assert not self.read_by_mma(("s", t, e)), "weights written under an MMA"
            if type(self.s_holds[t][e]) is not dict:
                self.s_holds[t][e] = {}
            self.s_holds[t][e][w] = u
            yield
            self.p_full[t][e].arrive()
        if self.n:
            yield from self.wait(self.o_done[t][(self.n - 1) & 1], (self.n - 1) >> 1)
            assert self.o_pages[t] == self.n and not self.read_by_mma(("o", t)), "O read before its products"

    def run(self):
        roles = [self.widen(w) for w in range(4)] + [self.softmax(t, w) for t in range(2) for w in range(4)]
        if self.n:
            roles.append(self.issuer())
        slow = self.rng.choice(roles)
        for _ in range(400 * (self.n + 1) + 100000):
            if not roles:
                assert not self.flight and not self.commits
                return
            if self.flight and self.rng.random() < 0.2:
                self.complete_one()
                continue
            r = self.rng.choice(roles)
            if r is slow and self.rng.random() < 0.9:
                continue
            try:
                next(r)
            except StopIteration:
                roles.remove(r)
        raise AssertionError("no end")


@pytest.mark.parametrize("n", [0, 1, 2, 3, 5, 8, 21])
def test_many_rows_hand_every_page_on(n):
    for seed in range(40):
        ManyRows(n, seed).run()


@pytest.mark.parametrize("broken", ["k_empty", "v_empty", "o_done before scores", "o_done before rescale"])
def test_many_rows_need_every_wait(broken):
    def fails(seed):
        try:
            ManyRows(12, seed, broken).run()
        except AssertionError:
            return True
        return False
    assert any(fails(seed) for seed in range(60))
