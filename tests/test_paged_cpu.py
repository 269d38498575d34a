"""Paged cache and rotary: what is refused before any GPU work, and PagedCache's page bookkeeping against a model that
keeps every session's tokens in a list."""
import ctypes
import random

import pytest
import torch

from lingbot_b200 import _lib, paged_cache, rope


def test_pages_and_tables_are_checked():
    z = torch.zeros
    with pytest.raises(TypeError):
        paged_cache.Pages(z(2, 1, 64, 128), z(2, 1, 64, 128), z(2, 1), z(2, 1))
    i8 = torch.int8
    with pytest.raises(ValueError, match="codes"):
        paged_cache.Pages(z(2, 1, 32, 128, dtype=i8), z(2, 1, 32, 128, dtype=i8), z(2, 1), z(2, 1))
    with pytest.raises(ValueError, match="CUDA"):
        paged_cache.Pages(z(2, 1, 64, 128, dtype=i8), z(2, 1, 64, 128, dtype=i8), z(2, 1), z(2, 1))
    with pytest.raises(TypeError, match="format"):
        paged_cache.alloc_pages(1, 1, "cpu", torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        rope.tables(4, 8, device="cpu")
    for bad in ({"type": "linear", "factor": 0.5}, {"type": "other", "factor": 2.0},
                {"type": "banded", "factor": 2.0, "original": 10, "low": 4, "high": 4}):
        with pytest.raises(ValueError):
            rope.tables(4, 8, scaling=bad, device="cpu")
    for rot in (0, 7):
        with pytest.raises(ValueError, match="rot"):
            rope.tables(4, rot, device="cpu")


def _aligned(nbytes=4096):
    buf = ctypes.create_string_buffer(nbytes + 256)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    return buf, at


def test_c_entries_refuse_bad_arguments():
    """Every call here is refused before a CUDA call is made."""
    lib = _lib.load()
    keep, p = _aligned()
    err = lib.lbq_last_error

    def read(**kw):
        a = dict(kp=p, ka=p, vp=p, va=p, n=4, heads=1, fmt=0, table=p, st=4, width=4, start=None, s0=0, lens=None, b=1, l=8,
                 ko=p, vo=p, s=(1024, 128, 128), dtype=0)
        a.update(kw)
        return lib.lbq_page_read(a["kp"], a["ka"], a["vp"], a["va"], a["n"], a["heads"], a["fmt"], a["table"], a["st"],
                                 a["width"], a["start"], a["s0"], a["lens"], a["b"], a["l"], a["ko"], *a["s"], a["vo"],
                                 *a["s"], a["dtype"], None)
    for kw, rc, word in [(dict(kp=None), 1, b"null"), (dict(kp=p + 16), 2, b"aligned"), (dict(fmt=2), 1, b"fmt"),
                         (dict(n=0), 1, b"pages"), (dict(n=1 << 25), 1, b"2^31"), (dict(heads=0), 1, b"heads"),
                         (dict(table=None), 1, b"table"), (dict(width=0), 1, b"table"), (dict(b=0), 1, b"batch"),
                         (dict(b=2, st=3), 1, b"table"), (dict(l=-1), 1, b"len"), (dict(dtype=2), 1, b"dtype"),
                         (dict(s0=-1), 1, b"start"), (dict(s0=250), 1, b"outside"), (dict(ko=p + 2), 2, b"aligned"),
                         (dict(s=(1024, 129, 128)), 2, b"strides")]:
        assert read(**kw) == rc and word in err(), (kw, err())

    def copy(pairs=(0,), to=(1,), n=4, layers=1, lb=0, la=0):
        s, d = ((ctypes.c_int32 * len(x))(*x) for x in (pairs, to))
        return lib.lbq_page_copy(p, p, p, p, n, 1, layers, lb, la, s, d, len(pairs), None)
    assert copy(pairs=(4,)) == 1 and b"outside" in err()
    assert copy(to=(-1,)) == 1 and b"outside" in err()
    assert copy(layers=0) == 1
    assert copy(layers=2, lb=4 * 8192 - 128, la=4) == 1 and b"layer" in err()
    assert copy(pairs=(), to=()) == 0

    def attn(**kw):
        a = dict(q=p, out=p, table=p, width=4, kv=None, kv0=100, b=1, lq=1, group=1, splits=1, ws=None, wsb=0, heads=1)
        a.update(kw)
        return lib.lbq_paged_attn(a["q"], 1024, 128, 128, p, p, p, p, 4, a["heads"], 0, a["table"], 4, a["width"], a["kv"],
                                  a["kv0"], None, a["b"], a["lq"], a["group"], 0, 0.0, a["out"], 1024, 128, 128, None,
                                  a["splits"], a["ws"], a["wsb"], 0, None)
    for kw, rc, word in [(dict(q=None), 1, b"null"), (dict(out=p + 8), 2, b"aligned"), (dict(kv0=257), 1, b"kv_len"),
                         (dict(kv0=-1), 1, b"kv_len"), (dict(group=0), 1, b"group"), (dict(group=1 << 25), 1, b"group"), (dict(b=70000), 1, b"batch"),
                         (dict(splits=9, kv0=1152, width=18), 1, b"workspace"),
                         (dict(splits=9, kv0=1152, width=18, ws=p, wsb=8), 1, b"workspace"),
                         (dict(lq=1 << 28, group=5), 1, b"large")]:
        assert attn(**kw) == rc and word in err(), (kw, err())
    assert attn(lq=0) == 0
    assert lib.lbq_paged_attn_workspace(1, 1, 12, 1, 1) == 0
    assert lib.lbq_paged_attn_workspace(1, 1, 12, 1, 8) == 0          # one cluster
    assert lib.lbq_paged_attn_workspace(4, 1, 12, 1, 8) > 0           # more CTAs than the GPU holds at once
    assert lib.lbq_paged_attn_workspace(1, 1, 12, 1, 9) >= 9 * 12 * 130 * 4
    assert lib.lbq_paged_attn_workspace(1, 100, 12, 1, 2) >= 2 * 12 * 100 * 130 * 4
    assert lib.lbq_paged_attn_splits(1, 1, 12, 1, 1, 0) == 1
    assert lib.lbq_paged_attn_splits(1, 1, 12, 1, 30160, 0) > 1

    def write(**kw):
        a = dict(k=p, start=None, s0=0, l=8, cos=None, sin=None, rs=0, rr=0, rot=0, inter=1)
        a.update(kw)
        return lib.lbq_page_write(a["k"], 1024, 128, 128, p, 1024, 128, 128, p, p, p, p, 4, 1, 0, p, 4, 4, a["start"], a["s0"],
                                  None, 1, a["l"], a["cos"], a["sin"], a["rs"], a["rr"], a["rot"], a["inter"], None, 0, 0, 0,
                                  0, None)
    for kw, rc, word in [(dict(k=None), 1, b"null"), (dict(s0=249), 1, b"outside"), (dict(cos=p), 1, b"rope"),
                         (dict(cos=p, sin=p, rs=64, rr=4, rot=130), 1, b"rot"),
                         (dict(cos=p, sin=p, rs=64, rr=0, rot=128), 1, b"rows"),
                         (dict(cos=p, sin=p, rs=64, rr=4, rot=12), 2, b"rope"),
                         (dict(cos=p, sin=p, rs=64, rr=4, rot=24, inter=0), 2, b"rope"),
                         (dict(cos=p, sin=p, rs=66, rr=4, rot=128), 2, b"rope")]:
        assert write(**kw) == rc and word in err(), (kw, err())

    def turn(**kw):
        a = dict(x=p, h=1, x2=None, h2=0, dim=128, rot=128, start=0, dtype=0, l=4)
        a.update(kw)
        return lib.lbq_rope(a["x"], 512, 128, 128, p, 512, 128, 128, a["h"], a["x2"], 0, 0, 0, None, 0, 0, 0, a["h2"], 1,
                            a["l"], a["dim"], p, p, 64, 4, a["rot"], 1, None, 0, 0, 0, a["start"], 0, a["dtype"], None)
    for kw, rc, word in [(dict(x=None), 1, b"null"), (dict(dtype=3), 1, b"dtype"), (dict(h=0), 1, b"heads"),
                         (dict(x2=p), 1, b"x2"), (dict(dim=514), 1, b"dim"), (dict(rot=130), 1, b"rot"),
                         (dict(rot=3), 1, b"rot"), (dict(start=-1), 1, b"start"), (dict(x=p + 1), 2, b"aligned")]:
        assert turn(**kw) == rc and word in err(), (kw, err())
    assert turn(l=0) == 0
    del keep


class Tokens:
    """Stand-in pool on the CPU: one head; a token's code is its row of the pages."""

    def __init__(self, monkeypatch, num_pages, layers=2):
        monkeypatch.setattr(paged_cache.Pages, "__init__", lambda self, *t: vars(self).update(zip(("k", "v"), t)))
        monkeypatch.setattr(paged_cache.Pages, "layer", lambda self, i: self)
        shape = (layers, num_pages, 1, 64, 128)
        self.mem = torch.full((num_pages, 64), -1, dtype=torch.long)
        self.cache = paged_cache.PagedCache(paged_cache.Pages(
            torch.empty(shape, dtype=torch.int8), torch.empty(shape, dtype=torch.int8), torch.empty(shape[:3]),
            torch.empty(shape[:3])), max_pages=8)
        self.moves = []

        def copy(pages, src, dst):
            assert len(set(dst)) == len(dst) and not set(dst) & set(src)
            self.moves += list(zip(src, dst))
            self.mem[list(dst)] = self.mem[list(src)]
        monkeypatch.setattr(paged_cache, "copy_pages", copy)

    def write(self, plan, fresh):
        for b, n in enumerate(plan.new):
            for i in range(n):
                t = int(plan.start[b]) + i
                self.mem[int(plan.table[b, t // 64]), t % 64] = fresh[b][i]

    def read(self, s):
        ids, n = self.cache.page_ids(s), self.cache.tokens(s)
        return [int(self.mem[ids[t // 64], t % 64]) for t in range(n)]


@pytest.mark.parametrize("seed", range(6))
def test_bookkeeping_keeps_every_sessions_tokens(monkeypatch, seed):
    r = random.Random(seed)
    pool = Tokens(monkeypatch, 40)
    c, model, stamp = pool.cache, {}, 0
    for _ in range(300):
        what = r.choice(["open", "step", "step", "step", "fork", "close", "evict", "compact"])
        some = list(model)
        if what == "open" and len(model) < 6:
            model[c.open()] = []
        elif what == "step" and some:
            chosen = r.sample(some, r.randint(1, len(some)))
            new = [r.choice([0, 1, r.randint(1, 90)]) for _ in chosen]
            before = (c.free_pages, {s: c.page_ids(s) for s in some})
            try:
                plan = c.plan(chosen, new)
            except (RuntimeError, ValueError):
                assert before == (c.free_pages, {s: c.page_ids(s) for s in some})
                continue
            fresh = [[(stamp := stamp + 1) for _ in range(n)] for n in new]
            pool.write(plan, [[-7] * n for n in new])               # a pass that the next one replaces
            pool.write(plan, fresh)
            if r.random() < 0.8:
                c.commit(plan)
                for s, f in zip(chosen, fresh):
                    model[s] = model[s] + f
        elif what == "fork" and some and len(model) < 6:
            s = r.choice(some)
            model[c.fork(s)] = list(model[s])
        elif what == "close" and some:
            s = r.choice(some)
            c.close(s)
            del model[s]
        elif what == "evict" and some:
            s = r.choice(some)
            n = len(model[s]) // 64
            sink = r.randint(0, n) * 64
            out = r.randint(0, n - sink // 64) * 64
            c.evict(s, sink, out)
            model[s] = model[s][:sink] + model[s][sink + out:]
        elif what == "compact":
            c.compact()
            used = {p for s in model for p in c.page_ids(s)}
            assert not used or max(used) < len(used)
        for s in model:
            assert pool.read(s) == model[s] and c.tokens(s) == len(model[s])
        used = [p for s in model for p in c.page_ids(s)]
        assert len(set(used)) + c.free_pages == c.num_pages


def test_stale_plans_and_bad_calls_are_refused(monkeypatch):
    pool = Tokens(monkeypatch, 12)
    c = pool.cache
    a = c.open()
    c.commit(c.plan([a], 70))
    plan = c.plan([a], 5)
    b = c.fork(a)
    for call in (lambda: c.commit(plan), lambda: c.attend(0, plan, None), lambda: c.write(0, plan, None, None)):
        with pytest.raises(RuntimeError, match="plan again"):
            call()
    plan = c.plan([a, b], [3, 4])                                   # both write the shared unfinished page
    assert len(pool.moves) == 1 and c.page_ids(a)[1] != c.page_ids(b)[1] and c.page_ids(a)[0] == c.page_ids(b)[0]
    c.commit(plan)
    with pytest.raises(RuntimeError, match="moved on"):
        c.commit(plan)
    with pytest.raises(ValueError, match="twice"):
        c.plan([a, a], 1)
    with pytest.raises(KeyError):
        c.plan([99], 1)
    with pytest.raises(ValueError, match="exceed"):
        c.plan([a], 8 * 64)
    with pytest.raises(ValueError, match="multiples"):
        c.evict(a, 0, 10)
    with pytest.raises(ValueError, match="fewer"):
        c.evict(a, 64, 64)
    with pytest.raises(ValueError, match="negative"):
        c.plan([a], [-1])
    old = c.plan([b], 1)
    c.evict(b, 0, 64)
    with pytest.raises(RuntimeError, match="plan again"):
        c.commit(old)
    fixed = c.fixed_plan(1)
    table = fixed.table
    got = c.plan([b], 60, into=fixed)
    assert got is fixed and fixed.table is table and int(fixed.kv_lens[0]) == c.tokens(b) + 60
    before = (c.free_pages, c.page_ids(a), c.page_ids(b))
    with pytest.raises(ValueError, match="cannot take"):
        c.plan([a, b], 100, into=fixed)
    with pytest.raises(ValueError, match="fixed_plan"):
        c.plan([b], 100, into=c.plan([b], 1))
    assert before == (c.free_pages, c.page_ids(a), c.page_ids(b))
    r = type("R", (), {})()
    k = torch.zeros(1, 60, 1, 128)
    with pytest.raises(ValueError, match="positions"):                # 64 tokens of b were evicted
        c.write(0, fixed, k, k, rope=r)


def test_copy_pages_refuses_overlap():
    for src, dst, word in [([1, 2], [3], "source"), ([1, 2], [3, 3], "twice"), ([1, 2], [2, 3], "both")]:
        with pytest.raises(ValueError, match=word):
            paged_cache.copy_pages(None, src, dst)
    paged_cache.copy_pages(None, [], [])


def _state(c):
    return c.free_pages, list(c._refs), {s: (c.page_ids(s), c.tokens(s)) for s in c._sessions}


def test_a_plan_that_does_not_fit_changes_nothing_beside_surplus_pages(monkeypatch):
    """A session that still holds the pages of a larger plan, never committed, lends none of them to the others."""
    pool = Tokens(monkeypatch, 8)
    c = pool.cache
    a, b = c.open(), c.open()
    c.plan([a], 300)
    before = _state(c)
    with pytest.raises(RuntimeError, match="free"):
        c.plan([a, b], [1, 400])
    assert _state(c) == before
    # the same with pages that are shared: the forks' unfinished page would have to be copied
    pool = Tokens(monkeypatch, 7)
    c = pool.cache
    a, b = c.open(), c.open()
    c.plan([a], 300)
    plan = c.plan([b], 10)
    pool.write(plan, [list(range(10))])
    c.commit(plan)
    d = c.fork(b)
    c.fork(b)
    before = _state(c)
    with pytest.raises(RuntimeError, match="free"):
        c.plan([a, b, d], 1)
    assert _state(c) == before and pool.read(b) == pool.read(d) == list(range(10))
    c.commit(c.plan([a, b], 1))                                     # what does fit
    assert pool.read(b)[:10] == pool.read(d) == list(range(10)) and c.free_pages == 0


def test_a_copy_that_fails_leaves_the_sessions_as_they_were(monkeypatch):
    pool = Tokens(monkeypatch, 8)
    c = pool.cache
    a = c.open()
    c.commit(c.plan([a], 10))
    c.fork(a)
    before = _state(c)

    def fails(pages, src, dst):
        raise RuntimeError("no copy")
    monkeypatch.setattr(paged_cache, "copy_pages", fails)
    with pytest.raises(RuntimeError, match="no copy"):
        c.plan([a], 1)
    assert _state(c) == before


def test_starts_near_the_end_of_64_bits_are_refused():
    """start + length would pass 64 bits and come out negative, a page in front of the table. Refused on the host, with
    lens (a device pointer, which the host does not read) as well as without."""
    lib = _lib.load()
    keep, p = _aligned()
    for s0 in ((1 << 63) - 1, (1 << 63) - 8, 1 << 62):
        for lens in (None, p):
            assert lib.lbq_page_read(p, p, p, p, 4, 1, 0, p, 4, 4, None, s0, lens, 1, 8, p, 1024, 128, 128, p, 1024, 128, 128, 0,
                                     None) == 1 and b"start" in lib.lbq_last_error()
            assert lib.lbq_page_write(p, 1024, 128, 128, p, 1024, 128, 128, p, p, p, p, 4, 1, 0, p, 4, 4, None, s0, lens, 1, 8,
                                      None, None, 0, 0, 0, 0, None, 0, 0, 0, 0, None) == 1 and b"start" in lib.lbq_last_error()
        assert lib.lbq_rope(p, 512, 128, 128, p, 512, 128, 128, 1, None, 0, 0, 0, None, 0, 0, 0, 0, 1, 4, 128, p, p, 64, 4, 128, 1,
                            None, 0, 0, 0, s0, 0, 0, None) == 1 and b"start" in lib.lbq_last_error()
    del keep


def test_a_plan_ends_when_its_session_goes_on(monkeypatch):
    """After a commit the plan writes no more: its pages hold the tokens of later plans, whose scale a write would change.
    It still attends until the next commit, to what was committed."""
    pool = Tokens(monkeypatch, 12)
    c = pool.cache
    calls = []
    monkeypatch.setattr(paged_cache, "write", lambda *a, **kw: calls.append("write"))
    monkeypatch.setattr(paged_cache, "attend", lambda *a, **kw: calls.append("attend"))
    a, b = c.open(), c.open()
    x = torch.zeros(2, 10, 1, 128)
    p1 = c.plan([a, b], [10, 0])
    c.write(0, p1, x, x)
    c.write(1, p1, x, x)
    c.attend(0, p1, x)
    c.commit(p1)
    c.attend(1, p1, x)
    assert calls == ["write", "write", "attend", "attend"]
    with pytest.raises(RuntimeError, match="moved on"):
        c.write(1, p1, x, x)
    p2 = c.plan([a], 5)
    c.write(0, p2, x, x)
    with pytest.raises(RuntimeError, match="moved on"):
        c.write(0, p1, x, x)
    c.commit(p2)
    for call in (lambda: c.write(0, p1, x, x), lambda: c.attend(0, p1, x), lambda: c.commit(p1), lambda: c.commit(p2)):
        with pytest.raises(RuntimeError, match="moved on"):
            call()
    c.attend(0, p2, x)


def test_attend_wants_a_query_for_every_planned_token(monkeypatch):
    """Fewer rows would be taken for the sequence's last tokens, under a causal mask that is shifted."""
    pool = Tokens(monkeypatch, 12)
    c = pool.cache
    monkeypatch.setattr(paged_cache, "attend", lambda q, *a, **kw: q.shape[1])
    a, b = c.open(), c.open()
    plan = c.plan([a, b], [90, 3])
    for n in (0, 60, 89):
        with pytest.raises(ValueError, match="90 tokens"):
            c.attend(0, plan, torch.zeros(2, n, 1, 128), causal=True)
    assert c.attend(0, plan, torch.zeros(2, 90, 1, 128)) == 90 and c.attend(0, plan, torch.zeros(2, 128, 1, 128)) == 128


def test_write_refuses_rope_tables_that_end_before_the_tokens(monkeypatch):
    pool = Tokens(monkeypatch, 12)
    c = pool.cache
    written = []
    monkeypatch.setattr(paged_cache, "write", lambda *a, rope=None, **kw: written.append(rope))
    r = type("R", (), {})()
    r.cos = torch.zeros(100, 64)
    a, b = c.open(), c.open()
    c.commit(c.plan([a], 100))
    k = torch.zeros(2, 101, 1, 128)
    c.write(0, c.plan([a, b], [0, 100]), k, k, rope=r)                # a writes nothing
    for new in ([1, 5], [0, 101]):
        plan = c.plan([a, b], new)
        with pytest.raises(ValueError, match="100 positions"):
            c.write(0, plan, k, k, rope=r)
        c.write(0, plan, k, k, rope=r, positions=torch.zeros(2, 101, dtype=torch.int32))
        c.write(0, plan, k, k)
    assert written == [r, r, None, r, None]


def _addresses(t):
    """Element offsets of a tensor, counted from the start of its storage."""
    at = torch.tensor(t.storage_offset())
    for n, st in zip(t.shape, t.stride()):
        at = at[..., None] + torch.arange(n) * st
    return at.flatten().tolist()


@pytest.mark.parametrize("seed", range(4))
def test_overlaps_are_found_exactly(seed):
    """Random views of one buffer against their lists of addresses: overlaps inside a tensor, and between two."""
    r = random.Random(seed)
    buf = torch.zeros(4000, dtype=torch.bfloat16)
    found = [0, 0, 0, 0]
    for _ in range(1500):
        dim = r.choice([1, 2, 8])
        pair = []
        for _ in range(2):
            shape = [r.randint(1, 4) for _ in range(3)] + [dim]
            nest = [dim * r.randint(1, 3)]
            nest += [nest[0] * r.randint(1, 4) + r.choice([0, 0, 1])]
            nest += [nest[1] * r.randint(1, 4) + r.choice([0, 0, 3])]
            if pair and r.random() < 0.5:
                nest = list(pair[0].stride()[:3])
            r.shuffle(nest)
            pair.append(buf.as_strided(shape, nest + [1], r.randint(0, 400)))
        for t in pair:
            want = len(set(_addresses(t))) < t.numel()
            found[want] += 1
            assert _lib.self_overlap(t) == want, (t.shape, t.stride())
        want = not set(_addresses(pair[0])).isdisjoint(_addresses(pair[1]))
        found[2 + want] += 1
        assert _lib.share_memory(*pair) == want, [(t.shape, t.stride(), t.storage_offset()) for t in pair]
    assert min(found) > 100
    e = buf[:64].view(1, 1, 8, 8).expand(1, 5, 8, 8)
    assert _lib.self_overlap(e) and not _lib.self_overlap(e[:, :1]) and _lib.share_memory(e, e[:, 2:, 3:5])
    assert not _lib.share_memory(e[:, :0], e) and not _lib.self_overlap(e[:, :0])


def test_key_splits_follow_the_key_lengths(monkeypatch):
    """A plan knows whether its sessions' lengths are unlike, whatever their new tokens; one that takes later values may be."""
    pool = Tokens(monkeypatch, 30)
    c = pool.cache
    seen = []
    monkeypatch.setattr(paged_cache, "attend", lambda *a, ragged, **kw: seen.append(ragged))
    a, b, d = c.open(), c.open(), c.open()
    c.commit(c.plan([a, b, d], [400, 390, 20]))
    q = torch.zeros(2, 64, 1, 128)
    for sessions, new in (([a, b], 1), ([a, b], [1, 64]), ([a, d], 1), ([a, d], [1, 64]), ([d], 1), ([a, b, d], [0, 0, 63])):
        c.attend(0, c.plan(sessions, new), q)
    c.attend(0, c.plan([a, b], 1, into=c.fixed_plan(2)), q)
    assert seen == [False, False, True, True, False, False, True]
    assert 3 * (400 + 390 + 83) > 2 * 3 * 400


def test_closing_a_long_session_takes_no_time(monkeypatch):
    """40000 pages freed one by one, into a pool whose free pages stay in order (sorting them all at each took 4 s)."""
    import time
    pool = Tokens(monkeypatch, 2, layers=1)
    shape = (1, 40000, 1, 64, 128)
    codes = torch.empty(1, dtype=torch.int8).expand(shape)
    c = paged_cache.PagedCache(paged_cache.Pages(codes, codes, None, None), max_pages=40000)
    del pool
    a, b = c.open(), c.open()
    c.plan([a], 64 * 39990)
    c.plan([b], 64 * 10)
    t0 = time.perf_counter()
    c.close(a)
    assert time.perf_counter() - t0 < 2
    assert c.free_pages == 39990 and c.page_ids(b) == list(range(39990, 40000))
    s = c.open()
    c.plan([s], 64 * 5)
    assert c.page_ids(s) == list(range(5))                           # the lowest free ids


def test_only_clusters_that_fit_at_once_merge_in_one():
    """The merge without scratch is for CTAs that run at once as clusters: up to 256 of them, not up to two an SM (on 148 SMs 72
    tiles of 4 splits took 22.2 us so, 16.9 with a merge launch)."""
    ws = _lib.load().lbq_paged_attn_workspace
    for batch, heads, splits, fit in ((8, 8, 4, True), (4, 8, 8, True), (8, 10, 3, True), (8, 9, 4, False), (8, 12, 3, False),
                                      (4, 9, 8, False), (8, 6, 6, False), (5, 8, 7, False), (7, 8, 5, False), (1, 1, 9, False)):
        assert (ws(batch, 1, heads, 1, splits) == 0) == fit, (batch, heads, splits)
