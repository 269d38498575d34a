"""A KV cache that stays in 8 bits, in pages of 64 tokens (lbq_page_write, lbq_page_read, lbq_page_copy, lbq_paged_attn).

The reference's cache is one bf16 buffer a layer whose whole window is quantized again for every attention call
(lingbot/layers/kv_cache.py:11-88, lingbot/layers/sage_preq.py:107-128; here `kv_cache`). In this one a token is
quantized once, when it is written (int8 or e4m3 codes, one scale per page, head and tensor), attention reads the codes
as they are (unquantized queries, fp32 sums, softmax weights in fp16), and a page table names the pages of a session, so
that sessions share a prefix, fork, drop their oldest pages and are packed together without touching other sessions.

Two levels:
  functions over tensors   write, window, attend, copy_pages on a `Pages` pool, a page table and lengths;
  `PagedCache`             the host's bookkeeping over them for all layers, with the steps of `kv_cache`: `plan` the new
                           tokens of some sessions, `write` and `attend` layer by layer, `commit`; `fork`, `evict`,
                           `close` and `compact`.
"""
from __future__ import annotations

import heapq
from array import array
from dataclasses import dataclass

import torch

from . import _lib
from .ops import HEAD_DIM
from .rope import Rope

__all__ = ["PAGE", "Pages", "alloc_pages", "write", "window", "attend", "copy_pages", "Plan", "PagedCache", "allocate"]

PAGE = 64
FORMATS = {torch.int8: 0, torch.float8_e4m3fn: 1}
_ACT = {torch.bfloat16: 0, torch.float16: 1}


class Pages:
    """A pool of pages: k, v codes [pages, heads, 64, 128] (int8 or float8_e4m3fn) and k_amax, v_amax f32 [pages, heads],
    or the same with a leading dimension of layers. value = code * amax / 127 (int8) or / 448 (e4m3)."""

    def __init__(self, k, v, k_amax, v_amax):
        self.k, self.v, self.k_amax, self.v_amax = k, v, k_amax, v_amax
        r = _lib.fast().pool(k, v, k_amax, v_amax)
        if r is None:
            self._refuse()
        self._dev, self.heads, self._args, self._copy_args = r

    def _refuse(self):
        k, v, ka, va = self.k, self.v, self.k_amax, self.v_amax
        if k.dtype not in FORMATS or v.dtype != k.dtype or ka.dtype != torch.float32 or va.dtype != torch.float32:
            raise TypeError("pages: int8 or float8_e4m3fn codes and float32 amax, got "
                            f"{k.dtype}, {v.dtype}, {ka.dtype}, {va.dtype}")
        if k.dim() not in (4, 5) or tuple(k.shape[-2:]) != (PAGE, HEAD_DIM) or v.shape != k.shape \
                or ka.shape != k.shape[:-2] or va.shape != ka.shape:
            raise ValueError(f"pages: codes [(layers,) pages, heads, {PAGE}, {HEAD_DIM}] and amax [(layers,) pages, heads], "
                             f"got {tuple(k.shape)}, {tuple(v.shape)}, {tuple(ka.shape)}, {tuple(va.shape)}")
        if not k.is_cuda or any(t.device != k.device for t in (v, ka, va)):
            raise ValueError("pages must be CUDA tensors of one device")
        raise ValueError("pages must be contiguous")

    @property
    def device(self):
        return self.k.device

    def layer(self, i) -> "Pages":
        """The pool of one layer."""
        if self.k.dim() != 5:
            raise ValueError("the pool has no layers")
        return Pages(self.k[i], self.v[i], self.k_amax[i], self.v_amax[i])

    def args(self):
        """The pool's arguments of the C ABI."""
        if self._args is None:
            raise ValueError("the pool has layers: take .layer(i)")
        return self._args


def alloc_pages(num_pages, heads, device, fmt=torch.int8, layers=None) -> Pages:
    """A zeroed pool of `num_pages` pages (`layers` of them with a layer dimension)."""
    lead = (num_pages, heads) if layers is None else (layers, num_pages, heads)
    if fmt not in FORMATS:
        raise TypeError(f"page format {fmt}: expected torch.int8 or torch.float8_e4m3fn")
    codes = [torch.zeros(*lead, PAGE, HEAD_DIM, dtype=torch.int8, device=device).view(fmt) for _ in range(2)]
    amax = [torch.zeros(*lead, dtype=torch.float32, device=device) for _ in range(2)]
    return Pages(*codes, *amax)


def _table(t, batch, device):
    if t.dtype is not torch.int32 or t.dim() != 2 or t.device != device:
        raise ValueError(f"page table: an int32 [batch, pages] tensor on {device}, got {t.dtype} {tuple(t.shape)} on "
                         f"{t.device}")
    _lib.check_sizes("page table", t)
    n, width = t.shape
    row, unit = t.stride()
    if n != batch or width == 0 or (unit != 1 and width > 1):
        raise ValueError(f"page table: [{batch}, pages] with unit last stride, got {tuple(t.shape)}, strides {t.stride()}")
    return t.data_ptr(), row, width


def _counts(name, t, batch, device):
    """A count for each sequence: (pointer, 0) of an int32 [batch] tensor, (None, value) of an int."""
    if isinstance(t, torch.Tensor):
        if t.dtype is not torch.int32 or t.dim() != 1 or t.shape[0] != batch or t.device != device \
                or (batch > 1 and t.stride(0) != 1):
            raise ValueError(f"{name}: a contiguous int32 [{batch}] tensor on {device}, got {t.dtype} {tuple(t.shape)} on "
                             f"{t.device}")
        return t.data_ptr(), 0
    t = int(t)
    if t < 0:
        raise ValueError(f"{name} {t} is negative")
    if t >= 1 << 62:                                             # ctypes would drop the upper bits
        raise ValueError(f"{name} {t} does not fit 64 bits")
    return None, t


def _check_rows(name, x, device):
    if x.dtype not in _ACT:
        raise TypeError(f"{name} must be bfloat16 or float16, got {x.dtype}")
    if x.dim() != 4 or x.shape[3] != HEAD_DIM or x.stride(3) != 1:
        raise ValueError(f"{name} must be [B, L, heads, {HEAD_DIM}] with unit channel stride, got {tuple(x.shape)}")
    if x.device != device:
        raise ValueError(f"{name} on {x.device}, pages on {device}")
    _lib.check_sizes(name, x)


def _overlap(a, b):
    """Whether the address ranges of two tensors meet."""
    def span(t):
        last = sum((n - 1) * st for n, st in zip(t.shape, t.stride()))
        return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()
    if not a.numel() or not b.numel():
        return False
    (a0, a1), (b0, b1) = span(a), span(b)
    return a0 < b1 and b0 < a1


def write(pages: Pages, page_table, start, k, v, lens=None, rope: Rope = None, positions=None):
    """Quantizes new tokens k, v [B, L, heads, 128] (bf16 or fp16) into the pages of tokens start[b] .. start[b] +
    lens[b] (start, lens: int32 [B] tensors or ints; lens None: all L). A page that already holds tokens before `start`
    keeps them: when its largest magnitude grows their codes are rounded to the new scale. Tokens at and past `start`
    are replaced (a page that holds earlier ones keeps its scale, if a replaced token's was larger). With `rope`, K is
    rotated on the way, by `positions` [B, L] or its token indices, to the same bits as rope.apply followed by a plain write.
    Two sequences of one call must not write the same page."""
    if rope is None or rope._dev == pages._dev:
        r = _lib.fast().page_write(pages._args, pages._dev, page_table, start, k, v, lens, None if rope is None else rope._args,
                                   positions)
        if r is not None:
            _lib.check("lbq_page_write", r)
            return
    args, heads, dev = pages.args(), pages.heads, pages.device
    _check_rows("k", k, dev)
    _check_rows("v", v, dev)
    if v.shape != k.shape or v.dtype != k.dtype or k.shape[2] != heads:
        raise ValueError(f"k {k.dtype} {tuple(k.shape)} and v {v.dtype} {tuple(v.shape)} differ, or are not of the pages' "
                         f"{heads} heads")
    _lib.no_gradient("the paged cache", k, v)
    b, l = k.shape[:2]
    if b == 0 or l == 0:
        return
    table = _table(page_table, b, dev)
    sp, s0 = _counts("start", start, b, dev)
    lp = None
    if lens is not None:
        lp, n = _counts("lens", lens, b, dev)
        if lp is None:
            if n > l:
                raise ValueError(f"lens {n} of {l} tokens")
            if n == 0:
                return
            l = n
    if rope is None:
        if positions is not None:
            raise ValueError("positions without rope")
        turn = (None, None, 0, 0, 0, 0, None, 0, 0, 0)
    else:
        if positions is not None and positions.shape[-1] > l:
            positions = positions[..., :l]
        turn = rope.args(positions, dev, b, l)
    sk, sv = k.stride(), v.stride()
    _lib.call_on(dev, "lbq_page_write", k.data_ptr(), sk[0], sk[1], sk[2], v.data_ptr(), sv[0], sv[1], sv[2], *args, *table,
                 sp, s0, lp, b, l, *turn, _ACT[k.dtype])


def window(pages: Pages, page_table, start, length, dtype=torch.bfloat16, lens=None, out=None):
    """Values (k, v) [B, length, heads, 128] in `dtype` of the tokens from start[b] on; rows past lens[b] (None: all) are
    0. The role of kv_cache.window, as a copy."""
    if out is None and dtype in _ACT:
        r = _lib.fast().page_read(pages._args, pages._dev, page_table, start, length, _ACT[dtype], lens)
        if r is not None:
            if type(r) is int:
                _lib.check("lbq_page_read", r)
            return r
    args, heads, dev = pages.args(), pages.heads, pages.device
    b, length = page_table.shape[0], int(length)
    if dtype not in _ACT:
        raise TypeError(f"window dtype {dtype}: expected bfloat16 or float16")
    if length < 0:
        raise ValueError(f"length {length} is negative")
    if length > 1 << 28:
        raise ValueError(f"length {length} is more than 2^28")
    _lib.check_sizes("page table", page_table)
    if out is None:
        k = torch.empty((b, length, heads, HEAD_DIM), dtype=dtype, device=dev)
        v = torch.empty_like(k)
    else:
        k, v = out
        for name, t in (("k out", k), ("v out", v)):
            _check_rows(name, t, dev)
            if tuple(t.shape[:3]) != (b, length, heads) or t.dtype != dtype:
                raise ValueError(f"{name} must be {dtype} [{b}, {length}, {heads}, {HEAD_DIM}], got {t.dtype} "
                                 f"{tuple(t.shape)}")
            if _lib.self_overlap(t):
                raise ValueError(f"{name} has elements that share memory")
        if _lib.share_memory(k, v):
            raise ValueError("k out and v out share memory")
    if b == 0 or length == 0:
        return k, v
    table = _table(page_table, b, dev)
    sp, s0 = _counts("start", start, b, dev)
    lp = None
    if lens is not None:
        if not isinstance(lens, torch.Tensor):
            lens = torch.full((b,), int(lens), dtype=torch.int32, device=dev)
        lp, _ = _counts("lens", lens, b, dev)
    sk, sv = k.stride(), v.stride()
    _lib.call_on(dev, "lbq_page_read", *args, *table, sp, s0, lp, b, length, k.data_ptr(), sk[0], sk[1], sk[2], v.data_ptr(),
                 sv[0], sv[1], sv[2], _ACT[dtype])
    return k, v


def attend(q, pages: Pages, page_table, kv_lens, q_lens=None, causal=False, sm_scale=None, out=None, return_lse=False,
           max_kv_len=None, num_splits=None, ragged=None):
    """Attention of q [B, Lq, heads, 128] (bf16 or fp16; a multiple of the pages' heads, query head h reading K/V head
    h // group) over the cached tokens j < kv_lens[b] (int32 [B] tensor or int) and, with causal, j <= kv_lens[b] -
    q_lens[b] + i: query i is token kv_lens[b] - q_lens[b] + i of its sequence, already written. q_lens (int32 [B]) marks
    a padded batch. sm_scale None (or not above 0) is 128 ** -0.5. Rows that see no token, and rows past q_lens[b], are 0.
    Returns out [B, Lq, heads, 128] in q's dtype, with return_lse also the rows' log-sum-exp f32 [B, Lq, heads] (-inf for
    those rows). max_kv_len bounds kv_lens where the page table is much wider than the longest sequence. ragged says whether
    the sequences' key lengths are unlike, their mean under about two thirds of the longest (None: yes for a kv_lens tensor,
    whose values the host does not read, no for an int); it only chooses the number of key splits, which num_splits
    overrides."""
    if out is None and not return_lse and max_kv_len is None and num_splits is None:
        r = _lib.fast().paged_attn(pages._args, pages._dev, q, page_table, kv_lens, q_lens, causal, float(sm_scale or 0.0),
                                   ragged)
        if r is not None:
            if type(r) is int:
                _lib.check("lbq_paged_attn", r)
            return r
    args, heads, dev = pages.args(), pages.heads, pages.device
    _check_rows("q", q, dev)
    b, lq, hq, _ = q.shape
    group = hq // heads
    if group * heads != hq or hq == 0:
        raise ValueError(f"q has {hq} heads, not a multiple of the pages' {heads}")
    _lib.no_gradient("the paged cache", q)
    if out is None:
        out = torch.empty_like(q)
    else:
        _check_rows("out", out, dev)
        if out.shape != q.shape or out.dtype != q.dtype:
            raise ValueError(f"out must be {q.dtype} {tuple(q.shape)}, got {out.dtype} {tuple(out.shape)}")
        if _lib.self_overlap(out):
            raise ValueError("out has elements that share memory")
        if (out.data_ptr() != q.data_ptr() or out.stride() != q.stride()) and _overlap(out, q):
            raise ValueError("out overlaps q without being it")
    lse = torch.empty((b, lq, hq), dtype=torch.float32, device=dev) if return_lse else None
    if b and lq:
        tp, ts, width = _table(page_table, b, dev)
        kp, k0 = _counts("kv_lens", kv_lens, b, dev)
        qp = None
        if q_lens is not None:
            qp, _ = _counts("q_lens", q_lens, b, dev)
            if qp is None:
                raise TypeError("q_lens must be an int32 tensor")
        longest = width * PAGE if kp is not None else k0
        if max_kv_len is not None:
            longest = min(longest, max(0, int(max_kv_len)))
            if kp is not None:
                width = max(1, min(width, (longest + PAGE - 1) // PAGE))
            elif k0 > longest:
                raise ValueError(f"kv_lens {k0} exceeds max_kv_len {longest}")
        lib = _lib.load()
        if num_splits is None:
            unlike = kp is not None if ragged is None else ragged
            num_splits = lib.lbq_paged_attn_splits(b, lq, heads, group, longest, int(b > 1 and bool(unlike)))
        ws, ws_bytes = None, 0
        if num_splits > 1:
            ws_bytes = lib.lbq_paged_attn_workspace(b, lq, heads, group, num_splits)
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev)
        sq, so = q.stride(), out.stride()
        _lib.call_on(dev, "lbq_paged_attn", q.data_ptr(), sq[0], sq[1], sq[2], *args, tp, ts, width, kp, k0, qp, b, lq, group,
                     1 if causal else 0, float(sm_scale or 0.0), out.data_ptr(), so[0], so[1], so[2],
                     None if lse is None else lse.data_ptr(), num_splits, None if ws is None else ws.data_ptr(), ws_bytes,
                     _ACT[q.dtype])
    return (out, lse) if return_lse else out


def copy_pages(pages: Pages, src, dst):
    """Copies page src[i] to dst[i] (host sequences of ints) in every layer of the pool. All pages named by dst are
    different and none of them is a source."""
    r = _lib.fast().page_copy(pages._copy_args, pages._dev, src, dst) if pages is not None else None
    if r is not None:
        _lib.check("lbq_page_copy", r)
        return
    src, dst = array("i", src), array("i", dst)
    if len(src) != len(dst):
        raise ValueError(f"{len(src)} source pages, {len(dst)} destinations")
    if not src:
        return
    to = set(dst)
    if len(to) != len(dst):
        raise ValueError("a page is written twice")
    if not to.isdisjoint(src):
        raise ValueError("a page is both read and written")
    _lib.call_on(pages.device, "lbq_page_copy", *pages._copy_args, src.buffer_info()[0], dst.buffer_info()[0], len(src))


@dataclass
class Plan:
    """One step of some sessions: what `write` and `attend` of every layer take. Made by PagedCache.plan."""
    sessions: list
    new: list                     # new tokens of each session
    held: list                    # tokens each held before
    table: torch.Tensor           # int32 [B, pages]
    start: torch.Tensor           # int32 [B]: held
    lens: torch.Tensor            # int32 [B]: new
    kv_lens: torch.Tensor         # int32 [B]: held + new
    versions: list                # of the sessions' page lists
    ragged: bool = True           # key lengths are unlike (of a plan whose tensors take later values: they may be)


class PagedCache:
    """Page bookkeeping of many sessions over one pool with layers. The host knows every length and page; the tensors of
    a `Plan` carry them to the kernels. Not thread-safe; a session is in one plan at a time, which ends when the session's
    tokens or pages change. Pages that close, evict, plan or compact free are handed out at once: calls of one cache belong on
    one stream, or behind one another by events, so that what still reads a page comes before what writes it next."""

    def __init__(self, pages: Pages, max_pages):
        if pages.k.dim() != 5:
            raise ValueError("PagedCache takes a pool with layers")
        self.pages = pages
        self.layers = [pages.layer(i) for i in range(pages.k.shape[0])]
        self.num_pages = pages.k.shape[1]
        self.max_pages = int(max_pages)
        self._free = list(range(self.num_pages))                  # a heap: the lowest ids are taken first
        self._refs = [0] * self.num_pages
        self._sessions = {}                                       # id -> [pages, tokens, version, evicted tokens]
        self._next = 0
        self._version = 0

    @property
    def free_pages(self):
        return len(self._free)

    def tokens(self, session):
        return self._get(session)[1]

    def page_ids(self, session):
        return list(self._get(session)[0])

    def _get(self, session):
        try:
            return self._sessions[session]
        except KeyError:
            raise KeyError(f"no open session {session}") from None

    def _touch(self, session):
        """Earlier plans of the session no longer hold."""
        self._version += 1
        self._sessions[session][2] = self._version

    def _take(self):
        page = heapq.heappop(self._free)
        self._refs[page] = 1
        return page

    def _drop(self, page):
        self._refs[page] -= 1
        if self._refs[page] == 0:
            heapq.heappush(self._free, page)

    def open(self):
        """A new, empty session."""
        return self._add([], 0)

    def _add(self, pages, tokens, evicted=0):
        self._version += 1
        self._sessions[self._next] = [pages, tokens, self._version, evicted]
        self._next += 1
        return self._next - 1

    def fork(self, session):
        """A new session with the same committed tokens. Their pages are shared; an unfinished last page is copied when
        one of the sessions is next planned to write into it. Plans of `session` made before end."""
        pages, tokens, _, evicted = self._get(session)
        pages = pages[:(tokens + PAGE - 1) // PAGE]
        for p in pages:
            self._refs[p] += 1
        self._touch(session)
        return self._add(pages, tokens, evicted)

    def close(self, session):
        """Ends a session and frees the pages that no other session holds."""
        pages = self._get(session)[0]
        del self._sessions[session]
        for p in pages:
            self._drop(p)

    def plan(self, sessions, new_tokens, into: Plan = None) -> Plan:
        """Pages for `new_tokens` (an int, or one per session) more tokens of each session. Shared unfinished pages are
        copied first. Raises without a change when the pool or max_pages does not suffice. `into`: an earlier plan of as
        many sessions whose tensors (fixed in a captured graph) take the new values; its table keeps max_pages columns."""
        sessions = list(sessions)
        new = [int(new_tokens)] * len(sessions) if isinstance(new_tokens, int) else [int(n) for n in new_tokens]
        if len(new) != len(sessions) or not sessions:
            raise ValueError(f"{len(new)} token counts for {len(sessions)} sessions")
        if len(set(sessions)) != len(sessions):
            raise ValueError("a session is planned twice")
        if min(new) < 0:
            raise ValueError("negative token count")
        if into is not None and tuple(into.table.shape) != (len(sessions), self.max_pages):
            raise ValueError(f"a plan whose table is {tuple(into.table.shape)} cannot take {len(sessions)} sessions of "
                             f"{self.max_pages} pages: make it with fixed_plan")
        need, refs, copies = 0, {}, []
        for s, n in zip(sessions, new):
            pages, tokens = self._get(s)[:2]
            total = (tokens + n + PAGE - 1) // PAGE
            if total > self.max_pages:
                raise ValueError(f"session {s}: {tokens + n} tokens exceed {self.max_pages} pages")
            need += max(0, total - len(pages))       # pages left from a larger plan that was not committed are no one else's
            if n and tokens % PAGE:
                last = pages[tokens // PAGE]
                left = refs.get(last, self._refs[last])
                if left > 1:
                    refs[last] = left - 1
                    need += 1
                    copies.append((s, tokens // PAGE))
        if need > len(self._free):
            raise RuntimeError(f"{need} pages needed, {len(self._free)} of {self.num_pages} free")
        if copies:
            src, dst = [self._sessions[s][0][at] for s, at in copies], [self._take() for _ in copies]
            try:
                copy_pages(self.pages, src, dst)
            except BaseException:
                for p in dst:
                    self._drop(p)
                raise
            for (s, at), old, new_page in zip(copies, src, dst):
                self._sessions[s][0][at] = new_page
                self._refs[old] -= 1
                self._touch(s)
        for s, n in zip(sessions, new):
            pages, tokens = self._sessions[s][:2]
            while len(pages) * PAGE < tokens + n:
                pages.append(self._take())
        held = [self._sessions[s][1] for s in sessions]
        rows = [self._sessions[s][0] for s in sessions]
        width = self.max_pages if into is not None else max(1, max(len(r) for r in rows))
        versions = [self._sessions[s][2] for s in sessions]
        dev = self.pages.k.device
        table = torch.tensor([r + [-1] * (width - len(r)) for r in rows], dtype=torch.int32)
        counts = torch.tensor([held, new, [h + n for h, n in zip(held, new)]], dtype=torch.int32)
        if into is None:
            table, counts = table.to(dev), counts.to(dev)
            total = [h + n for h, n in zip(held, new)]
            # few-row attention of 16 to 64 sessions, alike splits / unlike: lengths of mean 0.55 of the longest 70.6 / 61.3,
            # 113 / 98 and 67.8 / 49.5 us, of mean 0.68 73.2 / 73.7, of mean 0.77 76.5 / 76.9, 139 / 137 and 69.4 / 80.4, all
            # alike 83.9 / 99.9, 161 / 172 and 77.6 / 84.4
            return Plan(sessions, new, held, table, counts[0], counts[1], counts[2], versions,
                        ragged=3 * sum(total) < 2 * len(total) * max(total))
        into.table.copy_(table)
        for t, c in zip((into.start, into.lens, into.kv_lens), counts):
            t.copy_(c)
        into.sessions, into.new, into.held, into.versions, into.ragged = sessions, new, held, versions, True
        return into

    def fixed_plan(self, batch) -> Plan:
        """An empty plan of `batch` sessions with a table of max_pages columns, for plan(..., into=) under captured
        graphs."""
        dev = self.pages.k.device
        z = torch.zeros(3, batch, dtype=torch.int32, device=dev)
        return Plan([None] * batch, [0] * batch, [0] * batch,
                    torch.full((batch, self.max_pages), -1, dtype=torch.int32, device=dev), z[0], z[1], z[2], [-1] * batch)

    def _check(self, plan, committed=False):
        """The plan still holds: its sessions' pages are those of the plan, and their tokens too (with `committed`, also with
        the plan's own behind them)."""
        for s, v, n, h in zip(plan.sessions, plan.versions, plan.new, plan.held):
            entry = self._sessions.get(s)
            if entry is None or entry[2] != v:
                raise RuntimeError(f"session {s} was closed, forked, copied, evicted from or compacted since the plan was "
                                   "made: plan again")
            if entry[1] != h and not (committed and entry[1] == h + n):
                raise RuntimeError(f"session {s} moved on since the plan was made")

    def write(self, layer, plan: Plan, k, v, rope: Rope = None, positions=None):
        """Writes the plan's new tokens k, v [B, L, heads, 128] of one layer (L at least the longest session's new
        tokens). Writing a plan again replaces them (the passes of one chunk), until it is committed."""
        self._check(plan)
        if k.dim() == 4 and k.shape[1] < max(plan.new):
            raise ValueError(f"{k.shape[1]} tokens given, {max(plan.new)} planned")
        if rope is not None and positions is None and any(self._sessions[s][3] for s in plan.sessions):
            raise ValueError("tokens were evicted from a session of this plan: pass the new tokens' positions")
        if rope is not None and positions is None:
            last = max((h + n for h, n in zip(plan.held, plan.new) if n), default=0)
            if last > rope.cos.shape[0]:                             # their K would be stored as it is
                raise ValueError(f"tokens up to {last} planned, rope tables of {rope.cos.shape[0]} positions")
        write(self.layers[layer], plan.table, plan.start, k, v, lens=plan.lens, rope=rope, positions=positions)

    def attend(self, layer, plan: Plan, q, causal=False, sm_scale=None, out=None, return_lse=False):
        """Attention of the plan's new tokens q [B, L, heads, 128] (L at least the longest session's new tokens) over
        everything their sessions hold."""
        self._check(plan, committed=True)
        if q.dim() == 4 and q.shape[1] < max(plan.new):              # the rows there are would count as the last tokens
            raise ValueError(f"{q.shape[1]} queries given, {max(plan.new)} tokens planned")
        return attend(q, self.layers[layer], plan.table, plan.kv_lens, q_lens=plan.lens, causal=causal, sm_scale=sm_scale,
                      out=out, return_lse=return_lse, ragged=plan.ragged)

    def commit(self, plan: Plan):
        """The plan's new tokens belong to their sessions from now on."""
        self._check(plan)
        for s, n in zip(plan.sessions, plan.new):
            self._sessions[s][1] += n

    def evict(self, session, sink_tokens, evicted):
        """Drops `evicted` tokens after the first `sink_tokens` (both multiples of 64): their pages leave the session's
        table, nothing is copied. The tokens that stay keep their K as it was roped; `write` with rope then wants
        positions, since a token's index in the session is no longer its position."""
        if sink_tokens % PAGE or evicted % PAGE or sink_tokens < 0 or evicted < 0:
            raise ValueError(f"sink {sink_tokens} and evicted {evicted} must be non-negative multiples of {PAGE}")
        pages, tokens = self._get(session)[:2]
        if sink_tokens + evicted > tokens:
            raise ValueError(f"session {session} holds {tokens} tokens, fewer than {sink_tokens} + {evicted}")
        a, b = sink_tokens // PAGE, (sink_tokens + evicted) // PAGE
        gone = pages[a:b]
        self._sessions[session][:2] = pages[:a] + pages[b:], tokens - evicted
        self._sessions[session][3] += evicted
        self._touch(session)
        for p in gone:
            self._drop(p)

    def compact(self):
        """Moves live pages to the lowest ids, so that the pool's tail is free. Returns how many pages moved."""
        live = self.num_pages - len(self._free)
        src = [p for p in range(live, self.num_pages) if self._refs[p]]
        dst = [p for p in range(live) if not self._refs[p]]
        if not src:
            return 0
        copy_pages(self.pages, src, dst)
        to = dict(zip(src, dst))
        for s, entry in self._sessions.items():
            if not to.keys().isdisjoint(entry[0]):
                entry[0] = [to.get(p, p) for p in entry[0]]
                self._touch(s)
        for s, d in to.items():
            self._refs[d], self._refs[s] = self._refs[s], 0
        self._free = list(range(live, self.num_pages))
        return len(src)


def allocate(num_layers, num_pages, heads, max_pages, device, fmt=torch.int8) -> PagedCache:
    """A cache of `num_layers` pools of `num_pages` pages; a session holds at most `max_pages` of them."""
    return PagedCache(alloc_pages(num_pages, heads, device, fmt, layers=num_layers), max_pages)
