"""Cases, plain forms and 64-bit values of the paged 8-bit KV cache's operators: attention over its pages, the quantizing
write, the read-back of a window, page copies, and rotary positions.

Cache layout: a page holds 64 tokens of every K/V head. Codes [pages][heads][64][128] are int8 or float8_e4m3fn, and
amax [pages][heads] (fp32) is the largest magnitude a page and head hold: value = code * amax / Q with Q = 127 (int8)
or 448 (e4m3). Token t of sequence b is row t % 64 of page table[b][t // 64].
"""
import os
import random
import sys

import torch

own = False

PAGE = 64
DIM = 128
FLOOR = 2.0 ** -40          # smallest amax of a written page
DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
FORMATS = {"int8": (torch.int8, 127.0), "e4m3": (torch.float8_e4m3fn, 448.0)}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # Q and K of one video chunk (4 frames of 1508 tokens, 12 heads), every channel rotated, neighbouring pairs
        {"name": "rope_chunk", "op": "rope", "batch": 1, "len": 6032, "q_heads": 12, "k_heads": 12, "rot": 128,
         "interleaved": True, "dtype": "bf16", "positions": 32768},
        # one generated token of each of 64 sessions, half the head rotated, half layout, far positions
        {"name": "rope_decode", "op": "rope", "batch": 64, "len": 1, "q_heads": 16, "k_heads": 4, "rot": 64,
         "interleaved": False, "dtype": "fp16", "positions": 131072},
        # the chunk's K (roped on the way) and V written behind a memory of 24128 tokens, and read back
        {"name": "write_chunk", "op": "write", "batch": 1, "len": 6032, "heads": 12, "start": 24128, "format": "int8",
         "dtype": "bf16", "rot": 128},
        # one token of each of 64 sessions appended inside a page, whose scale may grow; the page read back
        {"name": "write_decode", "op": "write", "batch": 64, "len": 1, "heads": 8, "start": 2000, "format": "e4m3",
         "dtype": "bf16", "rot": 0},
        # a fork's unfinished last page and its neighbour, in all 30 layers
        {"name": "copy_fork", "op": "copy", "layers": 30, "heads": 12, "pages": 64, "moved": 2, "format": "int8"},
        # compaction of half a session's window (236 of 472 pages), in all 30 layers
        {"name": "copy_compact", "op": "copy", "layers": 30, "heads": 12, "pages": 472, "moved": 236, "format": "e4m3"},
        # one token against a short window: latency
        {"name": "decode_short", "op": "attend", "batch": 1, "q_len": 1, "kv_len": 1000, "kv_heads": 12, "group": 1,
         "causal": True, "ragged": False, "format": "int8", "dtype": "bf16"},
        # one token against the full video window
        {"name": "decode_window", "op": "attend", "batch": 1, "q_len": 1, "kv_len": 30160, "kv_heads": 12, "group": 1,
         "causal": True, "ragged": False, "format": "int8", "dtype": "bf16"},
        # one token of each of 32 sessions of unlike lengths, four query heads to a K/V head
        {"name": "decode_batch", "op": "attend", "batch": 32, "q_len": 1, "kv_len": 8192, "kv_heads": 8, "group": 4,
         "causal": True, "ragged": True, "format": "e4m3", "dtype": "bf16"},
        # five drafted tokens of each of 8 sessions checked at once
        {"name": "draft_check", "op": "attend", "batch": 8, "q_len": 5, "kv_len": 4100, "kv_heads": 4, "group": 8,
         "causal": True, "ragged": True, "format": "int8", "dtype": "fp16"},
        # prompts of unlike lengths behind cached prefixes, causal
        {"name": "prefill_ragged", "op": "attend", "batch": 4, "q_len": 1021, "kv_len": 8192, "kv_heads": 4, "group": 4,
         "causal": True, "ragged": True, "format": "e4m3", "dtype": "bf16"},
        # the video chunk against the full window
        {"name": "chunk_window", "op": "attend", "batch": 1, "q_len": 6032, "kv_len": 30160, "kv_heads": 12, "group": 1,
         "causal": False, "ragged": False, "format": "int8", "dtype": "bf16"},
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["rope", "write", "copy", "attend", "attend", "attend"])
    fmt = rng.choice(["int8", "e4m3"])
    dtype = rng.choice(["bf16", "fp16"])
    if op == "rope":
        tokens = _log(rng, 1, 8192)
        batch = min(tokens, _log(rng, 1, 64))
        k_heads = rng.choice([1, 2, 4, 8, 12])
        return {"op": op, "batch": batch, "len": max(1, tokens // batch), "q_heads": k_heads * rng.choice([1, 2, 4]),
                "k_heads": k_heads, "rot": rng.choice([32, 64, 96, 128]), "interleaved": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "positions": _log(rng, 10000, 200000)}
    if op == "write":
        length = rng.choice([1, _log(rng, 2, 64), _log(rng, 65, 6000)])
        return {"op": op, "batch": _log(rng, 1, 64) if length < 65 else rng.randint(1, 4), "len": length,
                "heads": rng.randint(1, 12), "start": rng.choice([0, _log(rng, 1, 8000)]), "format": fmt, "dtype": dtype,
                "rot": rng.choice([0, 64, 128])}
    if op == "copy":
        pages = _log(rng, 8, 472)
        return {"op": op, "layers": rng.randint(1, 30), "heads": rng.randint(1, 12), "pages": pages,
                "moved": _log(rng, 1, pages // 2), "format": fmt}
    kind = rng.choice(["token", "few", "many"])
    kv_heads, group = rng.choice([(1, 8), (2, 4), (4, 4), (8, 4), (8, 1), (12, 1), (3, 5), (16, 1)])
    case = {"op": op, "batch": 1, "q_len": 1, "kv_len": _log(rng, 1, 32768), "kv_heads": kv_heads, "group": group,
            "causal": rng.random() < 0.6, "ragged": rng.random() < 0.6, "format": fmt, "dtype": dtype}
    if kind == "token":
        case["batch"] = _log(rng, 1, 64)
        case["kv_len"] = min(case["kv_len"], 4_000_000 // (case["batch"] * kv_heads))
    elif kind == "few":
        case["batch"] = _log(rng, 1, 16)
        case["q_len"] = rng.randint(2, 32)
        case["kv_len"] = min(case["kv_len"], 2_000_000 // (case["batch"] * kv_heads))
    else:
        case["batch"] = rng.randint(1, 4)
        case["q_len"] = _log(rng, 33, 4096)
        # at most the work of the largest listed case
        most = 6032 * 30160 * 12 // (case["batch"] * case["q_len"] * kv_heads * group)
        case["kv_len"] = max(1, min(case["kv_len"], most))
    return case


def _lengths(case):
    """(kv lengths, query lengths) of the sequences; the same for every seed. A ragged batch holds a full-length
    sequence, and where it has room an empty one and one with fewer keys than queries."""
    batch, kv, q = case["batch"], case["kv_len"], case["q_len"]
    if not case["ragged"]:
        return [kv] * batch, [q] * batch
    r = random.Random(1000 * kv + 10 * q + batch)
    kvs = [kv] + [r.randint(1, kv) for _ in range(batch - 1)]
    qs = [q] + [r.randint(1, q) for _ in range(batch - 1)]
    if batch > 4:
        kvs[2] = 0
        kvs[3] = min(kv, max(1, q // 2))
    return kvs, qs


def _starts(case):
    """Tokens each sequence holds before a write, and the new tokens of each; the same for every seed."""
    r = random.Random(100 * case["start"] + case["batch"])
    starts = [case["start"]] + [r.randint(0, case["start"]) for _ in range(case["batch"] - 1)]
    new = [case["len"]] + [r.randint(1, case["len"]) for _ in range(case["batch"] - 1)]
    return starts, new


def _visible(case):
    """(row, key) pairs that a K/V head's queries see."""
    pairs = 0
    for kv, q in zip(*_lengths(case)):
        if case["causal"]:
            first = kv - q + 1                      # keys that the first query sees (negative: none)
            last = min(q, max(0, 1 - first))        # leading queries that see nothing
            n = q - last
            pairs += n * (first + last) + n * (n - 1) // 2
        else:
            pairs += q * kv
    return pairs * case["group"]


def work(case):
    op = case["op"]
    if op == "rope":
        tokens, size = case["batch"] * case["len"], DTYPES[case["dtype"]].itemsize
        heads = case["q_heads"] + case["k_heads"]
        return {"bytes": tokens * (heads * DIM * size * 2 + case["rot"] * 4 + 8), "flops": tokens * heads * case["rot"] * 3}
    if op == "write":
        starts, new = _starts(case)
        tokens = sum(new)
        back = sum(n + s % PAGE for s, n in zip(starts, new))
        row = case["heads"] * DIM * 2                # values of K and V of a token
        # new values read, their codes written; codes of the touched pages read back, their values written
        return {"bytes": tokens * row * 3 + back * row * 3, "flops": (tokens + back) * row * 2}
    if op == "copy":
        return {"bytes": 2 * case["layers"] * case["moved"] * case["heads"] * (2 * PAGE * DIM + 8), "flops": 0}
    kvs, qs = _lengths(case)
    keys = sum(kvs) * case["kv_heads"]
    rows = sum(qs) * case["kv_heads"] * case["group"]
    return {"bytes": keys * (2 * DIM) + (keys // PAGE) * 8 + rows * DIM * 4,
            "flops": 4 * DIM * _visible(case) * case["kv_heads"]}


# ---------------------------------------------------------------------------------------------------- inputs
def _angles(positions, rot, device):
    """Angles [positions][rot / 2] in 64 bits of a rotary stretched for long contexts: frequencies 10000^(-2i/rot),
    slowed 4 times where a full turn takes over 8192 positions, unchanged where it takes under 2048, blended between."""
    freq = 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    turn = 2 * torch.pi / freq
    keep = ((8192 / turn - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
    freq = freq / 4 * (1 - keep) + freq * keep
    return torch.arange(positions, dtype=torch.float64, device=device)[:, None] * freq[None, :]


def _codes(values, fmt):
    """values [..., 64, 128] of pages -> (codes, amax [...])."""
    dt, q = FORMATS[fmt]
    amax = values.abs().amax(dim=(-1, -2)).clamp_min(FLOOR)
    x = values * (q / amax[..., None, None])
    return (x.round().to(dt) if fmt == "int8" else x.clamp(-q, q).to(dt)), amax


def _pages(gen, pages, heads, fmt, dev):
    """Pages of K-like or V-like values: N(0, 1) with an offset a channel, magnitudes that differ from page to page."""
    v = torch.randn(pages, heads, PAGE, DIM, generator=gen, device=dev)
    v = v + torch.randn(1, heads, 1, DIM, generator=gen, device=dev)
    v = v * (0.5 + torch.rand(pages, heads, 1, 1, generator=gen, device=dev))
    return _codes(v.bfloat16().float(), fmt)


def _table(gen, counts, width, pages, dev):
    """A page table with `counts` pages a sequence, scattered over the pool; -1 where a sequence has no page."""
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=dev)
    ids = torch.randperm(pages, generator=gen, device=dev).int()
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = ids[at:at + n]
        at += n
    return table


def prepare(case, seed):
    dev = torch.device(DEVICE)
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    op = case["op"]
    if op == "rope":
        dt = DTYPES[case["dtype"]]
        shape = (case["batch"], case["len"])
        ang = _angles(case["positions"], case["rot"], dev)
        return {"case": case, "q": torch.randn(*shape, case["q_heads"], DIM, generator=gen, device=dev).to(dt),
                "k": torch.randn(*shape, case["k_heads"], DIM, generator=gen, device=dev).to(dt),
                "cos": ang.cos().float(), "sin": ang.sin().float(),
                "at": torch.randint(0, case["positions"], shape, generator=gen, device=dev, dtype=torch.int32)}
    if op == "write":
        dt = DTYPES[case["dtype"]]
        starts, new = _starts(case)
        counts = [(s + n + PAGE - 1) // PAGE for s, n in zip(starts, new)]
        total = sum(counts) + 3
        kc, ka = _pages(gen, total, case["heads"], case["format"], dev)
        vc, va = _pages(gen, total, case["heads"], case["format"], dev)
        shape = (case["batch"], case["len"], case["heads"], DIM)
        st = {"case": case, "k_pages": kc, "v_pages": vc, "k_amax": ka, "v_amax": va,
              "table": _table(gen, counts, max(counts), total, dev),
              "start": torch.tensor(starts, dtype=torch.int32, device=dev),
              "new": torch.tensor(new, dtype=torch.int32, device=dev),
              "first": torch.tensor([s // PAGE * PAGE for s in starts], dtype=torch.int32, device=dev),
              "back": torch.tensor([s % PAGE + n for s, n in zip(starts, new)], dtype=torch.int32, device=dev),
              "longest": max(s % PAGE + n for s, n in zip(starts, new)),
              "k": (2 * torch.randn(*shape, generator=gen, device=dev)).to(dt),
              "v": (2 * torch.randn(*shape, generator=gen, device=dev)).to(dt)}
        if case["rot"]:
            ang = _angles(max(s + n for s, n in zip(starts, new)), case["rot"], dev)
            st["cos"], st["sin"] = ang.cos().float(), ang.sin().float()
        return st
    if op == "copy":
        n, m = case["pages"], case["moved"]
        shape = (case["layers"], n, case["heads"], PAGE, DIM)
        dt = FORMATS[case["format"]][0]
        lim = 127 if case["format"] == "int8" else 126       # e4m3 codes 0..126 are its finite values from 0 up
        low = -lim if case["format"] == "int8" else 0
        ids = torch.randperm(n, generator=gen, device=dev).tolist()
        return {"case": case, "src": ids[:m], "dst": ids[m:2 * m],
                "k_pages": torch.randint(low, lim + 1, shape, generator=gen, device=dev, dtype=torch.int8).view(dt),
                "v_pages": torch.randint(low, lim + 1, shape, generator=gen, device=dev, dtype=torch.int8).view(dt),
                "k_amax": torch.rand(shape[:3], generator=gen, device=dev) + 0.5,
                "v_amax": torch.rand(shape[:3], generator=gen, device=dev) + 0.5}
    kvs, qs = _lengths(case)
    counts = [(n + PAGE - 1) // PAGE for n in kvs]
    total = sum(counts) + 2
    kc, ka = _pages(gen, total, case["kv_heads"], case["format"], dev)
    vc, va = _pages(gen, total, case["kv_heads"], case["format"], dev)
    q = torch.randn(case["batch"], case["q_len"], case["kv_heads"] * case["group"], DIM, generator=gen, device=dev)
    return {"case": case, "q": q.to(DTYPES[case["dtype"]]), "k_pages": kc, "v_pages": vc, "k_amax": ka, "v_amax": va,
            "table": _table(gen, counts, max(counts), total, dev),
            "kv_lens": torch.tensor(kvs, dtype=torch.int32, device=dev),
            "q_lens": torch.tensor(qs, dtype=torch.int32, device=dev) if case["ragged"] else None}


# ---------------------------------------------------------------------------------------------------- passes
def run(state):
    op = state["case"]["op"]
    if own:
        return {"rope": _own_rope, "write": _own_write, "copy": _own_copy, "attend": _own_attend}[op](state)
    return {"rope": _rope, "write": _write, "copy": _copy, "attend": _attend}[op](state)


_modules = []


def _package():
    if not _modules:
        at = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        sys.path.insert(0, os.path.join(at, "lingbot-world-v2-realtime_b200"))
        from lingbot_b200 import paged_cache, rope
        _modules.extend([paged_cache, rope])
    return _modules


def _own_rope(s):
    _, rope = _package()
    table = rope.Rope(s["cos"], s["sin"], interleaved=s["case"]["interleaved"])
    return rope.apply(s["q"], table, s["at"], k=s["k"])


def _own_pages(s):
    return _package()[0].Pages(s["k_pages"], s["v_pages"], s["k_amax"], s["v_amax"])


def _own_write(s):
    paged_cache, rope = _package()
    pages = _own_pages(s)
    table = rope.Rope(s["cos"], s["sin"], interleaved=True) if s["case"]["rot"] else None
    paged_cache.write(pages, s["table"], s["start"], s["k"], s["v"], lens=s["new"], rope=table)
    k, v = paged_cache.window(pages, s["table"], s["first"], s["longest"], s["k"].dtype, lens=s["back"])
    return {"k": k, "v": v}


def _own_copy(s):
    _package()[0].copy_pages(_own_pages(s), s["src"], s["dst"])
    return {"k": s["k_pages"], "v": s["v_pages"], "k_amax": s["k_amax"], "v_amax": s["v_amax"]}


def _own_attend(s):
    return _package()[0].attend(s["q"], _own_pages(s), s["table"], s["kv_lens"], q_lens=s["q_lens"],
                                causal=s["case"]["causal"])


def _rotate(x, cos, sin, interleaved):
    """x [B, L, H, 128] in 32 bits, cos / sin [B, L, rot / 2]."""
    rot = 2 * cos.shape[-1]
    c, s = cos[:, :, None, :], sin[:, :, None, :]
    turned, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = turned[..., 0::2], turned[..., 1::2]
        new = torch.stack([a * c - b * s, a * s + b * c], dim=-1).flatten(-2)
    else:
        a, b = turned[..., :rot // 2], turned[..., rot // 2:]
        new = torch.cat([a * c - b * s, a * s + b * c], dim=-1)
    return torch.cat([new, rest], dim=-1)


def _rope(s):
    cos, sin = s["cos"][s["at"].long()], s["sin"][s["at"].long()]
    return tuple(_rotate(x.float(), cos, sin, s["case"]["interleaved"]).to(x.dtype) for x in (s["q"], s["k"]))


def _write_one(codes, amax, page, old, new, at, x, fmt):
    """Writes x [B, L, H, 128] into the touched pages. page [B, N]; old / new [B, N, 64]: rows that the page held before
    and rows that come from x; at [B, N, 64]: x's row. In 64 bits: a value next to a border of two codes counts."""
    dt, q = FORMATS[fmt]
    batch, count, _ = old.shape
    rows = torch.arange(batch, device=x.device)[:, None, None]
    raw = codes.view(torch.int8)
    fresh = x[rows, at].permute(0, 1, 3, 2, 4).double()                    # [B, N, H, 64, 128]
    finite = torch.where(torch.isfinite(fresh) & new[:, :, None, :, None], fresh.abs(), 0.0)
    was = raw[page].view(dt).double()
    had = torch.where(old.any(-1)[..., None], amax[page].double(), 0.0)    # [B, N, H]
    top = torch.maximum(had, finite.amax(dim=(-1, -2))).clamp_min(FLOOR)
    kept = was * (had / top)[..., None, None]
    put = (torch.nan_to_num(fresh, nan=0.0, posinf=3e38, neginf=-3e38) * q / top[..., None, None]).clamp(-q, q)
    value = torch.where(new[:, :, None, :, None], put, kept)
    value = (value.round() if fmt == "int8" else value).float().to(dt).view(torch.int8)
    value = torch.where((old | new)[:, :, None, :, None], value, raw[page])
    touched = new.any(-1)
    raw[page[touched]] = value[touched]
    amax[page[touched]] = top[touched].float()


def _write(s):
    case = s["case"]
    k, v, start, count = s["k"], s["v"], s["start"].long(), s["new"].long()
    if case["rot"]:
        at = (start[:, None] + torch.arange(case["len"], device=k.device)).clamp_max(s["cos"].shape[0] - 1)
        k = _rotate(k.float(), s["cos"][at], s["sin"][at], True).to(k.dtype)
    blocks = (case["len"] + PAGE - 2) // PAGE + 1
    first = start // PAGE
    block = first[:, None] + torch.arange(blocks, device=k.device)
    page = s["table"].gather(1, block.clamp_max(s["table"].shape[1] - 1)).long().clamp_min(0)
    token = block[:, :, None] * PAGE + torch.arange(PAGE, device=k.device)
    i = token - start[:, None, None]
    new, old = (i >= 0) & (i < count[:, None, None]), i < 0
    at = i.clamp(0, case["len"] - 1)
    for x, codes, amax in ((k, s["k_pages"], s["k_amax"]), (v, s["v_pages"], s["v_amax"])):
        _write_one(codes, amax, page, old, new, at, x, case["format"])
    back = [_window(codes, amax, s, case["format"]).to(k.dtype) for codes, amax in
            ((s["k_pages"], s["k_amax"]), (s["v_pages"], s["v_amax"]))]
    return {"k": back[0], "v": back[1]}


def _window(codes, amax, s, fmt):
    """Values [B, longest, H, 128] of the tokens from `first` on, 0 behind `back` of them."""
    i = torch.arange(s["longest"], device=codes.device)
    token = s["first"].long()[:, None] + i
    keep = i < s["back"][:, None]
    page = s["table"].gather(1, (token // PAGE).clamp_max(s["table"].shape[1] - 1)).long().clamp_min(0)
    value = codes.view(torch.int8)[page, :, token % PAGE].view(codes.dtype).float() * amax[page][..., None] / FORMATS[fmt][1]
    return torch.where(keep[:, :, None, None], value, 0.0)


def _copy(s):
    for t in (s["k_pages"], s["v_pages"]):
        raw = t.view(torch.int8)
        raw[:, s["dst"]] = raw[:, s["src"]]
    for t in (s["k_amax"], s["v_amax"]):
        t[:, s["dst"]] = t[:, s["src"]]
    return {"k": s["k_pages"], "v": s["v_pages"], "k_amax": s["k_amax"], "v_amax": s["v_amax"]}


def _attend(s):
    case = s["case"]
    b, lq, hq, _ = s["q"].shape
    h, g = case["kv_heads"], case["group"]
    page = s["table"].long().clamp_min(0)
    kv = page.shape[1] * PAGE
    top = FORMATS[case["format"]][1]

    def values(codes, amax):
        x = codes.view(torch.int8)[page].view(codes.dtype).float() * (amax[page] / top)[..., None, None]       # [B, pages, H, 64, 128]
        return x.permute(0, 2, 1, 3, 4).reshape(b, h, kv, DIM)

    q = s["q"].float().reshape(b, lq, h, g, DIM).permute(0, 2, 1, 3, 4).reshape(b, h, lq * g, DIM)
    score = torch.matmul(q, values(s["k_pages"], s["k_amax"]).transpose(-1, -2)) * DIM ** -0.5
    i = torch.arange(lq, device=q.device)
    j = torch.arange(kv, device=q.device)
    kvs = s["kv_lens"].long()
    qs = s["q_lens"].long() if s["q_lens"] is not None else torch.full_like(kvs, lq)
    see = (j < kvs[:, None])[:, None, :].expand(b, lq, kv)
    if case["causal"]:
        see = see & (j <= (kvs - qs)[:, None, None] + i[None, :, None])
    see = (see & (i < qs[:, None])[:, :, None]).repeat_interleave(g, dim=1)[:, None]
    score = score.masked_fill_(~see, -torch.inf)
    peak = score.amax(-1, keepdim=True)
    p = torch.exp(score.sub_(torch.where(peak == -torch.inf, 0.0, peak)))
    total = p.sum(-1, keepdim=True)
    # masked keys have weight 0; their values are codes, finite always
    out = torch.matmul(p, values(s["v_pages"], s["v_amax"])) / torch.where(total == 0, 1.0, total)
    return out.reshape(b, h, lq, g, DIM).permute(0, 2, 1, 3, 4).reshape(b, lq, hq, DIM).to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    if case["op"] == "copy":
        return None                                  # nothing is computed
    s = prepare(case, seed)
    return {"rope": _exact_rope, "write": _exact_write, "attend": _exact_attend}[case["op"]](s)


def _exact_turn(x, angle, interleaved):
    """x [L, H, 128] in 64 bits as complex numbers, turned by angle [L, rot / 2]."""
    half = angle.shape[-1]
    out = x.clone()
    if interleaved:
        z = torch.complex(x[..., 0:2 * half:2], x[..., 1:2 * half:2])
    else:
        z = torch.complex(x[..., :half], x[..., half:2 * half])
    z = z * torch.polar(torch.ones_like(angle), angle)[:, None, :]
    if interleaved:
        out[..., 0:2 * half:2], out[..., 1:2 * half:2] = z.real, z.imag
    else:
        out[..., :half], out[..., half:2 * half] = z.real, z.imag
    return out


def _exact_rope(s):
    case = s["case"]
    ang = _angles(case["positions"], case["rot"], s["q"].device)[s["at"].long().flatten()]
    return tuple(_exact_turn(x.double().flatten(0, 1), ang, case["interleaved"]).reshape(x.shape)
                 for x in (s["q"], s["k"]))


def _exact_write(s):
    """Page by page: the codes that each touched page holds afterwards, and the values they stand for."""
    case = s["case"]
    dt, top = FORMATS[case["format"]]
    outs = {}
    for name in ("k", "v"):
        codes = s[name + "_pages"].double()
        amax = s[name + "_amax"].double().clone()
        back = torch.zeros(case["batch"], s["longest"], case["heads"], DIM, dtype=torch.float64, device=codes.device)
        for b, (start, n) in enumerate(zip(*_starts(case))):
            x = s[name][b, :n].double()
            if name == "k" and case["rot"]:
                ang = _angles(start + n, case["rot"], x.device)[start:]
                x = _exact_turn(x, ang, True).to(s[name].dtype).double()   # the cache is given the activation type
            for blk in range(start // PAGE, (start + n - 1) // PAGE + 1):
                page = int(s["table"][b, blk])
                lo, hi = max(start, blk * PAGE), min(start + n, (blk + 1) * PAGE)
                part = x[lo - start:hi - start]                             # [n, H, 128]
                held = lo - blk * PAGE                                      # rows the page held before
                biggest = part.abs().amax(dim=(0, 2)).clamp_min(FLOOR)
                if held:
                    biggest = torch.maximum(biggest, amax[page])
                    moved = codes[page, :, :held] * (amax[page] / biggest)[:, None, None]
                    codes[page, :, :held] = moved.round() if dt == torch.int8 else moved.float().to(dt).double()
                fresh = (part * top / biggest[:, None]).transpose(0, 1)
                codes[page, :, held:held + hi - lo] = fresh.round() if dt == torch.int8 else fresh.float().to(dt).double()
                amax[page] = biggest
                at = blk * PAGE - start // PAGE * PAGE
                size = held + hi - lo
                back[b, at:at + size] = (codes[page, :, :size] * (amax[page] / top)[:, None, None]).transpose(0, 1)
        outs[name] = back
    return outs


def _exact_attend(s):
    """Sequence by sequence and head by head, over the keys that it holds."""
    case = s["case"]
    g, top = case["group"], FORMATS[case["format"]][1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    for b, (kv, n) in enumerate(zip(*_lengths(case))):
        if kv == 0:
            continue
        page = s["table"][b, :(kv + PAGE - 1) // PAGE].long()
        for h in range(case["kv_heads"]):
            k, v = ((s[x + "_pages"].view(torch.int8)[page, h].view(FORMATS[case["format"]][0]).double() * (s[x + "_amax"][page, h].double() / top)[:, None, None])
                    .reshape(-1, DIM)[:kv] for x in "kv")
            for lo in range(0, n, 2048):
                q = s["q"][b, lo:min(n, lo + 2048), h * g:(h + 1) * g].double()        # [n, g, 128]
                score = torch.einsum("igd,jd->gij", q, k) / DIM ** 0.5
                if case["causal"]:
                    i = torch.arange(lo, lo + q.shape[0], device=k.device)
                    hidden = torch.arange(kv, device=k.device)[None, :] > kv - n + i[:, None]
                    score.masked_fill_(hidden, -torch.inf)
                weight = torch.softmax(score, dim=-1).nan_to_num_(0.0)                 # a row without keys: zeros
                out[b, lo:lo + q.shape[0], h * g:(h + 1) * g] = torch.einsum("gij,jd->igd", weight, v)
    return out
