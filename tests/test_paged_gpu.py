"""The paged 8-bit cache on the GPU against tests/_paged.py in float64: written codes and scales bit for bit, read-back
values within the output's rounding, attention within the tolerance derived in _paged.attend plus half a step of the
output type."""
import bisect
import math
from fractions import Fraction

import pytest
import torch

from tests import _paged as P

pytestmark = pytest.mark.gpu

FORMATS = pytest.mark.parametrize("fmt", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])


def pool(pages):
    from lingbot_b200 import paged_cache
    return paged_cache.Pages(*(t.cuda() for t in pages))


def raw(t):
    return t.cpu().view(torch.uint8)


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------------------ write and window
@FORMATS
@TYPES
@pytest.mark.parametrize("heads,length,starts,lens", [
    (3, 1, [0, 63, 64, 130], None), (2, 64, [0, 64], None), (1, 200, [5, 0, 127], [200, 1, 77]),
    (2, 130, [190, 64], [0, 130]), (12, 7, [60], None)])
def test_write_gives_the_exact_codes(fmt, dtype, heads, length, starts, lens):
    """Fresh pages, pages inside which the write begins (their scale grows or not), lengths of 0; pages and rows that no
    token enters keep their bits; writing again changes nothing; the values read back."""
    from lingbot_b200 import paged_cache as pc
    b = len(starts)
    counts = lens or [length] * b
    need = [(s + n + 63) // 64 for s, n in zip(starts, counts)]
    pages = P.make_pages(7 * length + heads, sum(need) + 2, heads, fmt, spread=2.5)
    table = P.make_table(1, need, sum(need) + 2)
    g = torch.Generator().manual_seed(length)
    # magnitudes around the held tokens', so that some pages' scales grow and others do not
    k, v = ((torch.randn(b, length, heads, 128, generator=g) * 2.0 ** torch.empty(b, 1, heads, 1).uniform_(-2, 1, generator=g))
            .to(dtype) for _ in range(2))
    got = pool(pages)
    start = starts[0] if b == 1 else i32(starts)
    args = (got, table.cuda(), start, k.cuda(), v.cuda())
    pc.write(*args, lens=None if lens is None else i32(lens))
    want = [t.clone() for t in pages]
    P.write(want[0], want[2], table, starts, counts, k, fmt)
    P.write(want[1], want[3], table, starts, counts, v, fmt)
    for x, y in zip((got.k, got.v, got.k_amax, got.v_amax), want):
        assert torch.equal(raw(x), raw(y))
    pc.write(*args, lens=None if lens is None else i32(lens))
    for x, y in zip((got.k, got.v, got.k_amax, got.v_amax), want):
        assert torch.equal(raw(x), raw(y))
    total = [s + n for s, n in zip(starts, counts)]
    back = pc.window(got, table.cuda(), 0, max(total) or 1, dtype, lens=i32(total))
    for x, codes, amax in zip(back, want[:2], want[2:]):
        for s in range(b):
            ref = P.gather(codes, amax, table[s], total[s], fmt)
            tol = ref.abs() * (torch.finfo(dtype).eps / 2 * (1 + 2.0 ** -10) + 2.0 ** -23) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
            assert bool(((x[s, :total[s]].cpu().double() - ref).abs() <= tol).all())
            assert not x[s, total[s]:].any()


@FORMATS
def test_write_non_finite_huge_and_tiny(fmt):
    """NaN becomes 0 and infinities the largest code, under the scale of the finite values; magnitudes at both ends of
    bf16; all-zero and all-NaN tokens; a subnormal below the floor."""
    from lingbot_b200 import paged_cache as pc
    k = torch.randn(6, 20, 2, 128, generator=torch.Generator().manual_seed(0)).bfloat16()
    k[0, 3, 0, 5], k[0, 4, 0, 6], k[0, 5, 1, 7] = float("nan"), float("inf"), float("-inf")
    k[1] = k[1] * 1e38
    k[1, 0, 0, 0] = 3.3895e38
    k[2] = k[2] * 1e-30
    k[3] = 0
    k[4] = float("nan")
    k[5] = k[5] * 2.0 ** -38
    pages = P.make_pages(3, 8, 2, fmt)
    table = P.make_table(2, [1] * 6, 8)
    got = pool(pages)
    pc.write(got, table.cuda(), 0, k.cuda(), k.cuda())
    want = [t.clone() for t in pages]
    P.write(want[0], want[2], table, [0] * 6, [20] * 6, k, fmt)
    for x, y in ((got.k, want[0]), (got.k_amax, want[2])):
        assert torch.equal(raw(x), raw(y))
    x, _ = pc.window(got, table.cuda(), 0, 20)
    assert bool(torch.isfinite(x).all())


def exact_code(x, fmt):
    """The code nearest to a fraction, half way cases to the even one."""
    grid = [float(i) for i in range(128)] if fmt == torch.int8 else P.values(torch.arange(127, dtype=torch.uint8).view(fmt)).tolist()
    hi = max(1, bisect.bisect_left(grid, abs(x)))
    below, above = abs(x) - Fraction(grid[hi - 1]), Fraction(grid[hi]) - abs(x)
    i = hi if above < below or (above == below and hi % 2 == 0) else hi - 1
    return -grid[i] if x < 0 else grid[i]


@FORMATS
@TYPES
def test_held_codes_half_way_between_two_go_to_the_even_one(fmt, dtype):
    """Every code a page can hold, under growths of its scale by simple ratios, against rational arithmetic: c * old / a
    is half way between two codes for many of them, whichever way old / a itself would be rounded in any precision."""
    from lingbot_b200 import paged_cache as pc
    ratios = [(n, d) for d in range(2, 24) for n in range(1, d) if math.gcd(n, d) == 1]
    held = torch.arange(256, dtype=torch.uint8).view(torch.int8)
    held = torch.where(held == -128, 0, held) if fmt == torch.int8 else torch.where((held & 127) == 127, 0, held).view(fmt)
    held = P.to_codes(P.values(held), fmt)
    n = len(ratios)
    codes = torch.zeros(1, n, 64, 128, dtype=torch.int8).view(fmt)
    codes.view(torch.int8)[0, :, :2] = held.view(torch.int8).reshape(2, 128)
    amax = torch.tensor([[float(r[0]) for r in ratios]])
    x = torch.zeros(1, 1, n, 128, dtype=dtype)
    x[0, 0, :, 0] = torch.tensor([float(r[1]) for r in ratios])
    got = pool((codes, codes.clone(), amax, amax.clone()))
    pc.write(got, i32([[0]]), 2, x.cuda(), x.cuda())
    ties = 0
    for h, (old, a) in enumerate(ratios):
        value = P.values(held).tolist()
        want = [exact_code(Fraction(c) * old / a, fmt) for c in value]
        ties += sum((Fraction(c) * old / a).denominator == 2 for c in value)
        for pages in (got.k, got.v):
            assert P.values(pages[0, h, :2].cpu()).flatten().tolist() == want, (old, a)
    assert fmt != torch.int8 or ties > 1000


@TYPES
@pytest.mark.parametrize("interleaved,rot", [(True, 128), (False, 128), (True, 8), (False, 48)])
def test_write_with_rope_equals_rope_then_write(dtype, interleaved, rot):
    from lingbot_b200 import paged_cache as pc, rope
    g = torch.Generator().manual_seed(rot)
    qkv = torch.randn(2, 150, 3 * 3, 128, generator=g).to(dtype).cuda()
    k, v = qkv[:, :, 3:6], qkv[:, :, 6:]                      # views of a fused projection
    table = P.make_table(5, [4, 4], 8).cuda()
    t = rope.tables(400, rot, interleaved=interleaved)
    starts = i32([70, 0])
    for positions in (None, torch.randint(0, 400, (2, 150), generator=g).cuda()):
        a, b = (pool(P.make_pages(1, 8, 3, torch.int8)) for _ in range(2))
        pc.write(a, table, starts, k, v, rope=t, positions=positions)
        rows = starts[:, None] + torch.arange(150, device="cuda") if positions is None else positions
        pc.write(b, table, starts, rope.apply(k, t, rows), v)
        for x, y in ((a.k, b.k), (a.v, b.v), (a.k_amax, b.k_amax)):
            assert torch.equal(raw(x), raw(y))


def test_bad_pages_and_positions_are_recorded_not_followed():
    from lingbot_b200 import _lib, paged_cache as pc, rope
    pages = P.make_pages(1, 4, 2, torch.int8)
    got = pool(pages)
    k = torch.randn(2, 70, 2, 128).bfloat16().cuda()
    table = torch.tensor([[0, 9], [-3, 2]], dtype=torch.int32)
    pc.write(got, table.cuda(), 0, k, k)
    assert _lib.device_status() == 0x305
    want = [t.clone() for t in pages]
    P.write(want[0], want[2], table[:1], [0], [64], k.cpu(), torch.int8)
    P.write(want[0], want[2], torch.tensor([[0, 2]]), [64], [6], k[1:, 64:].cpu(), torch.int8)
    assert torch.equal(raw(got.k), raw(want[0]))
    back, _ = pc.window(got, table.cuda(), 0, 128)
    assert _lib.device_status() == 0x305 and not back[0, 64:].any() and not back[1, :64].any() and back[1, 64:].any()
    pc.write(got, table[:1].cuda(), i32([128]), k[:1], k[:1])                   # past the table
    assert _lib.device_status() == 0x305
    pc.write(got, table[:1].cuda(), i32([-5]), k[:1], k[:1])
    assert _lib.device_status() == 0x305
    t = rope.tables(10, 128)
    pc.write(got, table[:1, :1].cuda().contiguous(), i32([8]), k[:1, :4], k[:1, :4], rope=t)
    assert _lib.device_status() == 0x306
    assert torch.equal(raw(got.v[1]), raw(pages[1][1])) and torch.equal(raw(got.v[3]), raw(pages[1][3]))
    # attention: the keys of a bad page count as masked; lengths past the table are cut
    q = torch.randn(2, 3, 2, 128).bfloat16().cuda()
    out = pc.attend(q, got, table.cuda(), i32([128, 128]))
    assert _lib.device_status() == 0x305
    for s, (row, lo) in enumerate(((0, 0), (1, 64))):
        good = int(table[row, 0 if s == 0 else 1])
        one = torch.tensor([[good]], dtype=torch.int32)
        ref, _, tol = P.attend(q[s:s + 1].cpu(), got.k.cpu(), got.v.cpu(), got.k_amax.cpu(), got.v_amax.cpu(), one, [64], [3],
                               False)
        assert bool(((out[s:s + 1].cpu().double() - ref).abs() <= tol + 2.0 ** -8 * ref.abs()).all())
    pc.attend(q, got, i32([[0], [2]]), i32([65, 64]))
    assert _lib.device_status() == 0x305
    pc.attend(q, got, i32([[0], [2]]), i32([-1, 64]))
    assert _lib.device_status() == 0x305


# ------------------------------------------------------------------------------------------------ copies
@pytest.mark.parametrize("layers,heads,total,moved", [(1, 1, 2, 1), (3, 5, 40, 17), (2, 2, 1100, 500)])
def test_copy_pages(layers, heads, total, moved):
    from lingbot_b200 import paged_cache as pc
    g = torch.Generator().manual_seed(total)
    codes = [torch.randint(-127, 128, (layers, total, heads, 64, 128), generator=g, dtype=torch.int8) for _ in range(2)]
    amax = [torch.rand(layers, total, heads, generator=g) for _ in range(2)]
    p = pool([*codes, *amax])
    ids = torch.randperm(total, generator=g).tolist()
    src, dst = ids[:moved], ids[moved:2 * moved]
    src[-1] = src[0]                                                           # one source twice
    pc.copy_pages(p, src, dst)
    for x, y in zip((p.k, p.v, p.k_amax, p.v_amax), codes + amax):
        y[:, dst] = y[:, src]
        assert torch.equal(x.cpu(), y)


# ------------------------------------------------------------------------------------------------ attention
def run_attend(q, pages, table, kvs, qs, causal, **kw):
    """Out and lse against the float64 evaluation."""
    from lingbot_b200 import paged_cache as pc
    p = pool(pages)
    ragged = qs != [q.shape[1]] * q.shape[0]
    out, lse = pc.attend(q.cuda(), p, table.cuda(), i32(kvs), q_lens=i32(qs) if ragged else None, causal=causal,
                         return_lse=True, **kw)
    ref, ref_lse, tol = P.attend(q, *pages, table, kvs, qs, causal, kw.get("sm_scale", 128 ** -0.5))
    err = (out.cpu().double() - ref).abs()
    tol = tol + torch.finfo(q.dtype).eps / 2 * ref.abs() * 1.01 + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    assert bool((err <= tol).all()), (float((err - tol).max()), float((err / tol).max()))
    none = ref_lse == -torch.inf
    assert torch.equal(lse.cpu() == -torch.inf, none) and not out.cpu()[none].any()
    # the sum of the weights is off by as much as a weight, the maximum by its score: at most 2^-11 and a rounding
    assert bool(((lse.cpu().double() - ref_lse)[~none].abs() <= 2.0 ** -11 + 2.0 ** -20 * ref_lse[~none].abs()).all())
    return out, lse


@FORMATS
@TYPES
@pytest.mark.parametrize("causal", [False, True], ids=["full", "causal"])
@pytest.mark.parametrize("kvs,lq,qs,heads,group", [
    ([1], 1, None, 1, 1), ([64], 1, None, 2, 1), ([65, 63], 1, None, 3, 4), ([1000], 1, None, 12, 1),
    ([300, 0, 17, 640], 5, None, 2, 3), ([300, 5, 129, 64], 9, [9, 7, 1, 0], 1, 8), ([2000], 1, None, 1, 16),
    ([513, 900], 40, [40, 33], 2, 1), ([130], 200, None, 1, 2), ([1111], 300, None, 2, 1), ([700, 64], 257, [130, 257], 1, 3)])
def test_attend_matches_float64(fmt, dtype, causal, kvs, lq, qs, heads, group):
    b = len(kvs)
    counts = [(n + 63) // 64 for n in kvs]
    pages = P.make_pages(sum(kvs) + lq, sum(counts) + 2, heads, fmt, spread=3.0)
    table = P.make_table(lq, counts, sum(counts) + 2, width=max(counts) + 3)
    g = torch.Generator().manual_seed(lq)
    q = (torch.randn(b, lq, heads * group, 128, generator=g) * 1.5).to(dtype)
    run_attend(q, pages, table, kvs, qs or [lq] * b, causal)


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 16, 40])
@pytest.mark.parametrize("lq,group", [(1, 1), (4, 8), (150, 2)])
def test_attend_key_splits(splits, lq, group):
    """Every split count, uneven ones and more than there are pages among them; sequences that end in the first split."""
    kvs = [1000, 40, 0, 641]
    pages = P.make_pages(11, 40, 2, torch.int8, spread=2.0)
    table = P.make_table(4, [16, 1, 0, 11], 40)
    q = torch.randn(4, lq, 2 * group, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    run_attend(q, pages, table, kvs, [lq] * 4, True, num_splits=splits)


@pytest.mark.parametrize("lq,group", [(1, 1), (3, 5), (90, 1)])
def test_attend_long_splits(lq, group):
    """Hundreds of pages in one split: the ring of page slots goes round many times in every warp's order."""
    kvs = [20000, 12345]
    pages = P.make_pages(12, 510, 1, torch.int8)
    table = P.make_table(5, [313, 193], 510)
    q = torch.randn(2, lq, group, 128, generator=torch.Generator().manual_seed(1)).bfloat16()
    outs = [run_attend(q, pages, table, kvs, [lq] * 2, True, num_splits=n)[0] for n in (1, 1, 1, 4)]
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@FORMATS
@pytest.mark.parametrize("lq", [1, 129], ids=["token", "chunk"])
def test_attend_wide_ranges(fmt, lq):
    """Pages whose V differ by 2^12 and K by 2^4, large query rows beside tiny ones, a softmax that picks one key."""
    kvs = [600]
    k, v, ka, va = P.make_pages(5, 10, 1, fmt, spread=4.0)
    va = 2.0 ** (torch.arange(10.0) * 12 / 9 - 6)[:, None]
    table = P.make_table(9, [10], 10)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(1, lq, 2, 128, generator=g)
    q[:, :, 1] *= 30
    q[:, ::2, 0] *= 2.0 ** -60
    run_attend(q.bfloat16(), (k, v, ka, va), table, kvs, [lq], False)
    run_attend(q.bfloat16(), (k, v, ka, va), table, kvs, [lq], False, sm_scale=1.5)


@pytest.mark.parametrize("lq", [1, 130], ids=["token", "chunk"])
def test_attend_strides_stale_rows_and_padding(lq):
    """q and out as views of larger tensors; garbage past a sequence's tokens, in other pages and in padded query rows
    (NaN there) changes nothing; rows past q_lens are 0; a broadcast query; a shared page table row."""
    from lingbot_b200 import paged_cache as pc
    kvs, qs = [100, 190], [max(1, lq - 3), lq]
    pages = P.make_pages(8, 8, 2, torch.float8_e4m3fn)
    table = P.make_table(3, [2, 3], 8)
    g = torch.Generator().manual_seed(0)
    big = torch.randn(2, lq, 3, 4, 128, generator=g).bfloat16().cuda()
    q = big[:, :, 1]
    p = pool(pages)
    want = pc.attend(q.contiguous(), p, table.cuda(), i32(kvs), q_lens=i32(qs))
    assert not want[0, qs[0]:].any()
    hold = torch.full((2, lq, 6, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = pc.attend(q, p, table.cuda(), i32(kvs), q_lens=i32(qs), out=hold[:, :, 1:5])
    assert torch.equal(got, want) and bool((hold[:, :, 0] == 7).all()) and bool((hold[:, :, 5] == 7).all())
    k2, v2 = (t.clone() for t in pages[:2])
    for t in (k2, v2):
        raw_t = t.view(torch.uint8)
        raw_t[table[0, 1].item(), :, 36:] = 0x7F                              # NaN codes behind the last token
        raw_t[[i for i in range(8) if i not in table.flatten().tolist()]] = 0xFF
    q2 = q.clone()
    q2[0, qs[0]:] = float("nan")
    again = pc.attend(q2, pool((k2, v2, *pages[2:])), table.cuda(), i32(kvs), q_lens=i32(qs))
    assert torch.equal(again, want)
    wide = torch.full((2, 50), -1, dtype=torch.int32)
    wide[:, :3] = table
    same = pc.attend(q, p, wide.cuda(), i32(kvs), q_lens=i32(qs), max_kv_len=190)
    assert torch.equal(same, want)
    e = q[:1].expand(2, lq, 4, 128)
    shared = table[1:].cuda().expand(2, 3)
    both = pc.attend(e, p, shared, 190)
    assert torch.equal(both[0], both[1])


def test_attend_rows_with_nan_or_inf_stay_alone():
    from lingbot_b200 import paged_cache as pc
    for lq in (4, 140):
        pages = P.make_pages(8, 4, 1, torch.int8)
        table = P.make_table(3, [4], 4).cuda()
        q = torch.randn(1, lq, 2, 128, generator=torch.Generator().manual_seed(0)).bfloat16().cuda()
        want = pc.attend(q, pool(pages), table, 250)
        q[0, 1, 0, 3] = float("nan")
        q[0, 2, 1, 9] = float("inf")
        got = pc.attend(q, pool(pages), table, 250)
        assert bool(got[0, 1, 0].isnan().all()) and bool(got[0, 2, 1].isnan().any())
        keep = torch.ones(lq, 2, dtype=torch.bool, device="cuda")
        keep[1, 0] = keep[2, 1] = False
        assert torch.equal(got[0][keep], want[0][keep])


def test_pool_larger_than_32_bits_of_bytes():
    """Pages behind the first 4 GiB of each tensor: written, read, copied and attended."""
    from lingbot_b200 import paged_cache as pc
    n, h = 45000, 12                                                           # 4.4 GB a tensor
    p = pc.alloc_pages(n, h, "cuda")
    ids = [n - 1, 3, n - 7, 20000]
    table = i32([ids])
    g = torch.Generator().manual_seed(0)
    k, v = (torch.randn(1, 250, h, 128, generator=g).bfloat16().cuda() for _ in range(2))
    pc.write(p, table, 0, k, v)
    small = pc.alloc_pages(4, h, "cuda")
    pc.write(small, i32([[0, 1, 2, 3]]), 0, k, v)
    for a, b in ((p.k, small.k), (p.v, small.v), (p.k_amax, small.k_amax)):
        assert torch.equal(a[ids], b)
    for lq in (1, 150):
        q = torch.randn(1, lq, h, 128, generator=g).bfloat16().cuda()
        assert torch.equal(pc.attend(q, p, table, 250), pc.attend(q, small, i32([[0, 1, 2, 3]]), 250))
    pc.copy_pages(p, [n - 1, n - 7], [5, n - 2])
    assert torch.equal(p.k[5], small.k[0]) and torch.equal(p.v[n - 2], small.v[2])
    x, y = pc.window(p, table, 0, 250), pc.window(small, i32([[0, 1, 2, 3]]), 0, 250)
    assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])


def test_streams_graphs_and_gradients():
    """Calls on two streams at once, and two captured graphs replayed in turn on changing lengths, give what eager calls
    give; a query that needs a gradient is refused."""
    from lingbot_b200 import paged_cache as pc
    pages = P.make_pages(8, 40, 4, torch.int8)
    p = pool(pages)
    table = P.make_table(3, [16, 16], 40).cuda()
    g = torch.Generator().manual_seed(0)
    qs = [torch.randn(2, lq, 8, 128, generator=g).bfloat16().cuda() for lq in (1, 3, 140)]
    lens = i32([1000, 700])
    want = [pc.attend(q, p, table, lens, causal=True) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for r in range(6):
        with torch.cuda.stream(streams[r % 2]):
            got += [pc.attend(q, p, table, lens, causal=True) for q in qs]
    torch.cuda.synchronize()
    for i, x in enumerate(got):
        assert torch.equal(x, want[i % 3])
    graphs, outs = [], []
    for q in qs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(pc.attend(q, p, table, lens, causal=True))
        graphs.append(graph)
    for new in ([1000, 700], [3, 0], [64, 1024]):
        lens.copy_(i32(new))
        for r in range(2):
            for graph in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for q, x in zip(qs, outs):
            assert torch.equal(x, pc.attend(q, p, table, i32(new), causal=True))
    with pytest.raises(RuntimeError, match="gradient"):
        pc.attend(qs[0].clone().requires_grad_(), p, table, lens)


def test_refusals():
    from lingbot_b200 import paged_cache as pc, rope
    p = pool(P.make_pages(8, 4, 2, torch.int8))
    table, lens = i32([[0, 1], [2, 3]]), i32([100, 128])
    q = torch.randn(2, 3, 4, 128).bfloat16().cuda()
    big = 1 << 70
    for exc, word, call in [
            (ValueError, "multiple", lambda: pc.attend(q[:, :, :3], p, table, lens)),
            (TypeError, "q must be", lambda: pc.attend(q.float(), p, table, lens)),
            (ValueError, "pages on", lambda: pc.attend(q.cpu(), p, table, lens)),
            (ValueError, "page table", lambda: pc.attend(q, p, table.long(), lens)),
            (ValueError, "page table", lambda: pc.attend(q, p, table[:1], lens)),
            (ValueError, "page table", lambda: pc.attend(q, p, table.cpu(), lens)),
            (ValueError, "kv_lens", lambda: pc.attend(q, p, table, lens.long())),
            (ValueError, "negative", lambda: pc.attend(q, p, table, -1)),
            (Exception, "outside", lambda: pc.attend(q, p, table, 129)),
            (TypeError, "q_lens", lambda: pc.attend(q, p, table, lens, q_lens=3)),
            (ValueError, "exceeds", lambda: pc.attend(q, p, table, 100, max_kv_len=99)),
            (ValueError, "overlaps", lambda: pc.attend(q[:, :2], p, table, lens, out=q[:, 1:])),
            (ValueError, "share memory", lambda: pc.attend(q, p, table, lens, out=torch.empty_like(q)[:, :1].expand(q.shape))),
            (ValueError, "heads", lambda: pc.write(p, table, 0, q, q)),
            (ValueError, "differ", lambda: pc.write(p, table, 0, q[:, :, :2], q[:, :2, :2])),
            (ValueError, "positions", lambda: pc.write(p, table, 0, q[:, :, :2], q[:, :, :2], positions=lens)),
            (ValueError, "of 3 tokens", lambda: pc.write(p, table, 0, q[:, :, :2], q[:, :, :2], lens=4)),
            (Exception, "outside", lambda: pc.write(p, table, 126, q[:, :, :2], q[:, :, :2])),
            (RuntimeError, "gradient", lambda: pc.write(p, table, 0, q[:, :, :2].clone().requires_grad_(), q[:, :, :2])),
            (Exception, "outside", lambda: pc.window(p, table, 100, 29)),
            (ValueError, "negative", lambda: pc.window(p, table, 0, -1)),
            (TypeError, "dtype", lambda: pc.window(p, table, 0, 1, torch.float32)),
            (ValueError, "twice", lambda: pc.copy_pages(p, [0, 1], [2, 2])),
            (ValueError, "both", lambda: pc.copy_pages(p, [0, 1], [1, 2])),
            (Exception, "outside", lambda: pc.copy_pages(p, [0], [4])),
            (Exception, "outside", lambda: pc.copy_pages(p, [-1], [3])),
            (Exception, None, lambda: pc.window(p, table, 0, big)),
            (ValueError, "64 bits", lambda: pc.window(p, table, big, 1)),
            (ValueError, "start", lambda: rope.apply(q, rope.tables(8, 64), start=big)),
            (ValueError, "start", lambda: rope.apply(q, rope.tables(8, 64), start=-1))]:
        with pytest.raises(exc, match=word):
            call()
    # in place, lengths as ints, nothing to do
    want = pc.attend(q, p, table, 128)
    x = q.clone()
    assert pc.attend(x, p, table, 128, out=x).data_ptr() == x.data_ptr() and torch.equal(x, want)
    assert torch.equal(pc.attend(q, p, table, i32([128, 128]), return_lse=True)[0], want)
    assert pc.attend(q[:0], p, table[:0], lens[:0]).shape == (0, 3, 4, 128)
    assert pc.attend(q[:, :0], p, table, lens).shape == (2, 0, 4, 128)
    before = p.k.clone()
    pc.write(p, table, 0, q[:, :0, :2], q[:, :0, :2])
    pc.write(p, table, 0, q[:, :, :2], q[:, :, :2], lens=0)
    pc.copy_pages(p, [], [])
    assert torch.equal(raw(p.k), raw(before))


def test_first_calls_of_a_process_can_be_captured():
    """Nothing needs a call outside a capture first."""
    import os
    import subprocess
    import sys
    code = """
import torch
from lingbot_b200 import paged_cache as pc, rope, _lib
p = pc.alloc_pages(8, 2, "cuda")
t = rope.tables(200, 128)
table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device="cuda")
k = torch.randn(1, 150, 2, 128, device="cuda").bfloat16()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    pc.write(p, table, 0, rope.apply(k, t), k)
    pc.copy_pages(p, [0], [5])
    outs = [pc.attend(k[:, :n].contiguous(), p, table, 150) for n in (1, 150)]
    back = pc.window(p, table, 0, 150)
g.replay()
torch.cuda.synchronize()
assert torch.equal(outs[0], pc.attend(k[:, :1].contiguous(), p, table, 150))
assert torch.equal(outs[1], pc.attend(k, p, table, 150)) and torch.equal(back[0], pc.window(p, table, 0, 150)[0])
assert torch.equal(p.k[5], p.k[0]) and bool(p.k.any()) and _lib.device_status() == 0
print("captured")
"""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lingbot-world-v2-realtime_b200")
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                       env=dict(os.environ, PYTHONPATH=root))
    assert r.returncode == 0 and "captured" in r.stdout, r.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ the cache as used
@FORMATS
def test_sessions_prefill_decode_fork_evict_compact(fmt):
    """Two layers: a prompt, generated tokens with rope, a fork that goes its own way, an eviction, compaction, a captured
    decode step; every attention against float64 on a model that keeps the sessions' codes as the formulas give them."""
    from lingbot_b200 import paged_cache as pc, rope
    heads, group, layers = 2, 2, 2
    c = pc.allocate(layers, 24, heads, max_pages=8, device="cuda", fmt=fmt)
    t = rope.tables(600, 64, interleaved=False)
    g = torch.Generator().manual_seed(5)

    def rand(b, n, h):
        return torch.randn(b, n, h, 128, generator=g).bfloat16().cuda()

    def step(sessions, new, causal=True, passes=1, at=None):
        plan = c.plan(sessions, new)
        b, n = len(sessions), max(plan.new)
        for layer in range(layers):
            for _ in range(passes):
                k, v, q = rand(b, n, heads), rand(b, n, heads), rand(b, n, heads * group)
                before = [x.cpu() for x in (c.layers[layer].k, c.layers[layer].v, c.layers[layer].k_amax, c.layers[layer].v_amax)]
                rows = plan.start[:, None] + torch.arange(n, device="cuda")
                if at is not None:
                    rows = rows + i32([at.get(s, 0) for s in sessions])[:, None]
                c.write(layer, plan, k, v, rope=t, positions=None if at is None else rows.contiguous())
                kr = rope.apply(k, t, rows)
                table = plan.table.cpu()
                P.write(before[0], before[2], table, plan.held, plan.new, kr.cpu(), fmt)
                P.write(before[1], before[3], table, plan.held, plan.new, v.cpu(), fmt)
                qr = rope.apply(q, t, rows)
                out = c.attend(layer, plan, qr, causal=causal)
                kvs = [h + m for h, m in zip(plan.held, plan.new)]
                ref, _, tol = P.attend(qr.cpu(), *before, table, kvs, plan.new, causal)
                assert bool(((out.cpu().double() - ref).abs() <= tol + 2.0 ** -8 * ref.abs() * 1.01).all())
                for x, y in zip((c.layers[layer].k, c.layers[layer].v), before):
                    assert torch.equal(raw(x), raw(y))
        c.commit(plan)
        return plan

    a, b = c.open(), c.open()
    step([a, b], [200, 131])
    step([a, b], 1)
    f = c.fork(a)
    step([a, f, b], [3, 1, 64], causal=False, passes=2)
    assert c.page_ids(a)[:3] == c.page_ids(f)[:3] and c.page_ids(a)[3] != c.page_ids(f)[3]
    kept = [c.layers[i].k[c.page_ids(a)].cpu() for i in range(layers)]
    c.evict(f, 64, 64)
    c.close(b)
    assert c.compact() > 0
    assert max(c.page_ids(a) + c.page_ids(f)) == c.num_pages - c.free_pages - 1
    for i in range(layers):
        assert torch.equal(raw(c.layers[i].k[c.page_ids(a)]), raw(kept[i]))
    with pytest.raises(ValueError, match="positions"):
        step([f, a], [1, 5])
    step([f, a], [1, 5], at={f: 64})                          # 64 tokens were evicted from f: positions follow on
    # a captured decode step: the plan's tensors take the next step's values
    plan = c.fixed_plan(2)
    k, v, q = rand(2, 1, heads), rand(2, 1, heads), rand(2, 1, heads * group)
    c.plan([a, f], 1, into=plan)
    c.write(0, plan, k, v)
    c.attend(0, plan, q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.write(0, plan, k, v)
        out = c.attend(0, plan, q, causal=True)
    for _ in range(3):
        for x, h in ((k, heads), (v, heads), (q, heads * group)):
            x.copy_(rand(2, 1, h))
        graph.replay()
        torch.cuda.synchronize()
        eager = pc.attend(q, c.layers[0], plan.table, plan.kv_lens, causal=True, num_splits=1)
        assert torch.allclose(out.float(), eager.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
        c.commit(plan)
        c.plan([a, f], 1, into=plan)


# ------------------------------------------------------------------------------------------------ ends of the ranges
def test_starts_that_pass_64_bits_are_refused():
    from lingbot_b200 import paged_cache as pc, rope
    p = pool(P.make_pages(8, 4, 2, torch.int8))
    table, one = i32([[0, 1], [2, 3]]), i32([1, 1])
    k = torch.randn(2, 3, 2, 128).bfloat16().cuda()
    for s0 in (1 << 62, (1 << 63) - 1):
        for lens in (None, one):
            with pytest.raises(ValueError, match="64 bits"):
                pc.window(p, table, s0, 3, lens=lens)
            with pytest.raises(ValueError, match="64 bits"):
                pc.write(p, table, s0, k, k, lens=lens)
        with pytest.raises(ValueError, match="start"):
            rope.apply(k, rope.tables(8, 64), start=s0)


@FORMATS
@pytest.mark.parametrize("lq", [4, 140], ids=["few", "many"])
def test_attend_tiny_rows_on_pages_of_zeros(fmt, lq):
    """Masked keys in pages whose K are zero (amax 2^-40, as a write leaves it, or 0) under query rows down to bf16's smallest
    normal: the scores are 0 and no row becomes NaN. Scores of magnitude 1 from such rows and a page of 2^120 are right."""
    k, v, ka, va = P.make_pages(13, 5, 1, fmt)
    k.view(torch.int8)[1:4] = 0
    ka[1:4] = torch.tensor([[2.0 ** -40], [2.0 ** -40], [0.0]])
    ka[4] = 1.9 * 2.0 ** 120
    table = torch.tensor([[0, 1, 2, 3], [4, 1, 3, -1]], dtype=torch.int32)
    q = torch.randn(2, lq, 2, 128, generator=torch.Generator().manual_seed(3)) * 2.0 ** -118
    q[0, ::4] *= 2.0 ** 118
    q[0, 1::4] *= 2.0 ** 20
    q[:, 3::4] = torch.where(q[:, 3::4] > 0, 2.0 ** -126, 0.0)
    assert bool((q.bfloat16().abs().amax(-1) > 0).all())
    for causal in (True, False):
        run_attend(q.bfloat16(), (k, v, ka, va), table, [250, 190], [lq, lq], causal)


@FORMATS
@pytest.mark.parametrize("lq", [1, 129], ids=["few", "many"])
def test_attend_values_up_to_the_largest(fmt, lq):
    """V scales from 2^125 to bf16's largest finite value, which the write stores: in every page, and in some."""
    k, v, ka, va = P.make_pages(15, 6, 1, fmt)
    table = P.make_table(2, [5], 6)
    q = torch.randn(1, lq, 2, 128, generator=torch.Generator().manual_seed(4)).bfloat16()
    for scales in ([1.5 * 2.0 ** 126] * 6, [2.0 ** 125, 3.3895e38, 1.1 * 2.0 ** 126, 2.0 ** 127, 2.0 ** 120, 2.0 ** 126]):
        va = torch.tensor(scales).bfloat16().float()[:, None]
        for splits in (1, 3):
            run_attend(q, (k, v, ka, va), table, [300], [lq], False, num_splits=splits)


@FORMATS
@pytest.mark.parametrize("lq", [2, 130], ids=["few", "many"])
def test_attend_subnormal_rows(fmt, lq):
    """bf16 query rows below its smallest normal, down to one smallest subnormal, and rows of zeros, against K so large that
    the scores matter; the largest finite rows against K so small."""
    k, v, ka, va = P.make_pages(16, 6, 1, fmt)
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32)
    ka = torch.tensor([1.9 * 2.0 ** 126] * 3 + [2.0 ** -40] * 3).bfloat16().float()[:, None]
    q = torch.randn(2, lq, 2, 128, generator=torch.Generator().manual_seed(5)).clamp(-3.9, 3.9)
    q[0] = q[0] * 2.0 ** -129
    q[0, 1::3] = 0
    q[0, 1::3, 0, 17] = 2.0 ** -133
    q[0, 1::3, 1] = 0
    q[1] = q[1] / 4 * 3.3e38
    q = q.bfloat16()
    assert bool((q[0].float().abs() < 2.0 ** -126).all()) and bool(torch.isfinite(q).all()) and bool(q[0, 0].any())
    for causal in (False, True):
        run_attend(q[:1], (k, v, ka, va), table[:1], [150], [lq], causal)
        run_attend(q[1:], (k, v, ka, va), table[1:], [190], [lq], causal, sm_scale=2.0 ** -85)


def run_unlike(q, pages, table, kv, causal, **kw):
    """run_attend for one sequence whose V scales lie any distance apart. A weight is 2^7 times p_j amax_j / M at least, M the
    row's largest p amax, and its rounding to fp16 is off by 2^-25 at most where 2^-11 relative is less: in the output by
    2^-32 M |d_j| / (Q sum p), d_j the code. That is not a part of |v_j| where amax_j is far below M, as the 64-bit
    evaluation's tolerance has it."""
    from lingbot_b200 import paged_cache as pc
    k, v, ka, va = pages
    out, lse = pc.attend(q.cuda(), pool(pages), table.cuda(), i32([kv]), causal=causal, return_lse=True, **kw)
    ref, ref_lse, tol = P.attend(q, *pages, table, [kv], [q.shape[1]], causal)
    row, lq, top = table[0], q.shape[1], P.TOP[v.dtype]
    amax = P.gather(torch.full_like(v.float(), top).to(v.dtype), va, row, kv, v.dtype)[:, 0, 0]
    d = P.gather(v, torch.full_like(va, top), row, kv, v.dtype)[:, 0].abs().sum(0)
    for h in range(q.shape[2]):
        x = q[0, :, h].double() @ P.gather(k, ka, row, kv, k.dtype)[:, 0].T * 128 ** -0.5
        if causal:
            x = x.masked_fill(torch.arange(kv)[None] > kv - lq + torch.arange(lq)[:, None], -torch.inf)
        p = torch.softmax(x, -1)
        tol[0, :, h] += 2.0 ** -32 * (p * amax).amax(-1, keepdim=True) * d / top
    err = (out.cpu().double() - ref).abs()
    tol = tol + torch.finfo(q.dtype).eps / 2 * ref.abs() * 1.01 + torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    assert bool((err <= tol).all()), (float((err - tol).max()), float((err / tol).max()))
    assert bool(((lse.cpu().double() - ref_lse).abs() <= 2.0 ** -11 + 2.0 ** -20 * ref_lse.abs()).all())


@FORMATS
@pytest.mark.parametrize("lq", [1, 40, 129], ids=["token", "few", "many"])
def test_attend_values_of_unlike_pages(fmt, lq):
    """V scales of one sequence from 2^-40 (a page of zeros) to 2^127, the large ones first, last and between: the small
    pages' keys count in full in the sum and the log-sum-exp, whatever the order, the splits and the scores."""
    g = torch.Generator().manual_seed(6)
    k, v, ka, va = P.make_pages(17, 14, 1, fmt)
    v.view(torch.int8)[2] = 0
    table = P.make_table(6, [13], 14)
    q = torch.randn(1, lq, 2, 128, generator=g).bfloat16()
    tiny, one, huge = 2.0 ** -40, 1.0, 1.7 * 2.0 ** 126
    for scales in ([tiny] * 13 + [huge], [huge] + [tiny] * 13, [tiny, huge] * 7, [tiny] * 6 + [one] + [huge] + [tiny] * 6,
                   [2.0 ** (-40 + 12.5 * i) for i in range(14)], [2.0 ** (122.5 - 12.5 * i) for i in range(14)]):
        by_place = torch.tensor(scales).bfloat16().float()
        va = torch.empty(14, 1)
        va[table[0].long(), 0] = by_place[:13]
        va[[i for i in range(14) if i not in table[0].tolist()], 0] = by_place[13]
        for splits in (1, 3, 9):
            run_unlike(q, (k, v, ka, va), table, 810, True, num_splits=splits)
        run_unlike(q * 40, (k, v, ka, va), table, 810, False)


def test_outputs_that_share_memory_are_refused():
    from lingbot_b200 import paged_cache as pc
    p = pool(P.make_pages(8, 4, 2, torch.int8))
    table, lens = i32([[0, 1], [2, 3]]), i32([100, 128])
    want = pc.window(p, table, 3, 20)
    buf = torch.zeros(2, 20, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
    got = pc.window(p, table, 3, 20, out=(buf[:, :, 0], buf[:, :, 1]))           # of one buffer, one after the other
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    k, v = torch.empty_like(want[0]), torch.empty_like(want[1])
    flat = torch.zeros(40000, dtype=torch.bfloat16, device="cuda")
    wide = torch.zeros(2, 20, 3, 128, dtype=torch.bfloat16, device="cuda")
    for out in ((k, k), (k, v[:, :1].expand(v.shape)), (k[:1].expand(k.shape), v), (wide[:, :, :2], wide[:, :, 1:]),
                (k, flat.as_strided(k.shape, (20 * 128, 128, 128, 1)))):
        with pytest.raises(ValueError, match="share memory"):
            pc.window(p, table, 3, 20, out=out)
    q = torch.randn(2, 3, 4, 128).bfloat16().cuda()
    with pytest.raises(ValueError, match="share memory"):
        pc.attend(q, p, table, lens, out=flat.as_strided(q.shape, (512, 256, 128, 1)))


def test_tensors_that_want_a_gradient_are_refused_both_ways():
    """requires_grad under grad mode, and forward-mode tangents, which grad mode does not switch off: in every argument,
    through the short path and the long one."""
    import torch.autograd.forward_ad as fwd
    from lingbot_b200 import paged_cache as pc, rope
    p = pool(P.make_pages(8, 4, 2, torch.int8))
    table, lens, t = i32([[0, 1], [2, 3]]), i32([100, 128]), rope.tables(64, 128)
    q = torch.randn(2, 3, 2, 128).bfloat16().cuda()

    def calls(x):
        return [lambda: pc.attend(x, p, table, lens), lambda: pc.attend(x, p, table, lens, out=torch.empty_like(q)),
                lambda: pc.write(p, table, 0, x, q), lambda: pc.write(p, table, 0, q, x, lens=2),
                lambda: rope.apply(x, t), lambda: rope.apply(q, t, k=x), lambda: rope.apply(x, t, out=torch.empty_like(q))]
    before = p.k.clone()
    for call in calls(q.clone().requires_grad_()):
        with pytest.raises(RuntimeError, match="gradient"):
            call()
    with fwd.dual_level():
        dual = fwd.make_dual(q, torch.ones_like(q))
        for mode in (torch.enable_grad, torch.no_grad):
            with mode():
                for call in calls(dual):
                    with pytest.raises(RuntimeError, match="tangent"):
                        call()
        assert torch.equal(pc.attend(fwd.unpack_dual(dual).primal, p, table, lens), pc.attend(q, p, table, lens))
    assert torch.equal(raw(p.k), raw(before))
    with torch.no_grad():
        for call in calls(q.clone().requires_grad_()):
            call()


def test_key_splits_follow_the_key_lengths_not_the_padding():
    """The same splits, so the same bits, with q_lens and without, and on the short path as on the long one; lengths as an
    int, or said to be alike, take the other rule's."""
    from lingbot_b200 import _lib, paged_cache as pc
    n, h, g = 16, 8, 4
    pages = P.make_pages(21, 16 * 40, h, torch.int8)
    p = pool(pages)
    table = torch.arange(n * 40, dtype=torch.int32).view(n, 40).cuda()
    q = torch.randn(n, 1, h * g, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    alike, unlike = (_lib.load().lbq_paged_attn_splits(n, 1, h, g, 2560, r) for r in (0, 1))
    assert alike != unlike
    lens, ones = torch.full((n,), 2560, dtype=torch.int32).cuda(), i32([1] * n)
    want = {r: pc.attend(q, p, table, lens, num_splits=s) for r, s in ((False, alike), (True, unlike))}
    assert not torch.equal(want[False], want[True])
    for kw, r in ((dict(), True), (dict(q_lens=ones), True), (dict(ragged=True), True), (dict(ragged=False), False),
                  (dict(q_lens=ones, ragged=False), False)):
        assert torch.equal(pc.attend(q, p, table, lens, **kw), want[r])
        assert torch.equal(pc.attend(q, p, table, lens, out=torch.empty_like(q), **kw), want[r])
    assert torch.equal(pc.attend(q, p, table, 2560), want[False])
    assert torch.equal(pc.attend(q, p, table, 2560, q_lens=ones, out=torch.empty_like(q)), want[False])


def test_sizes_that_pass_32_bits_are_refused():
    """Expanded dimensions of 2^32 + 5, which 32 bits would turn into 5."""
    from lingbot_b200 import paged_cache as pc, rope
    p = pool(P.make_pages(8, 4, 2, torch.int8))
    table, long = i32([[0, 1]]), (1 << 32) + 5
    k = torch.ones(1, 1, 2, 128, dtype=torch.bfloat16, device="cuda")
    before = p.k.clone()
    for call in (lambda: pc.write(p, table, 0, k.expand(1, long, 2, 128), k.expand(1, long, 2, 128)),
                 lambda: pc.write(p, table, 0, k.expand(1, long, 2, 128), k.expand(1, long, 2, 128), lens=5),
                 lambda: pc.write(p, table.expand(long, 2), 0, k.expand(long, 1, 2, 128), k.expand(long, 1, 2, 128)),
                 lambda: pc.attend(k.expand(1, long, 2, 128), p, table, 100),
                 lambda: pc.attend(k[:, :, :1].expand(1, 1, 2 * long, 128), p, table, 100),
                 lambda: pc.window(p, table, 0, long),
                 lambda: pc.window(p, table.expand(long, 2), 0, 5),
                 lambda: rope.apply(k.expand(1, long, 2, 128), rope.tables(64, 128))):
        with pytest.raises(ValueError, match="2.28"):
            call()
    assert torch.equal(raw(p.k), raw(before))


@pytest.mark.parametrize("lq", [3, 90], ids=["few", "many"])
def test_counts_past_the_given_tokens_are_recorded(lq):
    """q_lens and a write's lens outside [0, L] are cut to it, and recorded: the mask or the tokens are not what the caller
    meant. Counts at the ends are not."""
    from lingbot_b200 import _lib, paged_cache as pc
    p = pool(P.make_pages(8, 8, 2, torch.int8))
    table, lens = i32([[0, 1, 4], [2, 3, 5]]), i32([100, 128])
    q = torch.randn(2, lq, 2, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    for bad, as_if in (([lq + 1, 1], [lq, 1]), ([1, -1], [1, 0])):
        got = pc.attend(q, p, table, lens, q_lens=i32(bad), causal=True)
        assert _lib.device_status() == 0x305
        assert torch.equal(got, pc.attend(q, p, table, lens, q_lens=i32(as_if), causal=True))
        a, b = (pool(P.make_pages(8, 8, 2, torch.int8)) for _ in range(2))
        assert _lib.device_status() == 0
        pc.write(a, table, 10, q, q, lens=i32(bad))
        assert _lib.device_status() == 0x305
        pc.write(b, table, 10, q, q, lens=i32(as_if))
        assert _lib.device_status() == 0 and torch.equal(raw(a.k), raw(b.k)) and torch.equal(a.v_amax, b.v_amax)
