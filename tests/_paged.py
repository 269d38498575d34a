"""Plain 64-bit evaluation of the paged 8-bit cache and of rotary positions, for the tests: loops over sequences, pages
and heads, straight from the formulas of include/lbq.h."""
import torch

PAGE = 64
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def values(codes):
    """Codes as float64."""
    return codes.cpu().view(codes.dtype).to(torch.float32).double()


def to_codes(x, fmt):
    """Float64 values within the format's range -> codes (half to even)."""
    return x.round().to(torch.int8) if fmt == torch.int8 else x.float().to(fmt)


def make_pages(seed, pages, heads, fmt, device="cpu", spread=1.0):
    """Random codes and amax; magnitudes differ from page to page by up to 2^spread."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        amax = 2.0 ** (spread * torch.rand(pages, heads, generator=g))
        x = torch.randn(pages, heads, PAGE, 128, generator=g) / 4.5
        out.append((to_codes((x.clamp(-1, 1) * TOP[fmt]).double(), fmt), amax))
    (k, ka), (v, va) = out
    return k.to(device), v.to(device), ka.to(device), va.to(device)


def make_table(seed, counts, pages, width=None):
    """Page table [B, width] with distinct pages, -1 past a sequence's own."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randperm(pages, generator=g).tolist()
    width = max(1, max(counts)) if width is None else width
    rows, at = [], 0
    for n in counts:
        rows.append(ids[at:at + n] + [-1] * (width - n))
        at += n
    return torch.tensor(rows, dtype=torch.int32)


def rotate(x, cos, sin, rows, interleaved, inverse=False):
    """x [B, L, H, D] in float64 by rows [B, L] of cos / sin [P, rot / 2]; also the magnitude sum |x0 c| + |x1 s| that
    bounds the rounding of each result."""
    c, s = cos.double()[rows][:, :, None], sin.double()[rows][:, :, None]
    if inverse:
        s = -s
    half = c.shape[-1]
    y, size = x.clone(), x.abs().clone()
    i0 = torch.arange(half) * 2 if interleaved else torch.arange(half)
    i1 = i0 + 1 if interleaved else i0 + half
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    size[..., i0], size[..., i1] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, size


def write(codes, amax, table, starts, counts, x, fmt):
    """One tensor's write, in place on CPU copies: codes [P, H, 64, 128], amax [P, H], x [B, L, H, 128]."""
    top = TOP[fmt]
    for b, (start, n) in enumerate(zip(starts, counts)):
        for blk in range(start // PAGE, (start + n + PAGE - 1) // PAGE if n else 0):
            page = int(table[b, blk])
            lo, hi = max(start, blk * PAGE), min(start + n, (blk + 1) * PAGE)
            held = lo - blk * PAGE
            for h in range(codes.shape[1]):
                part = x[b, lo - start:hi - start, h].double()
                finite = part[torch.isfinite(part)].abs()
                a = max(float(finite.max()) if finite.numel() else 0.0, 2.0 ** -40)
                if held:
                    old = float(amax[page, h])
                    a = max(a, old)
                    if a > old:
                        codes[page, h, :held] = to_codes(values(codes[page, h, :held]) * old / a, fmt)
                amax[page, h] = a
                q = torch.where(part.isnan(), torch.zeros_like(part), part * top / a).clamp(-top, top)
                codes[page, h, held:held + hi - lo] = to_codes(q, fmt)


def gather(codes, amax, row, n, fmt):
    """Values [n, H, 128] in float64 of a sequence's first n tokens."""
    pages = [int(p) for p in row[:(n + PAGE - 1) // PAGE]]
    if not pages:
        return torch.zeros(0, codes.shape[1], 128, dtype=torch.float64)
    v = values(codes[pages]) * (amax[pages].double() / TOP[fmt])[..., None, None]
    return v.permute(0, 2, 1, 3).reshape(-1, codes.shape[1], 128)[:n]


def attend(q, k, v, ka, va, table, kvs, qs, causal, scale=128 ** -0.5):
    """(out, lse, tolerance without the output's rounding) in float64. q [B, L, Hq, 128] on CPU.

    The tolerance follows the kernel's roundings. With W = sum p |v| (p normalised): weights rounded to fp16, 2^-11
    relative (half of fp16's step) each, and 2^-25 absolute below fp16's normal range; a score is off by at most
    e = 2^-19 max_j sum_d |q_d k_jd| scale (128 products in fp32, the query row held to 2^-25 of its maximum), which
    moves every weight by e relative, and the sum of the weights likewise."""
    b, lq, hq, _ = q.shape
    heads = k.shape[1]
    g = hq // heads
    fmt = k.dtype
    out = torch.zeros(b, lq, hq, 128, dtype=torch.float64)
    lse = torch.full((b, lq, hq), -torch.inf, dtype=torch.float64)
    tol = torch.zeros_like(out)
    for s, (kv, n) in enumerate(zip(kvs, qs)):
        kk, vv = gather(k, ka, table[s], kv, fmt), gather(v, va, table[s], kv, fmt)
        if kv == 0 or n == 0:
            continue
        for h in range(hq):
            x = q[s, :n, h].double() @ kk[:, h // g].T * scale
            size = q[s, :n, h].double().abs() @ kk[:, h // g].abs().T * scale
            if causal:
                x = x.masked_fill(torch.arange(kv)[None] > kv - n + torch.arange(n)[:, None], -torch.inf)
            top = x.amax(-1, keepdim=True)
            p = torch.exp(x - torch.where(top == -torch.inf, 0.0, top))
            l = p.sum(-1, keepdim=True)
            ll = torch.where(l == 0, 1.0, l)
            out[s, :n, h] = p @ vv[:, h // g] / ll
            lse[s, :n, h] = (top + torch.log(l))[:, 0]
            w = p @ vv[:, h // g].abs() / ll
            e = 2.0 ** -19 * size.amax(-1, keepdim=True) + 2.0 ** -20
            tol[s, :n, h] = w * (2.0 ** -11 + 2 * e) + 2.0 ** -25 * vv[:, h // g].abs().sum(0)[None] / ll
    return out, lse, tol
