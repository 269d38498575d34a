"""Rotary positions on sm_100a (lbq_rope): neighbouring (2i, 2i+1) or half (i, i + rot/2) pairs, any leading part of the
head, tables stretched for long contexts.

The reference ropes a chunk's interleaved pairs by fp64 tables of its own (frame, row, column) grid
(models/lingbot_world/transformer.py:53-76, 134-146); the fused producers keep that form (`kv_cache.write(rope=)`). The
tables here are fp32 rows by position, shared by any number of sessions and by `paged_cache.write(rope=)`.
"""
from __future__ import annotations

import torch

from . import _lib

__all__ = ["Rope", "tables", "apply"]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POS = (torch.int32, torch.int64)


class Rope:
    """Rotary tables: cos, sin f32 [positions, rot / 2] on the GPU, rot the rotated channels of a head."""

    def __init__(self, cos, sin, interleaved=True):
        self.cos, self.sin, self.interleaved = cos, sin, interleaved
        r = _lib.fast().rope_table(cos, sin, interleaved)
        if r is None:
            self._refuse()
        self.rot, self._dev, self._args = r

    def _refuse(self):
        c, s = self.cos, self.sin
        if not (c.dtype == s.dtype == torch.float32 and c.dim() == 2 and c.shape == s.shape and c.stride() == s.stride()
                and c.stride(1) == 1 and c.device == s.device):
            raise ValueError("rope tables: two float32 [positions, rot / 2] tensors of one device and layout with unit "
                             f"last stride, got {c.dtype} {tuple(c.shape)} and {s.dtype} {tuple(s.shape)}")
        raise ValueError("rope tables must be CUDA tensors")

    def args(self, positions, device, b, l):
        """The table and position arguments of the C ABI, for tokens [b, l]."""
        if self.cos.device != device:
            raise ValueError(f"rope tables on {self.cos.device}, tensors on {device}")
        if positions is None:
            return (*self._args, None, 0, 0, 0)
        dt = positions.dtype
        if dt not in _POS or positions.device != device:
            raise TypeError("positions must be an int32 or int64 tensor on the tensors' device")
        shape = tuple(positions.shape)
        if shape == (b, l):
            sb, sl = positions.stride()
        elif shape == (l,) or shape == (1, l):
            sb, sl = 0, positions.stride(-1)
        else:
            raise ValueError(f"positions {shape} for tokens {(b, l)}")
        return (*self._args, positions.data_ptr(), 1 if dt is torch.int64 else 0, sb, sl)


def tables(num_positions, rot, base=10000.0, scaling=None, device="cuda", interleaved=True) -> Rope:
    """Tables of positions 0 .. num_positions - 1 for frequencies base^(-2i / rot), angles in 64 bits. `scaling`
    stretches them for contexts longer than the model was trained on:
      {"type": "linear", "factor": f}     positions divided by f
      {"type": "ntk", "factor": f}        base * f^(rot / (rot - 2)): the slowest frequency is divided by f
      {"type": "banded", "factor": f, "original": n, "low": a, "high": b}
                                          frequencies that turn fewer than a times over n positions divided by f, more
                                          than b times unchanged, blended linearly between
    """
    if rot <= 0 or rot % 2:
        raise ValueError(f"rot {rot} must be positive and even")
    if num_positions <= 0:
        raise ValueError(f"num_positions {num_positions} must be positive")
    kind = None if scaling is None else scaling.get("type")
    factor = 1.0 if scaling is None else float(scaling.get("factor", 0.0))
    if factor < 1.0:
        raise ValueError(f"rope scaling factor {factor} must be at least 1")
    if kind == "ntk":
        if rot == 2:
            raise ValueError("ntk scaling needs rot > 2")
        base = base * factor ** (rot / (rot - 2))
    freq = float(base) ** (-torch.arange(0, rot, 2, dtype=torch.float64, device=device) / rot)
    if kind == "linear":
        freq = freq / factor
    elif kind == "banded":
        low, high = float(scaling["low"]), float(scaling["high"])
        if not high > low:
            raise ValueError(f"banded scaling needs high > low, got {low}, {high}")
        turns = float(scaling["original"]) * freq / (2 * torch.pi)
        keep = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq / factor * (1 - keep) + freq * keep
    elif kind not in (None, "ntk"):
        raise ValueError(f"rope scaling type {kind!r}: expected linear, ntk or banded")
    ang = torch.arange(num_positions, dtype=torch.float64, device=device)[:, None] * freq[None, :]
    return Rope(ang.cos().float(), ang.sin().float(), interleaved)


def _check(name, x):
    if not x.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the kernels have no CPU implementation)")
    if x.dtype not in _DTYPES:
        raise TypeError(f"{name} must be bfloat16, float16 or float32, got {x.dtype}")
    if x.dim() != 4 or x.stride(3) != 1:
        raise ValueError(f"{name} must be [B, L, heads, dim] with unit channel stride, got {tuple(x.shape)}")
    _lib.check_sizes(name, x)


def _check_out(name, x, out):
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or (out.numel() and out.stride(3) != 1):
        raise ValueError(f"{name} out: {out.dtype} {tuple(out.shape)} does not match {x.dtype} {tuple(x.shape)}")
    same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
    if not same and out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr():
        raise ValueError(f"{name} out shares memory with its input without being it")
    if _lib.self_overlap(out):
        raise ValueError(f"{name} out has elements that share memory")


def apply(x, rope: Rope, positions=None, start=0, inverse=False, out=None, k=None, k_out=None):
    """Rotates the first rope.rot channels of every head of x [B, L, heads, dim] (bf16, fp16 or fp32; any strides with
    unit channel stride) by the table rows `positions` ([B, L] or [L], int32 / int64), or start + l. With `k` (the same
    B, L, dim and dtype, its own heads) both are rotated in one launch, and (x', k') is returned. out=x rotates in
    place. inverse=True turns back: apply(grad, ..., inverse=True) is the gradient."""
    if out is None and k_out is None:
        r = _lib.fast().rope(x, k, rope._args, rope._dev, positions, start, inverse)
        if r is not None:
            if type(r) is int:
                _lib.check("lbq_rope", r)
            return r
    _check("x", x)
    b, l, h, d = x.shape
    dev = x.device
    # (the gradient of the rotated tensor is rotated back with inverse=True)
    _lib.no_gradient("rope.apply", x, *(() if k is None else (k,)))
    start = int(start)
    if not 0 <= start < 1 << 62:
        raise ValueError(f"start {start} must be a non-negative 64-bit position")
    if (out is None) != (k_out is None) and k is not None:
        raise ValueError("out and k_out: give both or neither")
    if out is None:
        y = torch.empty_like(x)
    else:
        _check_out("x", x, out)
        y = out
    sx, sy = x.stride(), y.stride()
    table = rope.args(positions, dev, b, l)
    if k is None:
        if b and l and h:
            _lib.call_on(dev, "lbq_rope", x.data_ptr(), sx[0], sx[1], sx[2], y.data_ptr(), sy[0], sy[1], sy[2], h, None, 0, 0,
                         0, None, 0, 0, 0, 0, b, l, d, *table, start, 1 if inverse else 0, _DTYPES[x.dtype])
        return y
    _check("k", k)
    kb, kl, hk, kd = k.shape
    if kb != b or kl != l or kd != d or k.dtype != x.dtype or k.device != dev:
        raise ValueError(f"k {k.dtype} {tuple(k.shape)} does not go with x {x.dtype} {tuple(x.shape)}")
    if k_out is None:
        z = torch.empty_like(k)
    else:
        _check_out("k", k, k_out)
        z = k_out
        if h and hk and (y.data_ptr() == k.data_ptr() or z.data_ptr() == x.data_ptr()):
            raise ValueError("out and k_out are swapped: each is written while the other's input is read")
        if _lib.share_memory(y, z) or _lib.share_memory(y, k) or _lib.share_memory(z, x):
            raise ValueError("out and k_out share memory with one another or with the other's input")
    if not (h and hk):
        raise ValueError(f"x with {h} heads and k with {hk}: rotate the one that has heads alone")
    if b and l:
        sk, sz = k.stride(), z.stride()
        _lib.call_on(dev, "lbq_rope", x.data_ptr(), sx[0], sx[1], sx[2], y.data_ptr(), sy[0], sy[1], sy[2], h, k.data_ptr(),
                     sk[0], sk[1], sk[2], z.data_ptr(), sz[0], sz[1], sz[2], hk, b, l, d, *table, start,
                     1 if inverse else 0, _DTYPES[x.dtype])
    return y, z
