"""Rotary positions on sm_100a (lbq_rope): neighbouring (2i, 2i+1) or half (i, i + rot/2) pairs, any leading part of the
head, tables stretched for long contexts.

The reference ropes a chunk's interleaved pairs by fp64 tables of its own (frame, row, column) grid
(models/lingbot_world/transformer.py:53-76, 134-146); the fused producers keep that form (`kv_cache.write(rope=)`). The
tables here are fp32 rows by position, shared by any number of sessions and by `paged_cache.write(rope=)`.
"""
from __future__ import annotations

from dataclasses import dataclass

import torch

from . import _lib

__all__ = ["Rope", "tables", "apply"]

_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_POS = (torch.int32, torch.int64)


@dataclass
class Rope:
    """Rotary tables: cos, sin f32 [positions, rot / 2] on the GPU, rot the rotated channels of a head."""
    cos: torch.Tensor
    sin: torch.Tensor
    interleaved: bool = True

    def __post_init__(self):
        c, s = self.cos, self.sin
        if c.dtype != torch.float32 or s.dtype != torch.float32 or c.dim() != 2 or c.shape != s.shape \
                or c.stride() != s.stride() or c.stride(1) != 1 or c.device != s.device:
            raise ValueError("rope tables: two float32 [positions, rot / 2] tensors of one device and layout with unit "
                             f"last stride, got {c.dtype} {tuple(c.shape)} and {s.dtype} {tuple(s.shape)}")
        if not c.is_cuda:
            raise ValueError("rope tables must be CUDA tensors")

    @property
    def rot(self):
        return 2 * self.cos.shape[1]

    def args(self, positions, device, shape):
        """The table and position arguments of the C ABI, for tokens of `shape` [B, L]."""
        if self.cos.device != device:
            raise ValueError(f"rope tables on {self.cos.device}, tensors on {device}")
        pos, pos64, sb, sl = None, 0, 0, 0
        if positions is not None:
            if positions.dtype not in _POS or positions.device != device:
                raise TypeError("positions must be an int32 or int64 tensor on the tensors' device")
            p = positions if positions.dim() == 2 else positions[None]
            if p.dim() != 2 or p.shape[1] != shape[1] or p.shape[0] not in (1, shape[0]):
                raise ValueError(f"positions {tuple(positions.shape)} for tokens {tuple(shape)}")
            pos, pos64 = p.data_ptr(), int(p.dtype == torch.int64)
            sb, sl = (p.stride(0) if p.shape[0] > 1 else 0), p.stride(1)
        return (self.cos.data_ptr(), self.sin.data_ptr(), self.cos.stride(0), self.cos.shape[0], self.rot,
                int(self.interleaved), pos, pos64, sb, sl)


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


def _output(name, x, out):
    """The tensor that takes x's result: `out` (x itself for in place), or a new one."""
    if out is None:
        return torch.empty(x.shape, dtype=x.dtype, device=x.device)
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device or (out.numel() and out.stride(3) != 1):
        raise ValueError(f"{name} out: {out.dtype} {tuple(out.shape)} does not match {x.dtype} {tuple(x.shape)}")
    same = out.data_ptr() == x.data_ptr() and out.stride() == x.stride()
    if not same and out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr():
        raise ValueError(f"{name} out shares memory with its input without being it")
    if any(n > 1 and s == 0 for n, s in zip(out.shape, out.stride())):
        raise ValueError(f"{name} out has elements that share memory")
    return out


def apply(x, rope: Rope, positions=None, start=0, inverse=False, out=None, k=None, k_out=None):
    """Rotates the first rope.rot channels of every head of x [B, L, heads, dim] (bf16, fp16 or fp32; any strides with
    unit channel stride) by the table rows `positions` ([B, L] or [L], int32 / int64), or start + l. With `k` (the same
    B, L, dim and dtype, its own heads) both are rotated in one launch, and (x', k') is returned. out=x rotates in
    place. inverse=True turns back: apply(grad, ..., inverse=True) is the gradient."""
    _check("x", x)
    b, l, h, d = x.shape
    if torch.is_grad_enabled() and (x.requires_grad or (k is not None and k.requires_grad)):
        raise RuntimeError("rope.apply records no gradient: call it under torch.no_grad(), and rotate the gradient back "
                           "with inverse=True")
    y = _output("x", x, out)
    k_args, y2 = (None, 0, 0, 0, None, 0, 0, 0, 0), None
    if k is not None:
        _check("k", k)
        if k.shape[:2] != x.shape[:2] or k.shape[3] != d or k.dtype != x.dtype or k.device != x.device:
            raise ValueError(f"k {k.dtype} {tuple(k.shape)} does not go with x {x.dtype} {tuple(x.shape)}")
        y2 = _output("k", k, k_out)
        if (out is None) != (k_out is None):
            raise ValueError("out and k_out: give both or neither")
        if h and k.numel() and (y.data_ptr() == k.data_ptr() or y2.data_ptr() == x.data_ptr()):
            raise ValueError("out and k_out are swapped: each is written while the other's input is read")
        if k.shape[2]:
            k_args = (k.data_ptr(), *k.stride()[:3], y2.data_ptr(), *y2.stride()[:3], k.shape[2])
    table = rope.args(positions, x.device, (b, l))
    if b and l and h:
        _lib.call_on(x.device, "lbq_rope", x.data_ptr(), *x.stride()[:3], y.data_ptr(), *y.stride()[:3], h, *k_args, b, l,
                     d, *table, int(start), int(bool(inverse)), _DTYPES[x.dtype])
    elif k is not None and b and l and k.shape[2]:
        raise ValueError("x has no heads: rotate k alone")
    return y if k is None else (y, y2)
