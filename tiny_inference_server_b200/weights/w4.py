"""Weights of four bits: codes 0..15 with a scale, and perhaps a zero point, per group of entries along the sum.

A weight of a (K, N) matrix is ``(code[k, n] - zero[k // group, n]) * scale[k // group, n]`` (zero 8 where no zero points are
kept).  ``quantize_w4`` finds codes by rounding to nearest, ``pack_w4`` lays codes out once as ``kernels.ops.gemm_w4`` streams
them, ``unpack_w4`` gives the matrix back (for products of many rows).

Layout.  Eight strips of 16 columns are a tile; the chunks of 64 entries of the sum follow one another in it, each with its strips' 512
bytes one after another.  A strip's 512 bytes of a chunk are 16 of each lane of a warp, which are
that lane's parts of four 16 x 16 operands of the tensor cores (columns as rows).  Lane (g, t) = (lane // 4, lane % 4) holds columns g
and g + 8; its word s the entries 16 s + 4 t + (0..3) of the chunk: bits 0-3 and 16-19 the first two of column g, 4-7 and 20-23 those
of column g + 8, 8-11 and 24-27 the last two of column g, 12-15 and 28-31 those of column g + 8.  So a shift and a mask give two
neighbouring entries in the halves of a register, and a lane's registers are what ``mma.sync`` takes and, in another order, what a
store of 16 lanes by 256 bits into tensor memory takes.  Scales and zero points lie as pairs (column g, column g + 8) by strip and group.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional, Tuple

import torch

STRIP, CHUNK, TILE_STRIPS = 16, 64, 8


@dataclass(frozen=True)
class W4Weights:
    """Codes in the kernel's layout: ``words`` (tiles, chunks, 8, 32, 4) int32, ``scales`` (strips, groups, 8, 2) bfloat16, ``zeros``
    the same in uint8 (None: 8 everywhere).  They are read 16, 4 and 2 bytes at a time and start on such a place: parts of one buffer are cut at
    multiples of 16 bytes."""
    words: torch.Tensor
    scales: torch.Tensor
    zeros: Optional[torch.Tensor]
    k: int
    n: int
    group: int

    def __post_init__(self):
        strips, groups = -(-self.n // STRIP), _groups(self.k, self.group)
        want = {"words": (torch.int32, (-(-strips // TILE_STRIPS), -(-self.k // CHUNK), TILE_STRIPS, 32, 4), 16),
                "scales": (torch.bfloat16, (strips, groups, 8, 2), 4), "zeros": (torch.uint8, (strips, groups, 8, 2), 2)}
        for name, (dtype, shape, start) in want.items():
            x = getattr(self, name)
            if x is None and name == "zeros":
                continue
            if x.dtype != dtype or tuple(x.shape) != shape or not x.is_contiguous() or x.device != self.words.device:
                raise ValueError(f"{name}: {x.dtype} {tuple(x.shape)} on {x.device}; contiguous {dtype} {shape} is wanted")
            if x.device.type != "meta" and x.data_ptr() % start:
                raise ValueError(f"{name}: starts on a multiple of {start} bytes, not at {x.data_ptr() % start} behind one")

    @property
    def shape(self) -> Tuple[int, int]:
        return self.k, self.n

    @property
    def device(self) -> torch.device:
        return self.words.device


def _groups(k: int, group: int) -> int:
    if group < 32 or group & (group - 1):
        raise ValueError(f"groups of {group} entries: a power of two from 32 on is wanted (one of K or more: a scale per column)")
    return -(-k // group)


def quantize_w4(w: torch.Tensor, group: int = 128, zeros: bool = False):
    """(codes (K, N) uint8, scales (groups, N) bfloat16, zeros (groups, N) uint8 or None) of a matrix, rounded to nearest: without zero
    points the largest entry of a group by size becomes 7 or -7 steps; with them the group's range, zero included, 15 steps."""
    if w.dim() != 2 or not w.is_floating_point() or 0 in w.shape:
        raise ValueError(f"a matrix of floating-point weights is wanted, not {w.dtype} {tuple(w.shape)}")
    k, n = w.shape
    groups = _groups(k, group)
    x = torch.zeros((groups * group, n), dtype=torch.float32, device=w.device)
    x[:k] = w
    if not bool(torch.isfinite(x).all()):                     # (no scale: the whole group would be lost)
        raise ValueError("weights that are not finite in float32")
    x = x.reshape(groups, group, n)
    if zeros:
        low, high = x.amin(1).clamp(max=0.0), x.amax(1).clamp(min=0.0)
        span = high - low                                     # (of the largest numbers of both signs: beyond float32)
        scales = torch.where(torch.isfinite(span), span / 15.0, high / 15.0 - low / 15.0).to(torch.bfloat16)
    else:
        scales = (x.abs().amax(1) / 7.0).to(torch.bfloat16)
    scales = torch.where(scales > 0, scales, 1.0).to(torch.bfloat16)        # (a group of zeros)
    step = scales.float()[:, None]
    zero = (-low / step[:, 0]).round().clamp(0, 15) if zeros else None
    codes = ((x / step).round() + (zero[:, None] if zeros else 8.0)).clamp(0, 15)
    return codes.to(torch.uint8).reshape(groups * group, n)[:k].contiguous(), scales, None if zero is None else zero.to(torch.uint8)


def _pairs(x: torch.Tensor) -> torch.Tensor:
    """(groups, N) by strip and group as pairs of the columns g and g + 8 (columns beyond N: zero)."""
    groups, n = x.shape
    strips = -(-n // STRIP)
    y = torch.zeros((groups, strips * STRIP), dtype=x.dtype, device=x.device)
    y[:, :n] = x
    return y.reshape(groups, strips, 2, 8).permute(1, 0, 3, 2).contiguous()


def pack_w4(codes: torch.Tensor, scales: torch.Tensor, zeros: Optional[torch.Tensor] = None, group: int = 128) -> W4Weights:
    """Lay codes (K, N) uint8 (0..15), scales (groups, N) bfloat16 and zero points (groups, N) uint8 (0..15; None: 8) out for ``gemm_w4``.  On the
    device they are there when it returns."""
    if codes.dim() != 2 or codes.dtype != torch.uint8 or 0 in codes.shape:
        raise ValueError(f"codes (K, N) in uint8 are wanted, not {codes.dtype} {tuple(codes.shape)}")
    k, n = codes.shape
    groups = _groups(k, group)
    if scales.dtype != torch.bfloat16 or tuple(scales.shape) != (groups, n):
        raise ValueError(f"scales {scales.dtype} {tuple(scales.shape)}: bfloat16 ({groups}, {n}) is wanted")
    if zeros is not None and (zeros.dtype != torch.uint8 or tuple(zeros.shape) != (groups, n)):
        raise ValueError(f"zero points {zeros.dtype} {tuple(zeros.shape)}: uint8 ({groups}, {n}) is wanted")
    if scales.device != codes.device or (zeros is not None and zeros.device != codes.device):
        raise ValueError("codes, scales and zero points lie on different devices")
    if int(codes.max()) > 15 or (zeros is not None and int(zeros.max()) > 15):
        raise ValueError("codes and zero points are 0..15")
    strips, chunks = -(-n // STRIP), -(-k // CHUNK)
    tiles = -(-strips // TILE_STRIPS)
    words = torch.empty((tiles, chunks, TILE_STRIPS, 32, 4), dtype=torch.int32, device=codes.device)
    for a in range(0, tiles, 128):                            # (in pieces: the working copies are several times the codes)
        b = min(a + 128, tiles)
        x = torch.zeros((chunks * CHUNK, (b - a) * TILE_STRIPS * STRIP), dtype=torch.uint8, device=codes.device)
        part = codes[:, a * TILE_STRIPS * STRIP:b * TILE_STRIPS * STRIP]
        x[:k, : part.shape[1]] = part
        # chunk, word s, t, pair i, entry e of the pair; tile, strip, column half c, g
        x = x.reshape(chunks, 4, 4, 2, 2, b - a, TILE_STRIPS, 2, 8)
        # tile, chunk, strip, g, t, s, e, i, c: nibble 4 e + 2 i + c
        x = x.permute(5, 0, 6, 8, 2, 1, 4, 3, 7).reshape(b - a, chunks, TILE_STRIPS, 32, 4, 4, 2)
        x = x[..., 0] | (x[..., 1] << 4)                      # bytes, the low nibble first
        words[a:b] = x.contiguous().view(torch.int32).squeeze(-1)
    w = W4Weights(words, _pairs(scales), None if zeros is None else _pairs(zeros), k, n, group)
    if words.is_cuda:                                         # (products read weights without waiting for the kernel in front of them)
        torch.cuda.current_stream(words.device).synchronize()
    return w


def unpack_w4(w: W4Weights, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The (K, N) matrix of packed weights: every weight worked out in 32 bits and rounded to ``dtype`` once."""
    tiles, chunks = w.words.shape[:2]
    x = w.words.contiguous().view(torch.uint8).reshape(tiles, chunks, TILE_STRIPS, 8, 4, 4, 4)
    x = torch.stack([x & 15, x >> 4], -1).reshape(tiles, chunks, TILE_STRIPS, 8, 4, 4, 2, 2, 2)         # tile, chunk, strip, g, t, s, e, i, c
    codes = x.permute(1, 5, 4, 7, 6, 0, 2, 8, 3).reshape(chunks * CHUNK, tiles * TILE_STRIPS * STRIP)[: w.k, : w.n]

    def rows(pairs):
        strips = pairs.shape[0]
        y = pairs.permute(1, 0, 3, 2).reshape(pairs.shape[1], strips * STRIP)[:, : w.n]
        return y.repeat_interleave(w.group, 0)[: w.k].float()

    zero = rows(w.zeros) if w.zeros is not None else 8.0
    return ((codes.float() - zero) * rows(w.scales)).to(dtype)
