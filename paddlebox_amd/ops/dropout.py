"""Dropout whose mask is a function of (seed, offset, element) and is never stored.

Element ``i`` (row-major) takes 16 bits of Philox4x32-10 (Salmon et al.,
"Parallel random numbers: as easy as 1, 2, 3", 2011) with counter
``(i // 8, offset)`` and key ``seed``: half-word ``i % 8``, the low half of a
word first.  It is dropped iff they are under ``round(p * 2**16)``; ``p``
counts as that multiple of 2**-16.  The backward pass draws the same bits
again.

GPU tensors run ``csrc/hip/block_norm.hip``; the torch expressions here are
the CPU path and the reference the GPU tests compare against.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from .. import _native

Seed = Union[int, torch.Tensor]
_LOW = 0xFFFFFFFF


def wrap64(v: int) -> int:
    """v as a signed 64-bit value with the same bits."""
    v &= (1 << 64) - 1
    return v - (1 << 64) if v >> 63 else v


def mask_params(p: float, seed: Optional[Seed], offset: int, device: torch.device
                ) -> Tuple[int, Optional[torch.Tensor], int, int]:
    """(threshold, seed tensor or None, seed, offset) after the checks every
    user of the mask shares."""
    if isinstance(p, bool) or not isinstance(p, (int, float)) or not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout: p must be a number in [0, 1], not {p!r}")
    thr = round(p * 65536)
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or tuple(seed.shape) != (2,):
            raise ValueError("dropout: a seed tensor is int64 [2] = (seed, offset), "
                             f"not {seed.dtype} {list(seed.shape)}")
        if seed.device != device:
            raise ValueError(f"dropout: the seed tensor is on {seed.device}, the input on {device}")
        if offset:
            raise ValueError("dropout: a seed tensor holds the offset itself")
        return thr, seed.contiguous(), 0, 0
    if seed is None:
        if thr:
            raise ValueError("dropout: p > 0 needs a seed")
        seed = 0
    if isinstance(seed, bool) or not isinstance(seed, int) or isinstance(offset, bool) or not isinstance(offset, int):
        raise TypeError("dropout: seed and offset must be whole numbers, or seed an int64 tensor [2]")
    return thr, None, wrap64(seed), wrap64(offset)


def upscale(thr: int) -> float:
    """1 / (1 - p) of the threshold's p; 0 where nothing is kept."""
    return 65536.0 / (65536 - thr) if thr < 65536 else 0.0


def philox4x32(counter, key):
    """Ten rounds on four int64 tensors that hold 32-bit words -> four such tensors."""
    c, (k0, k1) = list(counter), key
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32 & _LOW) ^ c[1] ^ k0, p1 & _LOW, (p0 >> 32 & _LOW) ^ c[3] ^ k1, p0 & _LOW]
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    return c


def keep_mask(shape, thr: int, seed: Optional[torch.Tensor], seed_v: int, offset_v: int,
              device: torch.device) -> torch.Tensor:
    """The mask as booleans, in torch."""
    n = 1
    for s in shape:
        n *= s
    if thr == 0:
        return torch.ones(shape, dtype=torch.bool, device=device)
    s, o = (seed[0], seed[1]) if seed is not None else (torch.tensor(seed_v, device=device),
                                                       torch.tensor(offset_v, device=device))
    i = torch.arange((n + 7) // 8, dtype=torch.int64, device=device)
    z = torch.zeros_like(i)
    words = philox4x32([i & _LOW, i >> 32 & _LOW, z + (o & _LOW), z + (o >> 32 & _LOW)], (s & _LOW, s >> 32 & _LOW))
    bits = torch.stack([h for w in words for h in (w & 0xFFFF, w >> 16)], 1).reshape(-1)[:n]
    return (bits >= thr).reshape(shape)


def dropout(x: torch.Tensor, p: float, seed: Optional[Seed] = None, offset: int = 0, *, training: bool = True,
            mode: str = "upscale_in_train") -> torch.Tensor:
    """``x`` with each element dropped (set to zero, whatever it held) with
    probability ``p``.

    ``seed``: a whole number (with ``offset``, say the step and layer), or an
    int64 tensor [2] = (seed, offset) on x's device that the kernel reads, so
    that a captured graph draws a new mask whenever the program changes the
    tensor between replays.  The backward pass uses the values that the
    forward read.
    ``mode``: "upscale_in_train" scales kept values by 1 / (1 - p) in
    training, "downgrade_in_infer" scales by 1 - p at inference instead (the
    two of ``fluid.layers.dropout``).
    x: float32, bfloat16 or float16 of any shape; the result is contiguous.
    """
    if mode not in ("upscale_in_train", "downgrade_in_infer"):
        raise ValueError(f"dropout: unknown mode {mode!r}")
    if x.dtype not in (torch.float32, torch.bfloat16, torch.float16):
        raise TypeError(f"dropout: x must be float32, bfloat16 or float16, not {x.dtype}")
    thr, seed_t, seed_v, offset_v = mask_params(p, seed if training else 0, offset if training else 0, x.device)
    if not training:
        return x if mode == "upscale_in_train" else x * (1.0 - thr / 65536)
    up = upscale(thr) if mode == "upscale_in_train" else 1.0
    if x.is_cuda:
        return _native.hip().block_dropout(x, seed_t, thr, up, seed_v, offset_v)
    keep = keep_mask(x.shape, thr, seed_t, seed_v, offset_v, x.device)
    return torch.where(keep, x.float() * up, 0.0).to(x.dtype)
