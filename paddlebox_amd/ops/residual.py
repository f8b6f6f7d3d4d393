"""Gated residual connection with the norms before and after it, in one pass.

    u = norm_post(y)                             the block's output, normalised
    r = x_scale * x + y_scale * gate * drop(u)   the residual stream
    h = norm_pre(r)                              the next block's input

Memory bound, so fused: x, y (and a full gate) are read once, r and h written
once; the backward reads dr, dh, r and y once and redraws the dropout mask.
GPU tensors run ``csrc/hip/block_norm.hip``; the torch expressions here are
the CPU path and the reference the GPU tests compare against.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _native
from .dropout import Seed, keep_mask, mask_params, upscale

_KINDS = {"none": 0, "rms": 1, "layer": 2}
_TYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_COLUMNS = 16384
_NOT_GIVEN = object()  # a gate left out, as against gate=None


def _check_norm(name: str, kind: str, weight, bias, D: int, device):
    if kind not in _KINDS:
        raise ValueError(f"residual_norm: {name} must be one of {sorted(_KINDS)}, not {kind!r}")
    for part, t, need in (("weight", weight, kind != "none"), ("bias", bias, kind == "layer")):
        if (t is not None) != need:
            raise ValueError(f"residual_norm: {name}='{kind}' {'needs' if need else 'takes no'} {name}_{part}")
        if t is not None and (t.dtype != torch.float32 or tuple(t.shape) != (D,) or t.device != device):
            raise ValueError(f"residual_norm: {name}_{part} must be float32 [{D}] on {device}, "
                             f"not {t.dtype} {list(t.shape)} on {t.device}")


def _gate_kind(gate, act: str, y: torch.Tensor) -> int:
    """0 none, 1 [D], 2 [..., 1], 3 y's shape."""
    if act not in ("none", "sigmoid"):
        raise ValueError(f"residual_norm: gate_act must be 'none' or 'sigmoid', not {act!r}")
    if gate is _NOT_GIVEN and act != "none":
        raise ValueError("residual_norm: gate_act without a gate")
    if gate is None or gate is _NOT_GIVEN:
        return 0
    if gate.device != y.device:
        raise ValueError(f"residual_norm: the gate is on {gate.device}, the input on {y.device}")
    D = y.shape[-1]
    if gate.dim() == 1 and gate.shape[0] == D and (y.dim() > 1 or gate.dtype == torch.float32):
        kind, dtype = 1, torch.float32
    elif gate.shape == y.shape and not (D == 1 and gate.dtype == torch.float32 != y.dtype):
        kind, dtype = 3, y.dtype
    elif gate.shape == y.shape[:-1] + (1,):
        kind, dtype = 2, torch.float32
    else:
        raise ValueError(f"residual_norm: a gate has shape [{D}], {list(y.shape[:-1]) + [1]} or {list(y.shape)}, "
                         f"not {list(gate.shape)}")
    if gate.dtype != dtype:
        raise ValueError(f"residual_norm: a gate of shape {list(gate.shape)} must be {dtype}, not {gate.dtype}")
    return kind


def _norm(v, kind, weight, bias, eps):
    if kind == "none":
        return v
    c = v - v.mean(-1, keepdim=True) if kind == "layer" else v
    n = c / torch.sqrt((c * c).mean(-1, keepdim=True) + eps) * weight
    return n + bias if bias is not None else n


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, x_scale: float = 1.0, y_scale: float = 1.0,
                  gate: Optional[torch.Tensor] = _NOT_GIVEN, gate_act: str = "none",
                  post: str = "none", post_weight: Optional[torch.Tensor] = None,
                  post_bias: Optional[torch.Tensor] = None,
                  pre: str = "rms", pre_weight: Optional[torch.Tensor] = None,
                  pre_bias: Optional[torch.Tensor] = None, eps: float = 1e-6,
                  p: float = 0.0, seed: Optional[Seed] = None, offset: int = 0
                  ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """(r, h) of the module's formulas; h is None with ``pre="none"``.

    x, y: [..., D] of one shape, D <= 16384, at most 2**31 - 1 rows.  y is
    float32, bfloat16 or float16; x (the stream) has y's type or is float32,
    and r is like x, h like y.
    ``post`` / ``pre``: "none", "rms" (weight) or "layer" (weight and bias);
    weights and biases are float32 [D].
    ``gate``: None, float32 [D] (a value for each channel), float32 [..., 1]
    (one for each row) or y's shape and type; ``gate_act="sigmoid"`` takes its
    sigmoid.  A caller whose gate is optional passes ``gate=None`` with its
    ``gate_act``: no gate, nothing to activate.  ``gate_act`` with the gate left
    out is refused.
    ``p``, ``seed``, ``offset``: dropout on the normalised branch, as
    ``ops.dropout.dropout`` has it (pass p = 0 at inference).
    Differentiable once, in x, y, gate, weights and biases.
    """
    if x.dim() < 1 or x.shape != y.shape:
        raise ValueError(f"residual_norm: x {list(x.shape)} and y {list(y.shape)} must have one shape")
    if y.dtype not in _TYPES or x.dtype not in (y.dtype, torch.float32):
        raise TypeError("residual_norm: y must be float32, bfloat16 or float16 and x y's type or float32, "
                        f"not {x.dtype} and {y.dtype}")
    if x.device != y.device:
        raise ValueError(f"residual_norm: x is on {x.device}, y on {y.device}")
    D = x.shape[-1]
    if D < 1 or D > MAX_COLUMNS:
        raise ValueError(f"residual_norm: 1 to {MAX_COLUMNS} columns, not {D}")
    if x.numel() // D >= 1 << 31:
        raise ValueError("residual_norm: too many rows")
    if eps < 0:
        raise ValueError("residual_norm: eps must not be negative")
    _check_norm("post", post, post_weight, post_bias, D, x.device)
    _check_norm("pre", pre, pre_weight, pre_bias, D, x.device)
    kind = _gate_kind(gate, gate_act, y)
    if kind == 0:
        gate, gate_act = None, "none"
    thr, seed_t, seed_v, offset_v = mask_params(p, seed, offset, x.device)
    up = upscale(thr)
    if x.is_cuda:
        out = _native.hip().block_residual(x, y, gate, post_weight, post_bias, pre_weight, pre_bias, seed_t,
                                           _KINDS[post], _KINDS[pre], kind, gate_act == "sigmoid", x_scale, y_scale,
                                           eps, thr, up, seed_v, offset_v)
        return (out[0], out[1]) if pre != "none" else (out[0], None)
    f = torch.float32
    u = _norm(y.to(f), post, post_weight, post_bias, eps)
    if thr:
        u = torch.where(keep_mask(u.shape, thr, seed_t, seed_v, offset_v, u.device), u * up, 0.0)
    if gate is not None:
        g = gate.to(f)
        u = (torch.sigmoid(g) if gate_act == "sigmoid" else g) * u
    r = x_scale * x.to(f) + y_scale * u
    h = _norm(r, pre, pre_weight, pre_bias, eps) if pre != "none" else None
    return r.to(x.dtype), (h.to(y.dtype) if h is not None else None)
