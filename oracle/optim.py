"""AdamW with clipping by the global norm, and the 8-bit moments, restated in float64 on the CPU."""

from __future__ import annotations

import math

import torch

BLOCK = 256


def pack(x: torch.Tensor, signed: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Codes of a moment, their blocks' scales (fp32), and how far each value's place between two
    codes is from the border where it would take the other one (in steps)."""
    n = x.numel()
    blocks = -(-n // BLOCK)
    flat = torch.zeros(blocks * BLOCK, dtype=torch.float64)
    flat[:n] = x.reshape(-1)
    b = flat.view(blocks, BLOCK)
    scale = b.abs().amax(1).float()
    safe = torch.where(scale > 0, scale, torch.ones_like(scale)).double()[:, None]
    place = torch.sqrt(b.abs() / safe) * (127 if signed else 256)
    code = torch.floor(place + 0.5)
    code = torch.where(b < 0, -1.0, 1.0) * code.clamp(0, 127) if signed else (code - 1).clamp(0, 255)
    border = (place - torch.floor(place) - 0.5).abs()
    codes = code.to(torch.int8 if signed else torch.uint8)
    return codes.view(-1)[:n].view(x.shape), scale, border.view(-1)[:n].view(x.shape)


def unpack(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    c = codes.reshape(-1).double()
    s = scale.double().repeat_interleave(BLOCK)[: c.numel()]
    r = c / 127 if codes.dtype == torch.int8 else (c + 1) / 256
    return (r * r.abs() * s).view(codes.shape)


def global_norm(grads) -> float:
    return math.sqrt(sum(float((g.double() ** 2).sum()) for g in grads))


def adamw(p, g, m, v, t, lr, betas, eps, decay, coef=1.0):
    """One step of one tensor (all float64): p, m, v after it."""
    g = g * coef
    m = betas[0] * m + (1 - betas[0]) * g
    v = betas[1] * v + (1 - betas[1]) * g * g
    mh, vh = m / (1 - betas[0] ** t), v / (1 - betas[1] ** t)
    return p - lr * decay * p - lr * mh / (vh.sqrt() + eps), m, v
