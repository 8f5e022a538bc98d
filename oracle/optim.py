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


NEWTON_SCHULZ = (3.4445, -4.7750, 2.0315)


def orthogonalize(x, coefficients=(NEWTON_SCHULZ,) * 5, eps=1e-7, precise=False):
    """Newton-Schulz products of one float64 matrix by its singular values, each of which goes through the polynomials by
    itself, and the Frobenius norm of the error that a kernel's roundings make.

    The error is followed in the basis of the singular vectors, E[i, j] with its variance: a step multiplies it by a
    divided difference of s -> a s + b s^3 + c s^5 at s_i and +-s_j, and adds that of its own roundings, each taken as evenly
    spread and independent: the operands' (half a step of fp16, 2^-11; of two fp16 2^-22, three times that with the
    product of the two lower halves left out), sums in fp32 of K / 16 + 16 roundings of at most the norms of what they multiply,
    the fp16 parts' absolute step under 2^-14 (X is held times 2^12, A and P times 2^10).  ``precise``: two fp16
    everywhere; otherwise for a X alone, in the first three steps."""
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    m, n = x.shape
    u, s, vt = torch.linalg.svd(x / max(float(torch.linalg.norm(x)), eps), full_matrices=False)
    half, two = 2.0**-11, 3 * 2.0**-22
    op, subx, suba = (two if precise else half), 2.0**-25 / 2**12, 2.0**-25 / 2**10
    norm = torch.linalg.norm
    summed = lambda k: math.sqrt(k / 16 + 16) * 2.0**-24  # noqa: E731
    kept = lambda k: precise or k < min(3, len(coefficients))  # noqa: E731  (X into step k, in the end the result, is two fp16)
    first = (two if kept(0) else half) * norm(s)
    E = torch.full((m, m), float(first) ** 2 / (m * n) + subx**2, dtype=torch.float64)
    rest = torch.full((m,), (n - m) * float(E[0, 0]), dtype=torch.float64)  # the n - m directions that x has not
    for k, (a, b, c) in enumerate(coefficients):
        lam = s * s
        p = b * lam + c * lam * lam
        f = a * s + p * s
        diff, plus = s[:, None] - s[None], s[:, None] + s[None]
        slope = a + 3 * b * lam + 5 * c * lam * lam
        near = (slope[:, None].abs() + slope[None].abs()) / 2
        L = torch.where(diff.abs() > 1e-9, (f[:, None] - f[None]) / diff.where(diff.abs() > 1e-9, torch.ones_like(diff)), near).abs()
        L = torch.maximum(L, torch.where(plus > 1e-12, (f[:, None] + f[None]) / plus.clamp_min(1e-12), torch.full_like(plus, abs(a))).abs())
        vx = (op * norm(s)) ** 2 / (m * n) + subx**2
        va = (lam[:, None] + lam[None]) * vx + ((op * norm(lam)) ** 2 + (summed(n) * norm(s) ** 2) ** 2) / m**2 + suba**2
        vp = (abs(b) + abs(c) * (lam[:, None] + lam[None])) ** 2 * va + \
            ((op * norm(p)) ** 2 + (abs(c) * summed(m) * norm(lam) ** 2) ** 2) / m**2 + suba**2
        s = f.abs()
        own = ((two if kept(k + 1) else half) * norm(f)) ** 2 / (m * n) + subx**2 + (summed(m) * norm(p) * norm(f)) ** 2 / (m * n)
        E = L**2 * E + p[:, None] ** 2 * vx + vp * lam[None] + own
        rest = (a + p) ** 2 * rest + (n - m) * (p**2 * vx + own)
        u = u * torch.sign(f).where(f != 0, torch.ones_like(f))
    out = u @ (s[:, None] * vt)
    return (out.T if tall else out), float((E.sum() + rest.sum()).sqrt())


def muon(p, g, m, lr, momentum=0.95, nesterov=True, decay=0.1, adjust="original", precise=False, **kw):
    """One step of one matrix (all float64): p, m after it, and the norm of the update's error (``orthogonalize``)."""
    rows, cols = p.shape
    m = momentum * m + (1 - momentum) * g
    o, off = orthogonalize(momentum * m + (1 - momentum) * g if nesterov else m, precise=precise, **kw)
    rate = lr * (0.2 * math.sqrt(max(rows, cols)) if adjust == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols)))
    return p * (1 - lr * decay) - rate * o, m, abs(rate) * off
