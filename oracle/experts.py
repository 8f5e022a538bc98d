"""Routing to experts and the experts' MLPs, restated in float64 on the CPU, token by token."""

from __future__ import annotations

import math

import torch
from torch import Tensor


def scores(logits: Tensor, score: str, bias: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """Scores [T, E] (0 for masked experts) and which experts are not masked."""
    l = logits.double()
    ok = torch.isfinite(l)
    if bias is not None:
        ok = ok & torch.isfinite(bias.double())
    if score == "sigmoid":
        return torch.where(ok, torch.sigmoid(torch.where(ok, l, 0.0)), 0.0), ok
    low = torch.where(ok, l, -math.inf)
    return torch.softmax(low, dim=-1).nan_to_num(0.0), ok


def route(logits: Tensor, top_k: int, score: str = "softmax", bias: Tensor | None = None, groups: int = 1,
          top_groups: int = 1, renormalize: bool = True, scale: float = 1.0) -> tuple[Tensor, Tensor]:
    """``(weights, index)`` in float64 / int32 from logits [T, E]."""
    s, ok = scores(logits, score, bias)
    T, E = s.shape
    weights, index = torch.zeros(T, top_k, dtype=torch.float64), torch.full((T, top_k), -1, dtype=torch.int32)
    plain = bias is None and groups == 1
    for t in range(T):
        key = {e: float(logits[t, e]) if plain else float(s[t, e] + (bias[e].double() if bias is not None else 0.0))
               for e in range(E) if ok[t, e]}
        if groups > 1:
            per = E // groups
            rank = []
            for g in range(groups):
                best = sorted((key[e] for e in key if e // per == g), reverse=True)[:2]
                if best:
                    rank.append((-math.fsum(best), g))
            stay = {g for _, g in sorted(rank)[:top_groups]}
            key = {e: v for e, v in key.items() if e // per in stay}
        chosen = sorted(key, key=lambda e: (-key[e], e))[:top_k]
        w = torch.stack([s[t, e] for e in chosen]) if chosen else torch.zeros(0, dtype=torch.float64)
        if renormalize and float(w.sum()) > 0:
            w = w / w.sum()
        weights[t, : len(chosen)] = scale * w
        index[t, : len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return weights, index


def route_weights(logits: Tensor, index: Tensor, score: str, renormalize: bool, scale: float) -> Tensor:
    """The weights of a choice that is given, differentiable in the logits."""
    ok = torch.isfinite(logits)
    l = torch.where(ok, logits, 0.0)
    if score == "sigmoid":
        s = torch.where(ok, torch.sigmoid(l), 0.0)
    else:
        e = torch.where(ok, torch.exp(l), 0.0)
        s = e / e.sum(-1, keepdim=True).clamp_min(1e-300)
    have = index >= 0
    w = s.gather(-1, index.clamp_min(0).long()) * have
    if renormalize:
        total = w.sum(-1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    return scale * w


def gelu(z: Tensor) -> tuple[Tensor, Tensor]:
    """GELU(tanh) and its derivative."""
    c = math.sqrt(2 / math.pi)
    th = torch.tanh(c * (z + 0.044715 * z**3))
    return 0.5 * z * (1 + th), 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * c * (1 + 3 * 0.044715 * z * z)


def mlp(x: Tensor, weights: Tensor, index: Tensor, w1: Tensor, b1: Tensor | None, w2: Tensor, b2: Tensor | None,
        residual: Tensor | None) -> Tensor:
    """The definition, token by token: x [T, C], weights and index [T, k]."""
    rows = []
    for t in range(x.shape[0]):
        o = residual[t] if residual is not None else x.new_zeros(w2.shape[1])
        for s in range(index.shape[1]):
            e = int(index[t, s])
            if 0 <= e < w1.shape[0]:
                z = w1[e] @ x[t] + (b1[e] if b1 is not None else 0)
                o = o + weights[t, s] * (w2[e] @ gelu(z)[0] + (b2[e] if b2 is not None else 0))
        rows.append(o)
    return torch.stack(rows) if rows else x.new_zeros(0, w2.shape[1])


def mlp_bounds(x, weights, index, w1, b1, w2, b2, residual, dout=None) -> dict:
    """Every output and gradient in float64, by the formulas of the backward, each with a bound on
    what the bf16 operands and fp32 sums of a kernel may do to it: {name: (value, bound)}.

    u = 2^-24, v = 2^-8 (half a step of fp32 and bf16, relative).  A sum of n products in fp32 is off
    by at most n u of the sum of their magnitudes (any order), and its operands' own bounds are
    carried through; GELU and its derivative have slopes of at most 1.13 and 1.3 and are evaluated
    within 32 u of max(1, |z|); h (scaled by its pair's weight), gz and every output are rounded to
    bf16 once, gelu' to fp16 (v / 8, and 2^-24 below its normal numbers)."""
    u, v = 2.0**-24, 2.0**-8
    x, weights, w1, w2 = (a.double() for a in (x, weights, w1, w2))
    b1 = b1.double() if b1 is not None else None
    b2 = b2.double() if b2 is not None else None
    T, C = x.shape
    E, H, _ = w1.shape
    N, k = w2.shape[1], index.shape[1]
    out = torch.zeros(T, N, dtype=torch.float64)
    mag, bad = torch.zeros_like(out), torch.zeros_like(out)
    if residual is not None:
        out += residual.double()
        mag += residual.double().abs()
    res: dict = {}
    if dout is not None:
        g_all = dout.double()
        z64 = lambda *s: torch.zeros(*s, dtype=torch.float64)  # noqa: E731
        dx, dxm, dxb, dwt, dwtb = z64(T, C), z64(T, C), z64(T, C), z64(T, k), z64(T, k)
        dw1, dw1b, dw2, dw2b = z64(E, H, C), z64(E, H, C), z64(E, N, H), z64(E, N, H)
        db1, db1b, db2, db2b = z64(E, H), z64(E, H), z64(E, N), z64(E, N)
    for e in range(E):
        tok, slot = (index == e).nonzero(as_tuple=True)
        R = tok.numel()
        if not R:
            continue
        xe, a, b = x[tok], w1[e], w2[e]
        za = xe.abs() @ a.abs().T + (b1[e].abs() if b1 is not None else 0)
        z = xe @ a.T + (b1[e] if b1 is not None else 0)
        ez = (C + 2) * u * za
        h, d = gelu(z)
        eh0 = 1.13 * ez + 32 * u * z.abs().clamp_min(1)
        eh = eh0 + v * (h.abs() + eh0)
        y = h @ b.T + (b2[e] if b2 is not None else 0)
        ya = h.abs() @ b.abs().T + (b2[e].abs() if b2 is not None else 0)
        ey = eh @ b.abs().T + (H + 2) * u * (ya + eh @ b.abs().T)
        we = weights[tok, slot][:, None]
        out.index_add_(0, tok, we * y)
        mag.index_add_(0, tok, (we * y).abs())
        bad.index_add_(0, tok, we.abs() * ey)
        if dout is None:
            continue
        g = g_all[tok]
        dwt[tok, slot] = (g * y).sum(1)
        dwtb[tok, slot] = (g.abs() * ey).sum(1) + (N + 8) * u * (g * y).abs().sum(1)
        hs, ehs = we * h, we.abs() * (eh + u * h.abs())
        dw2[e] = g.T @ hs
        dw2b[e] = g.abs().T @ ehs + (R + 2) * u * (g.abs().T @ (hs.abs() + ehs))
        db2[e] = (we * g).sum(0)
        db2b[e] = (R + 2) * u * (we * g).abs().sum(0)
        gh, gha = g @ b, g.abs() @ b.abs()
        ed0 = 1.3 * ez + 32 * u * z.abs().clamp_min(1)
        ed = ed0 + v / 8 * (d.abs() + ed0) + u
        gz = we * gh * d
        egz0 = we.abs() * ((N + 4) * u * gha * (d.abs() + ed) + gh.abs() * ed)
        egz = egz0 + v * (gz.abs() + egz0)
        dw1[e] = gz.T @ xe
        dw1b[e] = egz.T @ xe.abs() + (R + 2) * u * ((gz.abs() + egz).T @ xe.abs())
        db1[e] = gz.sum(0)
        db1b[e] = egz.sum(0) + (R + 2) * u * (gz.abs() + egz).sum(0)
        r = gz @ a
        er0 = egz @ a.abs() + (H + 2) * u * ((gz.abs() + egz) @ a.abs())
        dx.index_add_(0, tok, r)
        dxm.index_add_(0, tok, r.abs())
        dxb.index_add_(0, tok, er0)
    half = lambda val, b: b + v * (val.abs() + b) + 1e-40  # noqa: E731  (the last rounding)
    res["out"] = (out, half(out, bad + (k + 2) * u * mag))
    if dout is not None:
        res["x"] = (dx, half(dx, dxb + (k + 1) * u * dxm))
        res["weights"] = (dwt, half(dwt, dwtb))
        res["w1"], res["w2"] = (dw1, half(dw1, dw1b)), (dw2, half(dw2, dw2b))
        if b1 is not None:
            res["b1"] = (db1, half(db1, db1b))
        if b2 is not None:
            res["b2"] = (db2, half(db2, db2b))
        if residual is not None:
            res["residual"] = (g_all, torch.zeros_like(g_all))
    return res
