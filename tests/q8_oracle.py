"""Plain restatement of the 8-bit cache in 64 bits on the CPU, and the error bounds its tests use."""
from __future__ import annotations

import math
from dataclasses import dataclass, field

import torch

TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


def quantise(rows: torch.Tensor, fmt: str):
    """fp16 block [B, D] -> codes and fp32 scale, by the documented formula (fp32 division, round to nearest even)."""
    x = rows.float()
    top = x.abs().max()
    if not math.isfinite(float(top)):
        return torch.zeros(rows.shape, dtype=torch.uint8).view(CODE[fmt]), torch.tensor(float("nan"))
    scale = top * torch.tensor(1.0 / TOP[fmt], dtype=torch.float32)
    if float(scale) == 0.0:
        return torch.zeros(rows.shape, dtype=torch.uint8).view(CODE[fmt]), scale
    y = x / scale
    if fmt == "int8":
        return torch.round(y).to(torch.int8), scale
    return y.clamp(-448, 448).to(torch.float8_e4m3fn), scale


def dequantise(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    return codes.float().double() * scale.double()


@dataclass
class Sequence:
    """fp16 rows [T, NKV, D] of K and V as they were written."""
    k: torch.Tensor
    v: torch.Tensor
    kept: list = field(default_factory=list)   # logical pages that an eviction left, in order (empty: all)


def cached(rows: torch.Tensor, block: int, fmt: str) -> torch.Tensor:
    """What the cache stands for: [T, NKV, D] in 64 bits, complete blocks through their codes, the rest as it is."""
    t, nkv, d = rows.shape
    out = rows.double().clone()
    for b in range(t // block):
        for h in range(nkv):
            codes, scale = quantise(rows[b * block:(b + 1) * block, h], fmt)
            out[b * block:(b + 1) * block, h] = dequantise(codes, scale)
    return out


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0, scale: float | None = None):
    """q [n, NH, D] of the last n tokens, k and v [T, NKV, D] in 64 bits -> out, weights [n, NH, T] and a bound.

    The bound on |kernel - out| counts: probabilities rounded to fp16 for the product with V (half a step, 2^-11 of
    each), those below fp16's normal range (half a subnormal step, 2^-25, under the kernel's headroom of 2^6 and V's
    power-of-two reference, at most twice V's largest value), fp32 accumulation of q.k over D terms (each score off by
    at most (D + 4) 2^-24 sum|q k|, which moves a weight by that relative amount, numerator and denominator alike) and
    the approximate exponential and the sums (2^-18 for up to 2^16 tokens' accumulation errors, which average out)."""
    n, nh, d = q.shape
    t, nkv, _ = k.shape
    qpk = nh // nkv
    scale = 1.0 / math.sqrt(d) if scale is None else scale
    out = torch.zeros((n, nh, d), dtype=torch.float64)
    bound = torch.zeros_like(out)
    weights = torch.zeros((n, nh, t), dtype=torch.float64)
    pos = torch.arange(t)
    for i in range(n):
        at = t - n + i
        seen = pos <= at
        if window:
            seen = seen & ((pos < sinks) | (pos > at - window))
        seen = seen.nonzero()[:, 0]
        if seen.numel() == 0:
            continue
        for h in range(nh):
            kk, vv, qq = k[seen, h // qpk], v[seen, h // qpk], q[i, h].double()
            s = (kk @ qq) * scale
            w = torch.softmax(s, 0)
            weights[i, h, seen] = w
            out[i, h] = w @ vv
            worst = float(((kk.abs() @ qq.abs()) * scale).max())
            rel = 2 * (d + 4) * 2.0 ** -24 * worst + 2.0 ** -18
            bound[i, h] = (2.0 ** -11 + rel) * (w @ vv.abs()) + rel * out[i, h].abs() + seen.numel() * 2.0 ** -30 * vv.abs().max()
    return out, weights, bound


def attend_block(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, window: int = 0, sinks: int = 0, products: int = 2,
                 bias: float = 0.0):
    """``attend`` for many tokens at once, on the device of its inputs: out and the bound. ``products`` 1: the kernel
    rounds the probabilities to fp16 (2^-11 each); 2: it keeps what that leaves in a second product, whose own rounding
    is 2^-22. ``bias``: largest magnitude that a score's codes are shifted by in the product and back in fp32, as a
    multiple of sum|q| (128 K scales for int8): it is part of the sum whose fp32 accumulation counts."""
    n, nh, d = q.shape
    t, nkv, _ = k.shape
    qpk = nh // nkv
    scale = 1.0 / math.sqrt(d)
    out, bound = torch.zeros((2, n, nh, d), dtype=torch.float64, device=q.device)
    pos, me = torch.arange(t, device=q.device), torch.arange(t - n, t, device=q.device)[:, None]
    seen = pos <= me
    if window:
        seen &= (pos < sinks) | (pos > me - window)
    for h in range(nh):
        kk, vv, qq = k[:, h // qpk], v[:, h // qpk], q[:, h].double()
        s = (qq @ kk.T * scale).masked_fill(~seen, float("-inf"))
        w = torch.softmax(s, 1).masked_fill(~seen, 0.0)
        out[:, h] = w @ vv
        worst = (qq.abs() @ kk.abs().T * scale).masked_fill(~seen, 0.0).amax(1) + qq.abs().sum(1) * scale * bias
        rel = (2 * (d + 4) * 2.0 ** -24 * worst + 2.0 ** -18)[:, None]
        half = 2.0 ** -11 if products == 1 else 2.0 ** -22
        top = torch.where(seen[:, :, None], vv.abs(), 0.0).amax(1) if n * t * d < 1 << 27 else vv.abs().amax(0).expand(n, d)
        bound[:, h] = (half + rel) * (w @ vv.abs()) + rel * out[:, h].abs() + seen.sum(1)[:, None] * 2.0 ** -30 * top.amax(1, keepdim=True)
    return out, bound


def masses(weights: torch.Tensor, nkv: int, block: int) -> torch.Tensor:
    """[1, NH, T] weights of one token -> [NKV, pages]."""
    _, nh, t = weights.shape
    pages = -(-t // block)
    w = torch.nn.functional.pad(weights[0], (0, pages * block - t))
    return w.view(nkv, nh // nkv, pages, block).sum((1, 3))


def evict(full: int, mass: torch.Tensor, budget: int, first: int, recent: int) -> list[int]:
    """Logical pages that stay, in order; mass [NKV, >= full] fp32."""
    if full <= budget:
        return list(range(full))
    rank = mass.double().sum(0).float()
    fixed = [p for p in range(full) if p < first or p >= full - recent]
    rest = [p for p in range(full) if first <= p < full - recent]

    def key(p):
        x = float(rank[p])
        return (1, 0.0, p) if math.isnan(x) else (0, -x, p)

    return sorted(fixed + sorted(rest, key=key)[:budget - len(fixed)])
