"""The 4-bit cache and what works on it, in float64 and plain indexing (the kernels' tests compare with this)."""

from __future__ import annotations

import math

import torch

BLOCK = 16


def scale_grid() -> torch.Tensor:
    """Every scale a byte can hold, up to 8192: byte i is grid[i]."""
    out = [m * 2.0**-17 for m in range(8)]
    out += [(8 + m) * 2.0 ** (e - 18) for e in range(1, 29) for m in range(8)]
    return torch.tensor([x for x in out if x <= 8192], dtype=torch.float64)


def quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """x [..., d] (CPU) -> codes [..., d] 0..15 and scale bytes [..., d/16], as integers."""
    g = x.double().reshape(*x.shape[:-1], -1, BLOCK)
    g = torch.where(torch.isnan(g), 0.0, g)
    grid = scale_grid()
    want = (g.abs().amax(-1) / 7).clamp(max=8192.0)
    high = torch.searchsorted(grid, want).clamp(max=len(grid) - 1)
    low = (high - 1).clamp(min=0)
    down, up = want - grid[low], grid[high] - want
    byte = torch.where((down < up) | ((down == up) & (low % 2 == 0)), low, high)
    s = grid[byte][..., None]
    code = torch.where(s > 0, torch.round((g / torch.where(s > 0, s, 1.0)).clamp(-7, 7)), 0.0) + 8
    return code.long().flatten(-2), byte


def values_of(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    g = (codes - 8).double().reshape(*codes.shape[:-1], codes.shape[-1] // BLOCK, BLOCK)
    return (g * scale_grid().to(codes.device)[scales][..., None]).flatten(-2)


def pack(k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Rows k, v [n, d] (n a multiple of 16) of one head -> records [n/16, 18 d] uint8."""
    halves = []
    for x in (k, v):
        code, byte = quantise(x)
        both = code[:, 0::2] + 16 * code[:, 1::2]
        halves += [both.reshape(-1, BLOCK * both.shape[1]), byte.reshape(-1, BLOCK * byte.shape[1])]
    return torch.cat(halves, 1).to(torch.uint8)


def unpack(records: torch.Tensor, d: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Records [m, 18 d] -> keys and values [16 m, d] in float64."""
    out = []
    for o in (0, 9 * d):
        c = records[:, o : o + 8 * d].long().reshape(-1, d // 2)
        s = records[:, o + 8 * d : o + 9 * d].long().reshape(-1, d // BLOCK)
        out.append(values_of(torch.stack((c % 16, c // 16), -1).flatten(-2), s))
    return out[0], out[1]


def attention(q, keys, values, lens, window, sinks, scale):
    """q [T, nq, d] float64; keys/values: per request [nkv, n, d]; lens: (n, t) per request.
    Returns out [T, nq, d], lse [T, nq], weights (per request [nkv, n]), and two sizes that bound errors:
    spread [T, nq, d] = sum_j p_j |v_j|, and reach [T, nq] = scale max_j sum |q| |k_j|."""
    T, nq, d = q.shape
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((T, nq), -math.inf, dtype=torch.float64, device=q.device)
    reach = torch.zeros((T, nq), dtype=torch.float64, device=q.device)
    weights = []
    at = 0
    for (n, t), k, v in zip(lens, keys, values):
        nkv = k.shape[0]
        G = nq // nkv
        w = torch.zeros((nkv, n), dtype=torch.float64, device=q.device)
        for i in range(t):
            last = n - t + i
            first = max(0, last - window + 1) if window else 0
            if last < 0:
                seen = torch.arange(0, device=q.device)
            else:
                seen = torch.arange(first, last + 1, device=q.device)
            for h in range(nq):
                x = q[at + i, h]
                kk, vv = k[h // G][seen], v[h // G][seen]
                z = kk @ x * scale
                full = torch.cat((z, sinks[h : h + 1])) if sinks is not None else z
                if full.numel() == 0:
                    continue
                lse[at + i, h] = torch.logsumexp(full, 0)
                p = torch.exp(z - lse[at + i, h])
                out[at + i, h] = p @ vv
                spread[at + i, h] = p @ vv.abs()
                if seen.numel():
                    reach[at + i, h] = (kk.abs() @ x.abs()).max() * scale
                w[h // G][seen] += p
        weights.append(w)
        at += t
    return out, lse, weights, spread, reach


def kept_rows(weights: list[float], budget: int, recent: int, first: int) -> list[int]:
    """Which of a head's rows stay, in order."""
    n = len(weights)
    if n <= budget:
        return list(range(n))
    size = [math.inf if math.isnan(w) else w for w in weights]
    rank = [0 if math.isnan(w) else 1 for w in weights]
    middle = sorted(range(first, n - recent), key=lambda i: (rank[i], -size[i], i))[: budget - first - recent]
    return sorted([*range(first), *middle, *range(n - recent, n)])
