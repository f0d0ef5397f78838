"""64-bit oracles of the epilogue, dropout and routing operators (test infrastructure only)."""

from __future__ import annotations

import math

import numpy as np
import torch

ACTIVATIONS = [None, "relu", "relu2", "silu", "gelu", "gelu_tanh"]


def philox4x32_10(counter: np.ndarray, key: tuple[int, int]) -> np.ndarray:
    """(n, 4) uint32 counters -> (n, 4) uint32 words (Salmon et al., SC 2011)."""
    c = [counter[:, i].astype(np.uint64) for i in range(4)]
    k0, k1 = key
    mask, sh = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> sh) ^ c[1] ^ np.uint64(k0), b & mask, (a >> sh) ^ c[3] ^ np.uint64(k1), a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, 1).astype(np.uint32)


def threshold(p: float) -> int:
    return math.floor(p * 65536 + 0.5)


def kept(shape, p: float, seed: int, device="cpu") -> torch.Tensor:
    n = math.prod(shape)
    g = np.arange((n + 7) // 8, dtype=np.uint64)
    ctr = np.zeros((g.size, 4), dtype=np.uint32)
    ctr[:, 0], ctr[:, 1] = g & np.uint64(0xFFFFFFFF), g >> np.uint64(32)
    s = seed & 0xFFFFFFFFFFFFFFFF
    words = philox4x32_10(ctr, (s & 0xFFFFFFFF, s >> 32))
    draws = np.stack([words & 0xFFFF, words >> 16], -1).reshape(-1)[:n]
    return torch.from_numpy(draws >= threshold(p)).reshape(shape).to(device)


def drop(x: torch.Tensor, p: float, seed: int) -> torch.Tensor:
    """x (float64) with dropout; a dropped element is 0 whatever it was."""
    if p == 0:
        return x
    t = threshold(p)
    scaled = x * (65536 / (65536 - t)) if t < 65536 else x
    return torch.where(kept(x.shape, p, seed, x.device), scaled, torch.zeros_like(x))


def activation(z: torch.Tensor, name: str | None) -> torch.Tensor:
    if name == "relu":
        return z.clamp_min(0)
    if name == "relu2":
        return z.clamp_min(0) ** 2
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    if name == "gelu_tanh":
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def derivative(z: torch.Tensor, name: str | None) -> torch.Tensor:
    """The formulas' derivatives (float64), written out."""
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "relu2":
        return 2 * z.clamp_min(0)
    if name == "silu":
        s = torch.sigmoid(z)
        return s + z * s * (1 - s)
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        th = torch.tanh(a * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + th) + 0.5 * z * (1 - th * th) * a * (1 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def half_step(dtype: torch.dtype) -> float:
    """The largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


def route(logits, k, bias=None, valid=None, renormalize=True):
    """One token at a time, on the CPU: (weights f64, experts, counts, offsets, rows, loss f64, prob f64)."""
    x32 = logits.detach().float().cpu().numpy()
    t, e = x32.shape
    b = np.zeros(e, np.float32) if bias is None else bias.detach().float().cpu().numpy()
    live = np.ones(t, bool) if valid is None else valid.cpu().numpy()
    weights, experts = np.zeros((t, k)), -np.ones((t, k), np.int64)
    prob = np.zeros((t, e))
    for i in range(t):
        if not live[i]:
            continue
        score = x32[i] + b  # fp32
        order = sorted(range(e), key=lambda j: (not np.isnan(score[j]), -score[j] if not np.isnan(score[j]) else 0.0, j))
        picks = [j for j in order if not score[j] == -np.inf][:k]
        if not picks:
            continue
        x = x32[i].astype(np.float64)
        z = np.exp(x - x.max())
        prob[i] = z / z.sum()
        w = prob[i][picks]
        if renormalize:
            zz = np.exp(x[picks] - x[picks].max())
            w = zz / zz.sum()
        weights[i, :len(picks)] = w
        experts[i, :len(picks)] = picks
    counts = np.bincount(experts[experts >= 0], minlength=e)
    offsets = np.concatenate([[0], np.cumsum((counts + 127) // 128 * 128)])
    rows = -np.ones((t, k), np.int64)
    fill = offsets[:-1].copy()
    for i in range(t):
        for j in range(k):
            if experts[i, j] >= 0:
                rows[i, j] = fill[experts[i, j]]
                fill[experts[i, j]] += 1
    n = int((experts[:, 0] >= 0).sum())
    loss = e * float((counts / max(1, counts.sum()) * prob.sum(0)).sum()) / n if n else 0.0
    return weights, experts, counts, offsets, rows, loss, prob


def route_gradient(weights, experts, counts, prob, grad_w, grad_loss, renormalize=True):
    """d (sum weights * grad_w + grad_loss * loss) / d logits, float64 numpy."""
    t, e = prob.shape
    n = int((experts[:, 0] >= 0).sum())
    c = grad_loss * e * (counts / max(1, counts.sum())) / max(1, n)
    g = prob * (c - (prob * c).sum(1, keepdims=True))
    for i in range(t):
        on = experts[i] >= 0
        if not on.any():
            g[i] = 0
            continue
        w, gw, at = weights[i][on], grad_w[i][on], experts[i][on]
        if renormalize:
            g[i, at] += w * (gw - (w * gw).sum())
        else:
            g[i, at] += w * gw
            g[i] -= prob[i] * (w * gw).sum()
    return g
