"""Decoder-step operators in 64 bits on the CPU (test infrastructure only): appending to the 8-bit
key/value cache, attention over it, and sampling, straight from their definitions in include/wbk.h.

The fp8 tables are oracle.fp8's; nothing here uses the library.
"""
from __future__ import annotations

import math

import numpy as np

from . import fp8

MIN_EXP = -64


def round_codes(values: np.ndarray, fmt: int) -> np.ndarray:
    """fp64 values (already divided by the scale) -> codes; NaN -> -max, infinities saturate."""
    mx = float(fp8.FMT_MAX[fmt])
    v = np.where(np.isnan(values), -mx, np.clip(values, -mx, mx))
    return fp8.encode_rne_satfinite(v.astype(np.float32), fmt)  # exact: at most 11 significant bits and a power of two


def scale_for(amax: float, fmt: int) -> float:
    """Least 2^E, E >= MIN_EXP, with amax <= max_fp8 * 2^E."""
    e = MIN_EXP
    mx = float(fp8.FMT_MAX[fmt])
    if amax > 0:
        e = max(MIN_EXP, math.frexp(amax / mx)[1] - 1)
        while amax > math.ldexp(mx, e):
            e += 1
    return math.ldexp(1.0, e)


def append_one(x: np.ndarray, codes: np.ndarray, scales: np.ndarray, table: np.ndarray, length: int, fmt: int) -> None:
    """x [H, n, D] appended behind `length` tokens of one sequence; codes [P, H, block, D] and scales [P, H] in place."""
    pages, heads, block, _ = codes.shape
    done, n = 0, x.shape[1]
    while done < n:
        blk, slot = divmod(length + done, block)
        count = min(block - slot, n - done)
        page = int(table[blk]) if blk < len(table) else -1
        if 0 <= page < pages:
            for h in range(heads):
                new = x[h, done:done + count].astype(np.float64)
                fine = np.abs(new[np.isfinite(new)])
                scale = scale_for(float(fine.max()) if fine.size else 0.0, fmt)
                if slot:
                    old = float(scales[page, h])
                    if scale > old:
                        held = fp8.decode(codes[page, h, :slot], fmt).astype(np.float64)
                        codes[page, h, :slot] = round_codes(held * (old / scale), fmt)
                    else:
                        scale = old
                codes[page, h, slot:slot + count] = round_codes(new / scale, fmt)
                scales[page, h] = scale
        done += count


def attention_one(q: np.ndarray, k: np.ndarray, v: np.ndarray, n: int, causal: bool, scale: float):
    """q [T, D], k and v [L, D] fp64 (masked-out tokens already removed); rows >= n are padding.
    Returns (out [T, D], sum_j p_j |v_j| [T, D])."""
    T, L = q.shape[0], k.shape[0]
    out, weight = np.zeros_like(q), np.zeros_like(q)
    for i in range(min(n, T)):
        vis = min(max(L - n + i + 1, 0), L) if causal else L
        if vis == 0:
            continue
        s = scale * (k[:vis] @ q[i])
        p = np.exp(s - s.max())
        p /= p.sum()
        out[i] = p @ v[:vis]
        weight[i] = p @ np.abs(v[:vis])
    return out, weight


def sample_one(logits: np.ndarray, noise: np.ndarray, temperature: float, top_k: int, top_p: float, min_p: float):
    """(token, logprob) of one row."""
    x = logits.astype(np.float64).copy()
    x[np.isnan(x)] = -np.inf
    x = np.minimum(x, float(np.finfo(np.float32).max))
    if x.max() == -np.inf:
        return -1, -math.inf
    top = x.max()
    logprob = (x - top) - math.log(np.exp(x - top).sum())
    order = np.lexsort((np.arange(x.size), -x))
    if temperature <= 0:
        return int(order[0]), float(logprob[order[0]])
    p = np.exp((x - top) / temperature)
    kept = order[: top_k if 0 < top_k < x.size else x.size]
    mass = np.cumsum(p[kept])
    before = np.concatenate([[0.0], mass[:-1]])
    ok = (p[kept] >= min_p) & (x[kept] > -np.inf)
    if top_p < 1:
        ok &= before < top_p * mass[-1]
    ok[0] = True
    kept = np.sort(kept[ok])
    score = p[kept] / np.maximum(noise[kept].astype(np.float64), 2.0 ** -126)
    token = int(kept[np.argmax(score)])
    return token, float(logprob[token])
