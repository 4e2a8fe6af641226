"""The 8-bit integer linear in 64 bits (numpy): a scale per token and per output
channel, exact integer sums."""

from __future__ import annotations

import numpy as np


def quantize(x: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
    """(codes int8 [M, K], scales fp32 [M]) of x [M, K]: scale = max|x| / 127 and codes
    rint(x / scale), both divisions in fp32. A row with an infinity or NaN: codes 0,
    scale NaN."""
    x = np.asarray(x, dtype=np.float32)
    top = np.abs(x).max(axis=1) if x.shape[1] else np.zeros(len(x), np.float32)
    bad = ~np.isfinite(x).all(axis=1)
    scale = np.where(bad, np.float32(np.nan), np.where(bad, 0, top) / np.float32(127)).astype(np.float32)
    some = scale > 0
    with np.errstate(all="ignore"):
        q = np.rint(x / np.where(some, scale, np.float32(1))[:, None])
    q = np.where(some[:, None], np.clip(q, -127, 127), 0)
    return q.astype(np.int8), scale


def linear(q: np.ndarray, scales: np.ndarray, w: np.ndarray, w_scales: np.ndarray) -> np.ndarray:
    """fp64 [M, N] of codes [M, K] and a weight [N, K]."""
    total = q.astype(np.float64) @ w.astype(np.float64).T  # whole numbers below 2^53
    return total * scales.astype(np.float64)[:, None] * w_scales.astype(np.float64)
