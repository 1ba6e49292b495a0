"""FP8 with fp32 scales per block of 128, on numpy and ml_dtypes (test infrastructure, not product).

Structure of the reference's block-scaled FP8 quantiser
(experiments/flashinfer-megamoe-sm90a/quant.py:47-75) with one fp32 scale per 1 x 128 or 128 x 128 block;
parity unpinned, the reference has no code for blocks of 128.
"""

from __future__ import annotations

import ml_dtypes
import numpy as np

TINY = np.float32(2.0 ** -126)


def block_scale(amax: np.ndarray) -> np.ndarray:
    return np.maximum(amax.astype(np.float32) / np.float32(448.0), TINY)


def _encode(x: np.ndarray, s: np.ndarray) -> np.ndarray:
    with np.errstate(invalid="ignore"):
        q = (x.astype(np.float32) / s).astype(np.float32)
    return np.clip(q, -448, 448).astype(ml_dtypes.float8_e4m3fn).view(np.uint8)


def _amax(x, axis):
    return np.where(np.isnan(x), 0, np.abs(x)).max(axis=axis)


def quantize_rows(x: np.ndarray):
    """(rows, k) -> (q (rows, k) bytes, sf (kblocks, rows))."""
    rows, k = x.shape
    q, sf = np.zeros((rows, k), np.uint8), np.zeros((-(-k // 128), rows), np.float32)
    for c in range(sf.shape[0]):
        part = x[:, 128 * c:128 * c + 128].astype(np.float32)
        sf[c] = block_scale(_amax(part, 1))
        q[:, 128 * c:128 * c + 128] = _encode(part, sf[c][:, None])
    return q, sf


def quantize_weight(w: np.ndarray):
    """(n, k) -> (q (n, k) bytes, sf (nblocks, kblocks))."""
    n, k = w.shape
    q, sf = np.zeros((n, k), np.uint8), np.zeros((-(-n // 128), -(-k // 128)), np.float32)
    for r in range(sf.shape[0]):
        for c in range(sf.shape[1]):
            part = w[128 * r:128 * r + 128, 128 * c:128 * c + 128].astype(np.float32)
            sf[r, c] = block_scale(_amax(part, None))
            q[128 * r:128 * r + 128, 128 * c:128 * c + 128] = _encode(part, sf[r, c])
    return q, sf


def silu_mul(gateup: np.ndarray) -> np.ndarray:
    """(rows, 2k) -> silu(gate) * up in float64."""
    x = gateup.astype(np.float64)
    k = x.shape[1] // 2
    return x[:, :k] / (1.0 + np.exp(-x[:, :k])) * x[:, k:]


def values(q: np.ndarray) -> np.ndarray:
    return q.view(ml_dtypes.float8_e4m3fn).astype(np.float64)


def dequantize_rows(q, sf):
    return values(q) * np.repeat(sf.T.astype(np.float64), 128, axis=1)[:q.shape[0], :q.shape[1]]


def dequantize_weight(q, sf):
    n, k = q.shape
    return values(q) * np.repeat(np.repeat(sf.astype(np.float64), 128, 0)[:n], 128, 1)[:, :k]


def product(a_q, a_sf, b_q, b_sf):
    """-> (y (m, n) float64, the sums of the magnitudes of its terms)."""
    a, b = dequantize_rows(a_q, a_sf), dequantize_weight(b_q, b_sf)
    return a @ b.T, np.abs(a) @ np.abs(b).T
