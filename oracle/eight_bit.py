"""float64 definitions of the 8-bit serving operators (TEST INFRASTRUCTURE ONLY).

The reference has no 8-bit activations, weights or cache; the attention follows
``oracle.hotpath`` (its ``tests/cpu_reference.py:55-89``) with the cached rows replaced by
the values that their codes stand for.
"""
import numpy as np

from .hotpath import prepare_rows, sigmoid

BLOCK, COLS = 64, 128


def e4m3_values():
    """The value of every e4m3 code (sign, 4 exponent bits of bias 7, 3 mantissa bits; 0x7F and 0xFF are NaN)."""
    c = np.arange(256)
    e, m = c >> 3 & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((c & 127) == 127, np.nan, v)
    return np.where(c >> 7, -v, v)


def decode(codes):
    return e4m3_values()[np.asarray(codes).view(np.uint8)]


def norm(x, weights, residual=None, epsilon=1e-6):
    """(sum as stored in fp32, normed rows in float64)."""
    s = x if residual is None else (x + residual).astype(np.float32)
    d = s.astype(np.float64)
    return s, d / np.sqrt((d * d).mean(-1, keepdims=True) + epsilon) * weights.astype(np.float64)


def column_scales(y):
    """max|y| / 448 of every row and 128 columns: [blocks][tokens], float64; NaN where a value is not finite."""
    tokens, width = y.shape
    out = np.empty((-(-width // COLS), tokens))
    for b in range(out.shape[0]):
        part = y[:, b * COLS:(b + 1) * COLS]
        out[b] = np.where(np.isfinite(part).all(-1), np.abs(part).max(-1) / 448, np.nan)
    return out


def product(codes, scales, weights, weight_scales):
    """(out, the sum of the terms' magnitudes), both [tokens][rows] float64."""
    x, w = decode(codes), decode(weights)
    tokens, width = x.shape
    out, size = np.zeros((tokens, w.shape[0])), np.zeros((tokens, w.shape[0]))
    row_block = np.arange(w.shape[0]) // COLS
    for b in range(-(-width // COLS)):
        cols = slice(b * COLS, (b + 1) * COLS)
        f = scales[b].astype(np.float64)[:, None] * weight_scales[row_block, b].astype(np.float64)[None]
        out += x[:, cols] @ w[:, cols].T * f
        size += np.abs(x[:, cols]) @ np.abs(w[:, cols]).T * np.abs(f)
    return out, size


def pack(rows):
    """int8 codes [blocks][4][64][256] and fp32 scales [blocks][4] of fp16 rows [64 n][4][256]."""
    x = rows.astype(np.float64).reshape(-1, BLOCK, 4, 256).transpose(0, 2, 1, 3)
    amax = np.abs(x).max((2, 3))
    finite = np.isfinite(x).all((2, 3))
    scales = np.where(finite, amax / 127, np.nan).astype(np.float32)
    divisor = np.where(finite & (scales > 0), scales, 1).astype(np.float64)[:, :, None, None]
    codes = np.where(finite[:, :, None, None], np.rint(np.where(np.isfinite(x), x, 0) / divisor), 0)
    return codes.astype(np.int8), scales


def unpack(codes, scales):
    """The values of the codes, float64 rows [64 n][4][256]."""
    v = codes.astype(np.float64) * scales.astype(np.float64)[:, :, None, None]
    return v.transpose(0, 2, 1, 3).reshape(-1, 4, 256)


def attention(key_rows, value_rows, q_gate, q_norm, position, epsilon=1e-6):
    """(out [T][24][256], the sum of p |v| times the gate, the largest sum |q k| / 16 of any score), float64:
    queries at position .. position + T - 1 over the rows [0, position + t] of float64 K/V [n][4][256]."""
    T = q_gate.shape[0]
    q = prepare_rows(q_gate[..., :256], q_norm, position + np.arange(T)[:, None], epsilon)
    gate = sigmoid(q_gate[..., 256:])
    out, size, top = np.zeros((T, 24, 256)), np.zeros((T, 24, 256)), 0.0
    for h in range(24):
        k, v = key_rows[:, h // 6], value_rows[:, h // 6]
        for t in range(T):
            n = position + t + 1
            s = k[:n] @ q[t, h] / 16
            with np.errstate(invalid='ignore'):
                top = max(top, float(np.nanmax(np.abs(k[:n]) @ np.abs(q[t, h]))) / 16)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ v[:n] * gate[t, h]
                size[t, h] = p @ np.abs(v[:n]) * gate[t, h]
    return out, size, top
