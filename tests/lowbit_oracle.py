"""Oracle of the low-bit formats in numpy, 64 bits: every value by search among what a format holds, ties to the even code."""
from __future__ import annotations

import numpy as np
import torch

BLOCK = {"mxfp4": 32, "nvfp4": 16}
CODES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E4M3 = np.array([(m / 8 * 2.0 ** -6) if e == 0 else (1 + m / 8) * 2.0 ** (e - 7) for e in range(16) for m in range(8)][:127])      # 0 .. 448


def nearest_even(x, table):
    """Index of the entry of ``table`` (ascending) next to every x >= 0, of two equally near ones the even index; the last for what lies beyond."""
    hi = np.clip(np.searchsorted(table, x), 1, len(table) - 1)
    lo = hi - 1
    a, b = x - table[lo], table[hi] - x
    return np.where(a < b, lo, np.where(b < a, hi, np.where(lo % 2 == 0, lo, hi)))


def round4(x: torch.Tensor, fmt: str):
    """(codes [R, K], scale bytes [R, K / block], row factors or None) of a 2-D tensor."""
    x = x.double().numpy()
    R, K = x.shape
    b = x.reshape(R, K // BLOCK[fmt], BLOCK[fmt])
    fine = np.isfinite(b).all(-1)
    size = np.where(fine, np.abs(np.where(fine[..., None], b, 0)).max(-1), 0)
    if fmt == "mxfp4":
        byte = np.where(size > 0, np.clip(np.floor(np.log2(np.where(size > 0, size, 1))) - 2 + 127, 0, 254), 0).astype(int)
        s, row, zero = 2.0 ** (byte - 127.0), None, np.zeros_like(size, bool)
    else:
        most = size.max(-1, keepdims=True)
        row = np.where(most > 0, 2.0 ** np.maximum(np.floor(np.log2(np.where(most > 0, most, 1))) - 10, -126), 1.0)
        byte = nearest_even(size / row / 6, E4M3)
        s, zero = E4M3[byte] * row, byte == 0
    with np.errstate(invalid="ignore", divide="ignore"):
        q = np.where(zero[..., None] | ~fine[..., None], 0, b / np.where(s > 0, s, 1)[..., None])
    code = nearest_even(np.abs(q), CODES) + 8 * np.signbit(b)
    byte = np.where(fine, byte, 255 if fmt == "mxfp4" else 0x7F)
    if row is not None:
        row = np.where(fine.all(-1), row[:, 0], np.nan)
    return code.reshape(R, K), byte, row


def scale_byte(scales: np.ndarray, r: int, b: int) -> int:
    return scales[r // 128, b // 4, r % 32, r // 32 % 4, b % 4]


def unpack(q):
    """(codes, scale bytes, row factors) of a QuantRows of one matrix, by the documented layout."""
    codes, scales = q.codes.cpu().numpy(), q.scales.cpu().numpy()
    R, K = q.rows, q.cols
    code = np.empty((R, K), dtype=int)
    code[:, 0::2], code[:, 1::2] = codes & 15, codes >> 4
    r, b = np.arange(R)[:, None], np.arange(K // BLOCK[q.fmt])[None, :]
    return code, scale_byte(scales, r, b).astype(int), None if q.row_scale is None else q.row_scale.cpu().double().numpy()


def values(q) -> np.ndarray:
    """[R, K] (or [E, R, K]) in 64 bits."""
    if q.experts is not None:
        from vllm_omni_b200.ops.lowbit import QuantRows
        return np.stack([values(QuantRows(q.codes[e], q.scales[e], q.fmt, None if q.row_scale is None else q.row_scale[e])) for e in range(q.experts)])
    code, byte, row = unpack(q)
    v = CODES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = np.where(byte == 255, np.nan, 2.0 ** (byte - 127.0)) if q.fmt == "mxfp4" else np.where(byte == 127, np.nan, E4M3[np.minimum(byte, 126)]) * row[:, None]
    return (v.reshape(q.rows, -1, BLOCK[q.fmt]) * s[..., None]).reshape(q.rows, q.cols)


def value_of(x: np.ndarray, fmt: str) -> np.ndarray:
    """What rows [R, K] become when they are quantised."""
    code, byte, row = round4(torch.from_numpy(x), fmt)
    v = CODES[code & 7] * np.where(code & 8, -1.0, 1.0)
    s = 2.0 ** (byte - 127.0) if fmt == "mxfp4" else E4M3[np.minimum(byte, 126)] * row[:, None]
    return (v.reshape(x.shape[0], -1, BLOCK[fmt]) * s[..., None]).reshape(x.shape)
