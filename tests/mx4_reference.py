"""Microscaled 4-bit rows restated in float64 on the host (numpy), for the tests."""
import math

import numpy as np
import torch

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantise(x: torch.Tensor):
    """[rows, cols] -> codes uint8 [rows, 16 * blocks], scale bytes uint8 [rows, blocks], value by value"""
    a = x.detach().cpu().double().numpy()
    rows, cols = a.shape
    blocks = (cols + 31) // 32
    v = np.zeros((rows, blocks * 32))
    v[:, :cols] = a
    v = v.reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(2)
    v = np.where(bad[..., None], 0.0, v)
    top = np.abs(v).max(2)
    exponent = np.frexp(top)[1] - 1                     # floor(log2), exactly
    byte = np.where(top > 0, np.maximum(exponent - 2 + 127, 0), 0)
    r = np.ldexp(v, (127 - byte)[..., None])
    m = np.abs(r)
    code = np.zeros(m.shape, dtype=np.int64)
    for k in range(7):                                  # between VALUES[k] and VALUES[k + 1]
        mid = (VALUES[k] + VALUES[k + 1]) / 2
        code += (m > mid) | ((m == mid) & (k % 2 == 1))
    code |= np.signbit(r).astype(np.int64) << 3
    code = np.where(bad[..., None], 0, code).reshape(rows, -1, 2)
    byte = np.where(bad, 255, byte)
    return (torch.from_numpy((code[..., 0] | code[..., 1] << 4).astype(np.uint8)), torch.from_numpy(byte.astype(np.uint8)))


def values(codes: torch.Tensor, scales: torch.Tensor, cols: int) -> torch.Tensor:
    """-> float64 [rows, cols]"""
    c = codes.cpu().numpy().astype(np.int64)
    c = np.stack([c & 15, c >> 4], 2).reshape(c.shape[0], -1, 32)
    v = np.array(VALUES)[c & 7] * np.where(c & 8, -1.0, 1.0)
    s = scales.cpu().numpy().astype(np.int64)
    unit = np.where(s == 255, math.nan, np.ldexp(1.0, np.where(s == 255, 0, s - 127)))
    return torch.from_numpy((v * unit[..., None]).reshape(c.shape[0], -1)[:, :cols].copy())


def tiled(scales: torch.Tensor, cols: int) -> torch.Tensor:
    """plain scale bytes [rows, blocks] in the order of the products"""
    rows, blocks = scales.shape
    kts = 2 * ((cols + 255) // 256)
    out = torch.zeros((rows + 127) // 128, kts, 32, 4, 4, dtype=torch.uint8)
    for r in range(rows):
        for j in range(blocks):
            out[r // 128, j // 4, r % 32, r // 32 % 4, j % 4] = scales[r, j]
    return out.reshape(-1)
