"""8-bit rows with a scale per block of 128, restated on the host (numpy, float64 but where the format says fp32), for the tests."""
import numpy as np
import torch


def e4m3(y):
    """float64 -> the nearest e4m3 number, ties to even, at most 448"""
    a = np.abs(y)
    exponent = np.maximum(np.frexp(a)[1] - 1, -6)          # numbers below 2^-6 are 2^-9 apart
    step = np.ldexp(1.0, exponent - 3)
    return np.copysign(np.minimum(np.rint(a / step) * step, 448.0), y)


def blocks(v, block_rows):
    rows, cols = v.shape
    padded = np.zeros((-(-rows // block_rows) * block_rows, -(-cols // 128) * 128))
    padded[:rows, :cols] = v
    return padded.reshape(-1, block_rows, padded.shape[1] // 128, 128)


def quantise(x: torch.Tensor, block_rows: int = 1):
    """[rows, cols] -> numbers float64 [rows, cols], scales float32 [row blocks, column blocks]"""
    v = blocks(x.detach().cpu().double().numpy(), block_rows)
    bad = ~np.isfinite(v).all((1, 3))
    v = np.where(bad[:, None, :, None], 0.0, v)
    top = np.abs(v).max((1, 3)).astype(np.float32)
    scale = np.maximum(top / np.float32(448), np.float32(2.0 ** -126))
    inv = np.float32(1) / scale
    y = (v * inv.astype(np.float64)[:, None, :, None]).astype(np.float32).astype(np.float64)
    code = e4m3(y).reshape(-1, v.shape[2] * 128)[: x.shape[0], : x.shape[1]]
    return torch.from_numpy(code.copy()), torch.from_numpy(np.where(bad, np.float32(np.nan), scale))


def per_element(scales: torch.Tensor, block_rows: int, rows: int, cols: int) -> torch.Tensor:
    return scales.double().repeat_interleave(block_rows, 0)[:rows].repeat_interleave(128, 1)[:, :cols]


def values(codes: torch.Tensor, scales: torch.Tensor, block_rows: int = 1) -> torch.Tensor:
    """-> float64 [rows, cols]"""
    return codes.double() * per_element(scales, block_rows, *codes.shape)
