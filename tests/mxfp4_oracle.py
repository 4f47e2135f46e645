"""The 4-bit microscaled format in plain 64-bit arithmetic (test infrastructure only): a block
of 32 values, scale 2^(floor(log2 max) - 2) at least 2^-127, elements the nearest of
{0, .5, 1, 1.5, 2, 3, 4, 6} with ties to the even code; a block with an infinity or NaN is NaN."""
import numpy as np
import torch

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def quantize(x: torch.Tensor):
    """(packed codes uint8 [rows, blocks * 16], scales uint8 [rows, blocks]) of x's rows."""
    v = x.detach().cpu().double().numpy()
    rows, cols = v.shape
    blocks = -(-cols // 32)
    v = np.concatenate([v, np.zeros((rows, blocks * 32 - cols))], axis=1).reshape(rows, blocks, 32)
    bad = ~np.isfinite(v).all(axis=2)
    v = np.where(bad[:, :, None], 0.0, v)
    top = np.abs(v).max(axis=2)
    _, exponent = np.frexp(top)                           # top = m * 2^exponent, m in [.5, 1)
    exponent = np.where(top > 0, exponent - 3, -127).clip(-127, None)
    size = np.abs(v) * np.ldexp(1.0, -exponent)[:, :, None]
    codes = np.zeros(v.shape, dtype=np.uint8)
    for code in range(1, 8):
        border = (GRID[code - 1] + GRID[code]) / 2
        codes[(size > border) if code % 2 else (size >= border)] = code
    codes |= np.signbit(v).astype(np.uint8) << 3
    codes[bad] = 0
    codes = codes.reshape(rows, blocks * 16, 2)
    scales = np.where(bad, 255, np.where(top > 0, exponent + 127, 0)).astype(np.uint8)
    return torch.from_numpy(codes[..., 0] | (codes[..., 1] << 4)), torch.from_numpy(scales)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 [rows, blocks * 32] that codes and scales stand for."""
    c, s = codes.cpu().numpy(), scales.cpu().numpy().astype(np.int64)
    rows, blocks = s.shape
    halves = np.stack([c & 15, c >> 4], axis=2).reshape(rows, blocks, 32)
    v = GRID[halves & 7] * np.where(halves & 8, -1.0, 1.0) * np.ldexp(1.0, s - 127)[:, :, None]
    v = np.where((s == 255)[:, :, None], np.nan, v)
    return torch.from_numpy(v.reshape(rows, blocks * 32))
