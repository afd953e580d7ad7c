"""numpy restatement, in 64 bits, of the 4-bit microscaled formats and their product (include/cache_dit_b200.h)."""
from __future__ import annotations

import numpy as np

BLOCK = {"nvfp4": 16, "mxfp4": 32}
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
E2M1 = np.concatenate([MAGNITUDES, -MAGNITUDES])


def e4m3_values() -> np.ndarray:
  """The 127 non-negative finite e4m3 numbers by their byte."""
  out = []
  for b in range(127):
    e, m = b >> 3, b & 7
    out.append((m / 8) * 2.0**-6 if e == 0 else (1 + m / 8) * 2.0**(e - 7))
  return np.array(out)


E4M3 = e4m3_values()


def nearest(x: np.ndarray, grid: np.ndarray) -> np.ndarray:
  """Index of the nearest grid value, ties to the even index, saturating (x >= 0, grid ascending)."""
  hi = np.clip(np.searchsorted(grid, x), 1, len(grid) - 1)
  lo = hi - 1
  below, above = x - grid[lo], grid[hi] - x
  return np.where(below < above, lo, np.where(below > above, hi, np.where(lo % 2 == 0, lo, hi)))


def quantize(x: np.ndarray, fmt: str):
  """x [rows, cols] float64 -> codes 0..15 [rows, cols], scale bytes [rows, cols / block], row scales [rows] (or None).
  Finite inputs only."""
  rows, cols = x.shape
  blocks = x.reshape(rows, cols // BLOCK[fmt], BLOCK[fmt])
  top = np.abs(blocks).max(axis=2)
  if fmt == "nvfp4":
    least = np.maximum(top.max(axis=1) / 2688, 2.0**-100)
    mant, exp = np.frexp(least)
    row = np.ldexp(1.0, np.where(mant == 0.5, exp - 1, exp))
    byte = nearest(top / (6 * row[:, None]), E4M3)
    step = E4M3[byte] * row[:, None]
  else:
    row = None
    exp = np.where(top > 0, np.frexp(top)[1] - 1 - 2, -127)
    byte = np.maximum(exp, -127) + 127
    step = np.ldexp(1.0, byte - 127)
  y = blocks / np.where(step > 0, step, np.inf)[:, :, None]
  code = nearest(np.abs(y), MAGNITUDES) + 8 * (y < 0)
  return code.reshape(rows, cols).astype(np.uint8), byte.astype(np.uint8), row


def scale_values(byte: np.ndarray, fmt: str) -> np.ndarray:
  return E4M3[byte] if fmt == "nvfp4" else np.ldexp(1.0, byte.astype(np.int64) - 127)


def values(code, byte, row, fmt: str) -> np.ndarray:
  step = scale_values(byte, fmt)
  if row is not None:
    step = step * np.asarray(row, dtype=np.float64)[:, None]
  return E2M1[code] * np.repeat(step, BLOCK[fmt], axis=1)


def tile_scales(byte: np.ndarray, fmt: str) -> np.ndarray:
  """Row-major scale bytes -> the tiled layout (one flat array), written from its definition byte by byte."""
  rows, per_row = byte.shape
  per_step = 256 // BLOCK[fmt]
  tiles = -(-per_row // per_step) * per_step // 4
  out = np.zeros(-(-rows // 128) * tiles * 512, dtype=np.uint8)
  r, k = np.meshgrid(np.arange(rows), np.arange(per_row), indexing="ij")
  out[((r // 128) * tiles + k // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + k % 4] = byte
  return out


def pack(code: np.ndarray) -> np.ndarray:
  return code[:, 0::2] | (code[:, 1::2] << 4)


def gelu_tanh(x: np.ndarray) -> np.ndarray:
  return 0.5 * x * (1 + np.tanh(np.sqrt(2 / np.pi) * (x + 0.044715 * x**3)))
