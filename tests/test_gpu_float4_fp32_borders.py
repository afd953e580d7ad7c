"""Quantisation of float32 rows one last place from every border of a decision: as exact as that of 16-bit rows."""
import numpy as np
import pytest
import torch

import cache_dit_b200 as cd
from oracle import fp4_oracle as F4
from tests.test_gpu_float4 import _check_quantised

pytestmark = pytest.mark.gpu
BORDERS = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=np.float32)


def _neighbours(v):
  v = np.asarray(v, dtype=np.float32)
  return np.concatenate([np.nextafter(v, np.float32(0)), v, np.nextafter(v, np.float32(np.inf))])


@pytest.mark.parametrize("exponent", [-90, -20, 0, 31, 110])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_codes(fmt, exponent):
  """Every mantissa a block scale can have, every border between two codes, and the float32 numbers on either side."""
  block = F4.BLOCK[fmt]
  blocks = [np.zeros(block, dtype=np.float32)]
  blocks[0][0] = 2688.0  # nvfp4: the row scale is then 2^exponent
  for scale in (F4.E4M3[8:127] if fmt == "nvfp4" else 2.0**np.arange(-9, 9)):
    values = _neighbours(BORDERS * np.float32(scale))
    for part in np.array_split(values * np.where(np.arange(len(values)) % 2, -1, 1).astype(np.float32), -(-len(values) // (block - 1))):
      b = np.zeros(block, dtype=np.float32)
      b[0] = 6 * scale
      b[1:1 + len(part)] = part
      blocks.append(b)
  while len(blocks) * block % 256:
    blocks.append(blocks[1])
  row = np.concatenate(blocks) * np.float32(2.0**exponent)
  x = torch.from_numpy(np.stack([row, -row]).astype(np.float32))
  _check_quantised(x, cd.float4_quantize_rows(x.cuda(), fmt), fmt)


@pytest.mark.parametrize("exponent", [-90, 0, 110])
def test_block_scales(exponent):
  """Largest magnitudes of blocks around every border between two e4m3 scales (six times the mean of neighbours)."""
  borders = (F4.E4M3[1:127] + F4.E4M3[:126]) / 2 * 6
  tops = _neighbours(borders.astype(np.float32))
  assert np.array_equal(borders.astype(np.float32).astype(np.float64), borders)
  x = np.zeros((2, (tops.size + 1 + 15) // 16 * 16, 16), dtype=np.float32)
  x[:, 0, 0] = 2688.0
  x[0, 1:1 + tops.size, 3] = tops
  x[1, 1:1 + tops.size, 3] = -tops
  x[:, 1:1 + tops.size, 4] = tops / 3
  t = torch.from_numpy(x.reshape(2, -1) * np.float32(2.0**exponent))
  _check_quantised(t, cd.float4_quantize_rows(t.cuda(), "nvfp4"), "nvfp4")
