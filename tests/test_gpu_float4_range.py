"""The 4-bit product where one operand's scales are huge and the other's tiny: what is finite comes out finite."""
import numpy as np
import pytest
import torch

import cache_dit_b200 as cd
from oracle import fp4_oracle as F4

pytestmark = pytest.mark.gpu


def _quantised(x, fmt):
  return cd.float4_quantize_rows(x.cuda(), fmt), F4.values(*F4.quantize(x.double().numpy(), fmt), fmt)


def _compare(a, w, fmt):
  """a @ w^T against 64 bits.  fp32 accumulation (a whole step of the running sum each 16 columns), scales that are powers
  of two or were multiplied in exactly, one rounding to bfloat16; numbers whose bfloat16 is subnormal to half its step."""
  (qa, va), (qw, vw) = _quantised(a, fmt), _quantised(w, fmt)
  want = va @ vw.T
  got = cd.float4_scaled_mm(qa, qw).double().cpu().numpy()
  k = a.shape[1]
  bound = (k / 16 + 4) * 2.0**-23 * (np.abs(va) @ np.abs(vw).T + np.abs(want)) + 2.0**-8 * np.abs(want) + 2.0**-126
  assert np.abs(want).max() < 3.3e38 and np.isfinite(got).all(), got
  assert (np.abs(got - want) <= bound).all(), (np.abs(got - want) / bound).max()


SCALES = [(127, -10), (127, -40), (127, -120), (120, -8), (-90, 100), (-100, 90), (60, 50), (-60, -50), (-100, -20), (20, -110)]


@pytest.mark.parametrize("m", [1, 3, 130, 300])
@pytest.mark.parametrize("n", [16, 264])
@pytest.mark.parametrize("ea,ew", SCALES)
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_far_apart_scales(fmt, ea, ew, m, n):
  g = torch.Generator().manual_seed(m + n)
  draw = lambda rows, e: torch.ldexp(torch.rand(rows, 96, generator=g) * 2 - 1, torch.tensor(e)).to(torch.bfloat16)
  _compare(draw(m, ea), draw(n, ew), fmt)


@pytest.mark.parametrize("m", [1, 3, 130, 300])
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_one_loud_element(fmt, m):
  a = torch.zeros(m, 64)
  a[:, 0] = 3e38
  a[:, 40] = 1.0
  w = torch.full((136, 64), 1e-3)
  w[:, 32:] = 2.0
  _compare(a.to(torch.bfloat16), w.to(torch.bfloat16), fmt)


@pytest.mark.parametrize("m", [1, 3, 130])
def test_block_scales_whose_product_is_beyond_fp32(m):
  """mxfp4 blocks of 2^98 and 2^30: their scales' product is 2^128, their sums of codes 0.25 and 0."""
  a, w = torch.zeros(m, 64), torch.zeros(24, 64)
  a[:, 0], a[:, 1] = 2.0**97, 2.0**100
  w[:, 0], w[:, 2] = 2.0**29, 2.0**32
  _compare(a.to(torch.bfloat16), w.to(torch.bfloat16), "mxfp4")
  w[:, 0] = 0.0
  _compare(a.to(torch.bfloat16), w.to(torch.bfloat16), "mxfp4")
