"""The 4-bit, norm and attention operators on tensors of more than 2^31 elements: the last rows are what they are alone."""
import pytest
import torch

import cache_dit_b200 as cd
from tests.test_gpu_cross_attention import _check

pytestmark = pytest.mark.gpu
ROWS, COLS = 140_011, 16_384  # 2.29e9 elements
TAIL = 133


@pytest.fixture(autouse=True)
def _free():
  yield
  torch.cuda.empty_cache()


def _big(rows=ROWS, cols=COLS, seed=0):
  g = torch.Generator(device="cuda").manual_seed(seed)
  x = torch.empty(rows, cols, device="cuda", dtype=torch.bfloat16)
  for i in range(0, rows, 20_000):
    x[i:i + 20_000].normal_(generator=g)
  assert x.numel() > 2**31
  return x


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@torch.no_grad()
def test_quantised_and_back(fmt):
  x = _big()
  t = cd.float4_quantize_rows(x, fmt)
  for rows in (slice(0, 128), slice(ROWS // 128 * 128 - 128, ROWS)):  # whole panels of scales
    part = cd.float4_quantize_rows(x[rows].clone(), fmt)
    assert torch.equal(t.codes[rows], part.codes)
    panel = t.block_scales.numel() // -(-ROWS // 128)
    at = rows.start // 128 * panel
    assert torch.equal(t.block_scales[at:at + part.block_scales.numel()], part.block_scales)
    assert fmt == "mxfp4" or torch.equal(t.row_scale[rows], part.row_scale)
    back = cd.float4_dequantize_rows(t)
    assert torch.equal(back[rows], cd.float4_dequantize_rows(part))
    del back


@torch.no_grad()
def test_product_with_a_large_output():
  m, n, k = 262_147, 8_200, 96
  a = cd.float4_quantize_rows(torch.randn(m, k, device="cuda").to(torch.bfloat16))
  w = cd.float4_quantize_rows(torch.randn(n, k, device="cuda").to(torch.bfloat16))
  out = cd.float4_scaled_mm(a, w)
  assert out.numel() > 2**31
  wf = cd.float4_dequantize_rows(w, torch.float32).double()
  af = cd.float4_dequantize_rows(a, torch.float32)[-TAIL:].double()
  want = af @ wf.t()
  # fp32 accumulation of 96 products, one rounding to bfloat16
  assert ((out[-TAIL:].double() - want).abs() <= 2.0**-8 * want.abs() + 10 * 2.0**-23 * (af.abs() @ wf.abs().t())).all()


@pytest.mark.parametrize("quantize", [None, "nvfp4"])
@torch.no_grad()
def test_norm(quantize):
  x, y = _big(), _big(seed=1)
  gate = torch.randn(COLS, device="cuda").to(torch.bfloat16)
  x2, h = cd.gated_residual_norm(x, y, gate, norm="layer", quantize=quantize)
  for rows in (slice(0, TAIL), slice(ROWS - TAIL, ROWS)):
    x2p, hp = cd.gated_residual_norm(x[rows], y[rows], gate, norm="layer", quantize=quantize)
    assert torch.equal(x2[rows], x2p)
    assert torch.equal(h[rows], hp) if quantize is None else torch.equal(h.codes[rows], hp.codes)


@torch.no_grad()
def test_attention_over_a_long_context():
  heads, keys, d = 32, 1_100_003, 64
  k, v = (_big(keys, heads * d, seed=s).view(1, keys, heads, d) for s in (2, 3))
  q = torch.randn(1, 3, heads, d, device="cuda").to(torch.bfloat16)
  got = cd.cross_attention(q, k, v)
  for h in (0, 17, 31):
    _check(got[:, :, h:h + 1], q[:, :, h:h + 1], k[:, :, h:h + 1], v[:, :, h:h + 1])
  mask = torch.zeros(1, keys, dtype=torch.bool, device="cuda")
  mask[:, -TAIL:] = True
  got = cd.cross_attention(q, k, v, mask)
  _check(got, q, k[:, -TAIL:], v[:, -TAIL:])
  mask[:, :] = False
  mask[:, 0] = mask[:, -1] = True
  got = cd.cross_attention(q, k, v, mask)
  two = [t[:, [0, -1]] for t in (k, v)]
  _check(got, q, *two)


@torch.no_grad()
def test_attention_of_many_queries():
  heads, queries, d = 24, 800_011, 128
  q = _big(queries, heads * d, seed=4).view(1, queries, heads, d)
  k, v = (torch.randn(1, 77, heads, d, device="cuda").to(torch.bfloat16) for _ in range(2))
  got = cd.cross_attention(q, k, v)
  for rows in (slice(0, 300), slice(queries - 300, queries)):
    _check(got[:, rows], q[:, rows], k, v)
