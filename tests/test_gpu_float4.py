"""4-bit microscaled rows and their product on the GPU against the 64-bit restatement in oracle/fp4_oracle.py.

Quantisation decisions are exact for 16-bit inputs (quotients of an at most 11-bit number by an at most 4-bit one either
hit a rounding boundary or miss it by more than fp32 can blur), so codes and scales are compared for equality.
"""
import numpy as np
import pytest
import torch

import cache_dit_b200 as cd
from cache_dit_b200 import _native
from oracle import fp4_oracle as F4

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
FORMATS = ["nvfp4", "mxfp4"]


def _rows(rows, cols, dtype, seed, spread=1.0):
  g = torch.Generator().manual_seed(seed)
  x = torch.randn(rows, cols, generator=g) * torch.exp(spread * torch.randn(rows, 1, generator=g))
  x = x * torch.exp(spread * torch.randn(1, cols, generator=g))
  return x.to(dtype)


def _check_quantised(x, got, fmt):
  rows, cols = x.shape
  code, byte, row = F4.quantize(x.double().numpy(), fmt)
  codes = got.codes.cpu().numpy().reshape(rows, cols // 2)
  value = lambda c: F4.E2M1[np.stack([c & 15, c >> 4], axis=2).reshape(rows, cols)]
  assert np.array_equal(got.block_scales.cpu().numpy(), F4.tile_scales(byte, fmt))
  assert np.array_equal(value(codes), value(F4.pack(code)))  # as values: a zero may carry a sign
  if fmt == "nvfp4":
    assert np.array_equal(got.row_scale.cpu().numpy().astype(np.float64).reshape(rows), row)
  else:
    assert got.row_scale is None


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (127, 96), (129, 256), (5, 512), (64, 1056), (33, 2080), (7, 4096),
                                       (300, 5120), (9, 8224), (2, 16384), (1000, 160)])
def test_quantise_rows(rows, cols, dtype, fmt):
  x = _rows(rows, cols, dtype, rows * 7 + cols)
  _check_quantised(x, cd.float4_quantize_rows(x.cuda(), fmt), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
def test_quantise_edges(dtype, fmt):
  """Zero rows and blocks, ties of every code, the smallest and largest numbers of the type, a wide spread in a row."""
  x = torch.zeros(12, 256, dtype=dtype)
  x[1, 5] = 1.0
  x[2] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 32, dtype=torch.float32).to(dtype)
  x[3] = -x[2]
  info = torch.finfo(dtype)
  x[4, ::3] = info.tiny
  x[5, 0] = info.max
  x[5, 200] = info.min
  x[6] = torch.logspace(-6, 2, 256).to(dtype)
  x[7, :] = -0.0
  x[8, 16:32] = 1.5
  x[9, 0] = 2.0**-14
  x[10] = torch.linspace(-7, 7, 256).to(dtype)
  x[11] = 6 * 448  # largest magnitude = 2688 / 2048 exactly: the border of the row scale's exponent
  _check_quantised(x, cd.float4_quantize_rows(x.cuda(), fmt), fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantise_takes_strided_rows_and_any_leading_shape(fmt):
  wide = _rows(70, 512, torch.bfloat16, 3).cuda()
  for x in (wide[:, 128:128 + 96], wide[:, 3:3 + 64], wide[::2, :256], wide.t()[:, :64], wide.view(2, 35, 512)[..., :160],
            wide[:1, :64].expand(40, 64), wide[5, :32]):
    got = cd.float4_quantize_rows(x, fmt)
    want = cd.float4_quantize_rows(x.contiguous().clone(), fmt)
    assert got.shape == x.shape and got.codes.shape == (*x.shape[:-1], x.shape[-1] // 2)
    for a, b in zip(got._triple(), want._triple()):
      assert (a is None and b is None) or torch.equal(a, b)
  assert cd.float4_quantize_rows(wide[:0, :64], fmt).shape == (0, 64)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_non_finite_inputs_stand_for_nan(fmt, bad):
  x = _rows(5, 512, torch.bfloat16, 1)
  x[2, 100] = bad
  t = cd.float4_quantize_rows(x.cuda(), fmt)
  back = cd.float4_dequantize_rows(t).float().cpu()
  hit = torch.zeros(5, 512, dtype=torch.bool)
  if fmt == "nvfp4":
    hit[2] = True  # the row's scale
  else:
    hit[2, 96:128] = True  # the block's
  assert torch.equal(torch.isnan(back), hit) and torch.isfinite(back[~hit]).all()
  w = cd.float4_quantize_rows(_rows(64, 512, torch.bfloat16, 2).cuda(), fmt)
  for rows in (5, 200):  # the few-row kernel and a tile kernel
    xs = x.repeat(rows // 5, 1)
    out = cd.float4_scaled_mm(cd.float4_quantize_rows(xs.cuda(), fmt), w).float().cpu()
    row_hit = (torch.arange(rows) % 5) == 2
    assert torch.isnan(out[row_hit]).all() and torch.isfinite(out[~row_hit]).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (130, 96), (77, 4128), (3, 16384)])
def test_dequantise_rows(rows, cols, dtype, fmt):
  x = _rows(rows, cols, torch.bfloat16, 11)
  t = cd.float4_quantize_rows(x.cuda(), fmt)
  want = torch.from_numpy(F4.values(*F4.quantize(x.double().numpy(), fmt), fmt)).to(dtype)  # products exact in fp32
  assert torch.equal(cd.float4_dequantize_rows(t, dtype).cpu(), want)


def _operands(m, n, k, fmt, seed, dtype=torch.bfloat16):
  a, w = _rows(m, k, dtype, seed, 0.5), (_rows(n, k, dtype, seed + 1, 0.3).float() * k**-0.5).to(dtype)
  qa, qw = cd.float4_quantize_rows(a.cuda(), fmt), cd.float4_quantize_rows(w.cuda(), fmt)
  va = F4.values(*F4.quantize(a.double().numpy(), fmt), fmt)
  vw = F4.values(*F4.quantize(w.double().numpy(), fmt), fmt)
  return qa, qw, va, vw


def _product_bound(va, vw, y, k, dtype):
  # fp32 accumulation over k terms, each step off by at most a whole step (2^-23: the tensor core may truncate) of the
  # running sum, itself at most sum |a||w|; one rounding to the output type at the end
  return (k / 16 + 4) * 2.0**-23 * (np.abs(va) @ np.abs(vw).T + np.abs(y)) + torch.finfo(dtype).eps / 2 * np.abs(y) + \
      torch.finfo(dtype).tiny


SHAPES = [(1, 8, 32), (1, 128, 256), (2, 264, 544), (3, 136, 5120), (4, 1000, 1024), (5, 8, 64), (128, 128, 256), (129, 64, 96),
          (100, 200, 320), (77, 640, 4096), (257, 520, 288), (256, 256, 512), (300, 1032, 1056), (1000, 512, 2048),
          (520, 2304, 768), (2100, 4104, 512)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(m, n, k, fmt):
  qa, qw, va, vw = _operands(m, n, k, fmt, m + n + k)
  y = va @ vw.T
  got = cd.float4_scaled_mm(qa, qw).double().cpu().numpy()
  assert _native.gemm_device_status(torch.device("cuda")) == 0
  assert (np.abs(got - y) <= _product_bound(va, vw, y, k, torch.bfloat16)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("n,k", [(8, 2016), (8, 2048), (136, 4096), (264, 8224), (1000, 16384), (4744, 1056), (9480, 2080), (19000, 544)])
def test_product_of_one_row(n, k, fmt):
  """Few columns split K over the warps of a block, many do not; K ends inside a warp's share."""
  qa, qw, va, vw = _operands(1, n, k, fmt, n + k)
  y = va @ vw.T
  got = cd.float4_scaled_mm(qa, qw)
  assert torch.equal(got, cd.float4_scaled_mm(qa, qw))
  assert (np.abs(got.double().cpu().numpy() - y) <= _product_bound(va, vw, y, k, torch.bfloat16)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k,gelu", [(1, 72, 96, True), (4, 256, 512, False), (60, 320, 512, True), (700, 1288, 1024, True),
                                        (700, 1288, 1024, False)])
def test_linear_bias_and_gelu(m, n, k, gelu, dtype, fmt):
  a, w = _rows(m, k, dtype, 5, 0.5), (_rows(n, k, dtype, 6, 0.3).float() * k**-0.5).to(dtype)
  bias = (0.5 * torch.randn(n, generator=torch.Generator().manual_seed(7))).to(dtype)
  va, vw = (F4.values(*F4.quantize(t.double().numpy(), fmt), fmt) for t in (a, w))
  y = va @ vw.T + bias.double().numpy()
  bound = _product_bound(va, vw, y, k, torch.float32) + 2.0**-23 * np.abs(bias.double().numpy())
  want = y
  if gelu:
    want = F4.gelu_tanh(y)
    # slope of the tanh-GELU is at most 1.13; its own fp32 evaluation (ex2.approx, fast division) is within 2^-20
    bound = 1.13 * bound + 2.0**-20 * np.abs(want) + 2.0**-24
  bound = bound + torch.finfo(dtype).eps / 2 * (np.abs(want) + bound) + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
  x = a.cuda().view(1, m, k)
  got = cd.float4_linear(x, cd.float4_quantize_rows(w.cuda(), fmt), bias.cuda(), gelu=gelu)
  assert got.shape == (1, m, n) and got.dtype == dtype
  assert (np.abs(got[0].double().cpu().numpy() - want) <= bound).all()


TILES = [(0, 64), (0, 128), (1, 128), (1, 256)]


@pytest.fixture
def tile(request):
  pair, cols = request.param
  assert _native.lib().cdb_tuning_set_fp4_tile(pair, cols) == 0
  yield request.param
  assert _native.lib().cdb_tuning_set_fp4_tile(0, 0) == 0


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile", TILES, indirect=True)
@pytest.mark.parametrize("m,n,k", [(3, 8, 32), (130, 200, 288), (257, 264, 1312), (300, 720, 2048)])
def test_every_tile_shape(m, n, k, tile, fmt):
  qa, qw, va, vw = _operands(m, n, k, fmt, m + n + k)
  y = va @ vw.T
  got = cd.float4_scaled_mm(qa, qw).double().cpu().numpy()
  assert (np.abs(got - y) <= _product_bound(va, vw, y, k, torch.bfloat16)).all()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tile", TILES, indirect=True)
def test_many_tiles_per_cta(tile, fmt):
  """More tiles than SMs, so every CTA goes round its accumulators, scale slots and ring several times."""
  m, n, k = 3500, 8200, 1056
  g = torch.Generator().manual_seed(1)
  a, w = (torch.randn(r, k, generator=g).cuda() for r in (m, n))
  qa, qw = cd.float4_quantize_rows(a, fmt), cd.float4_quantize_rows(w, fmt)
  va, vw = (cd.float4_dequantize_rows(q, torch.float32).double() for q in (qa, qw))
  y = va @ vw.t()
  bound = (k / 16 + 4) * 2.0**-23 * (va.abs() @ vw.abs().t() + y.abs()) + 2.0**-8 * y.abs() + 1e-30
  for _ in range(3):
    got = cd.float4_scaled_mm(qa, qw).double()
    assert ((got - y).abs() <= bound).all()
  assert _native.gemm_device_status(torch.device("cuda")) == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_dequantise_into_rows_that_are_only_16_byte_aligned(dtype):
  t = cd.float4_quantize_rows(_rows(33, 96, torch.bfloat16, 2).cuda())
  want = cd.float4_dequantize_rows(t, dtype)
  room = torch.full((33 * 96 + 64, ), 7.0, dtype=dtype, device="cuda")
  off = 16 // room.element_size()
  out = room[off:off + 33 * 96].view(33, 96)
  _native.fp4_dequant_rows(*t._triple(), 33, 96, "nvfp4", out)
  assert torch.equal(out, want) and (room[:off] == 7).all() and (room[off + 33 * 96:] == 7).all()
