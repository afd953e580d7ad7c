"""A `Float4Linear` keeps what its kernels read when the model around it changes type."""
import pytest
import torch

import cache_dit_b200 as cd
from cache_dit_b200.quantization import float4

CASTS = {"to_bfloat16": lambda m: m.to(torch.bfloat16), "bfloat16": lambda m: m.bfloat16(), "half": lambda m: m.half(), "float": lambda m: m.float(),
         "double": lambda m: m.double(), "type": lambda m: m.type(torch.float16)}


def _module(rows4, fmt, device):
  bias = torch.arange(16, device=device).to(torch.bfloat16) / 3
  return torch.nn.Sequential(cd.Float4Linear(rows4, bias), torch.nn.LayerNorm(16, device=device))


@pytest.mark.parametrize("cast", list(CASTS))
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_types_stay(fmt, cast):
  rows4 = float4.empty_rows((16, ), 64, fmt, "cpu")
  rows4.codes.fill_(0x21)
  rows4.block_scales.fill_(0x38)
  if rows4.row_scale is not None:
    rows4.row_scale.copy_(torch.ldexp(torch.ones(16), torch.arange(16) * 7 - 50))  # beyond float16
  m = _module(rows4, fmt, "cpu")
  before = {k: v.clone() for k, v in m[0].state_dict().items()}
  CASTS[cast](m)
  after = m[0].state_dict()
  assert set(after) == set(before)
  for k in before:
    assert after[k].dtype == before[k].dtype and torch.equal(after[k], before[k]), k
  assert m[1].weight.dtype != torch.float32 or cast == "float"  # the rest of the model did change
  float4._check_rows(m[0].weight_rows, "w")


def test_devices_are_followed():
  rows4 = float4.empty_rows((16, ), 64, "nvfp4", "cpu")
  m = _module(rows4, "nvfp4", "cpu").to("meta", torch.float16)
  assert all(t.device.type == "meta" for t in m[0].state_dict().values())
  assert m[0].weight_row_scale.dtype == torch.float32 and m[0].bias.dtype == torch.bfloat16


@pytest.mark.gpu
@pytest.mark.parametrize("cast", list(CASTS))
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_outputs_stay(fmt, cast):
  lin = torch.nn.Linear(320, 264).to("cuda", torch.bfloat16)
  m = torch.nn.Sequential(cd.Float4Linear.from_linear(lin, fmt))
  x = torch.randn(5, 320, device="cuda").to(torch.bfloat16)
  with torch.no_grad():
    want = m(x)
    assert torch.equal(CASTS[cast](m)(x), want)
    assert torch.equal(m.cpu().cuda()(x), want)
