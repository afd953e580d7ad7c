"""What the 4-bit, norm and cross-attention entry points refuse, on CPU tensors or before any kernel is reached; the
config's 4-bit types; layouts and plans that need no GPU."""
import ctypes

import numpy as np
import pytest
import torch

import cache_dit_b200 as cd
from cache_dit_b200 import _native as nat
from cache_dit_b200.quantization import float4
from oracle import fp4_oracle as F4


def _rows4(rows, cols, fmt="nvfp4"):
  return float4.empty_rows((rows, ), cols, fmt, "cpu")


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (128, 256), (129, 288), (1000, 5120)])
def test_scale_bytes_agree(rows, cols, fmt):
  byte = np.zeros((rows, cols // F4.BLOCK[fmt]), dtype=np.uint8)
  want = F4.tile_scales(byte, fmt).size
  assert nat.fp4_block_scale_bytes(rows, cols, fmt) == want
  assert nat.lib().cdb_fp4_block_scale_bytes(rows, cols, nat.FP4_FORMATS[fmt]) == want


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
def test_oracle_values_are_nearest(fmt):
  """The 64-bit restatement against the definition: no other code of a block is nearer, ties have the even code."""
  x = np.random.default_rng(0).normal(size=(7, 64)) * np.exp(np.arange(7))[:, None]
  code, byte, row = F4.quantize(x, fmt)
  step = F4.scale_values(byte, fmt) * (1 if row is None else row[:, None])
  step = np.repeat(step, F4.BLOCK[fmt], axis=1)
  err = np.abs(F4.E2M1[code] * step - x)
  best = np.abs(F4.E2M1[None, None, :] * step[:, :, None] - x[:, :, None]).min(axis=2)
  assert (err <= best * (1 + 1e-12)).all()


def test_quantisation_refusals():
  with pytest.raises(ValueError, match="format"):
    cd.float4_quantize_rows(torch.zeros(2, 32), "fp4")
  for bad in (31, 48, 16384 + 32, 0):
    with pytest.raises(ValueError, match="multiple of 32"):
      cd.float4_quantize_rows(torch.zeros(2, bad))
  with pytest.raises(RuntimeError, match="float32, bfloat16"):
    cd.float4_quantize_rows(torch.zeros(2, 32, dtype=torch.float64))
  with pytest.raises(RuntimeError, match="CUDA"):
    cd.float4_quantize_rows(torch.zeros(2, 32))
  with pytest.raises(RuntimeError, match="CUDA"):
    cd.float4_dequantize_rows(_rows4(2, 32))


def test_product_refusals():
  a, w = _rows4(4, 64), _rows4(16, 64)
  bad = lambda t, **kw: cd.Float4Rows(**{**dict(codes=t.codes, block_scales=t.block_scales, row_scale=t.row_scale, format=t.format,
                                               cols=t.cols), **kw})
  with pytest.raises(RuntimeError, match="do not match"):
    cd.float4_scaled_mm(a, _rows4(16, 96))
  with pytest.raises(RuntimeError, match="do not match"):
    cd.float4_scaled_mm(a, _rows4(16, 64, "mxfp4"))
  with pytest.raises(RuntimeError, match="multiple of 8"):
    cd.float4_scaled_mm(a, _rows4(12, 64))
  with pytest.raises(RuntimeError, match="block scales"):
    cd.float4_scaled_mm(a, bad(w, block_scales=w.block_scales[:-1]))
  with pytest.raises(RuntimeError, match="codes"):
    cd.float4_scaled_mm(bad(a, codes=a.codes[:, :-1]), w)
  with pytest.raises(RuntimeError, match="one contiguous float32"):
    cd.float4_scaled_mm(bad(a, row_scale=None), w)
  with pytest.raises(RuntimeError, match="no row scale"):
    cd.float4_scaled_mm(bad(_rows4(4, 64, "mxfp4"), row_scale=torch.ones(4)), w)
  with pytest.raises(RuntimeError, match="bias"):
    cd.float4_scaled_mm(a, w, torch.zeros(16))
  with pytest.raises(RuntimeError, match="writes bfloat16"):
    cd.float4_scaled_mm(a, w, out_dtype=torch.float32)
  with pytest.raises(RuntimeError, match="CUDA"):
    cd.float4_scaled_mm(a, w)
  with pytest.raises(RuntimeError, match="columns"):
    cd.float4_linear(torch.zeros(2, 32, dtype=torch.bfloat16), w)
  with pytest.raises(RuntimeError, match="bfloat16"):
    cd.float4_linear(torch.zeros(2, 64), w)


def test_norm_refusals():
  x = torch.zeros(2, 3, 64)
  call = cd.gated_residual_norm
  for kw, match in ((dict(norm="batch"), "norm must be"), (dict(y=x, post_norm="batch"), "post_norm must be"), (dict(gate=x[:, 0]), "missing"),
                    (dict(residual_scale=0.5), "missing"), (dict(y=x, post_weight=x[0, 0]), "post_norm"), (dict(norm=None), "nothing"),
                    (dict(y=x, norm=None, weight=x[0, 0]), "nothing"), (dict(scale=x[:, 0]), "together"), (dict(quantize="int4"), "format"),
                    (dict(y=x), "CUDA")):
    with pytest.raises((RuntimeError, ValueError), match=match):
      call(x, **kw)
  with pytest.raises(RuntimeError, match="multiple of 32"):
    call(torch.zeros(2, 3, 40), quantize="nvfp4")
  with pytest.raises(RuntimeError, match="1 to 16384"):
    call(torch.zeros(1, 1, 16385))
  with pytest.raises(RuntimeError, match="float32, bfloat16"):
    call(torch.zeros(2, 3, 64, dtype=torch.float64))
  with pytest.raises(RuntimeError, match="batch, tokens"):
    call(torch.zeros(64))


def test_cross_attention_refusals():
  h = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype)
  q, k = h(2, 4, 6, 64), h(2, 5, 3, 64)
  for args, kw, match in (((q, k, h(2, 6, 3, 64)), {}, "got"), ((q, h(2, 5, 4, 64), h(2, 5, 4, 64)), {}, "multiple of the key heads"),
                          ((q.float(), k.float(), k.float()), {}, "bfloat16"), ((q, k.half(), k.half()), {}, "bfloat16"),
                          ((h(2, 4, 6, 60), h(2, 5, 3, 60), h(2, 5, 3, 60)), {}, "multiple of 8"),
                          ((h(2, 4, 6, 136), h(2, 5, 3, 136), h(2, 5, 3, 136)), {}, "at most 128"),
                          ((q, k, k, torch.ones(2, 4, dtype=torch.bool)), {}, "key_mask"), ((q, k, k, torch.ones(2, 5)), {}, "key_mask"),
                          ((q, k, k), dict(scale=0.0), "scale"), ((q, k, k), dict(scale=float("nan")), "scale"), ((q, k, k), {}, "CUDA")):
    with pytest.raises(RuntimeError, match=match):
      cd.cross_attention(*args, **kw)


def test_c_entries_refuse_without_a_gpu():
  L = nat.lib()
  assert L.cdb_fp4_quant_rows(None, 1, 32, 32, 1, 0, None, None, None, None) == 1
  assert L.cdb_fp4_quant_rows(None, 0, 32, 32, 1, 0, None, None, None, None) == 0
  assert L.cdb_fp4_dequant_rows(None, None, None, 1, 33, 0, None, 1, None) == 1
  assert L.cdb_fp4_gemm(None, None, None, None, 1, 8, 32, 8, 0, 1, 0, None, None) == 1
  assert L.cdb_fp4_linear(None, 32, None, None, None, 1, 8, 32, 8, 0, 1, 0, None, 0, None, None) == 1
  assert L.cdb_gated_residual_norm(None, 1, None) == 1
  args = nat.NormArgs(dim=64, batch=1, tokens=1, norm=1, format=-1)
  assert L.cdb_gated_residual_norm(ctypes.byref(args), 1, None) == 1
  assert L.cdb_cross_attention(None, None, None, None, 0, None, 1, 1, 1, 1, 1, 64, 1.0, 1, None, 0, None, None) == 1
  assert L.cdb_cross_attention_workspace_bytes(1, 1, 0, 1, 1, 64, 0) == 0
  assert L.cdb_cross_attention_workspace_bytes(2, 4096, 512, 24, 24, 128, 1) > 0
  assert L.cdb_tuning_set_fp4_tile(0, 256) == 1 and L.cdb_tuning_set_fp4_tile(1, 64) == 1 and L.cdb_tuning_set_fp4_tile(0, 0) == 0


def test_config_takes_the_four_bit_types():
  for name in ("nvfp4_per_row", "mxfp4", "MXFP4"):
    assert cd.QuantizeConfig(quant_type=name).quant_type == name.lower()
  with pytest.raises(NotImplementedError):
    cd.QuantizeConfig(quant_type="nvfp4")  # one scale per tensor: not what is built
  assert cd.load_quantize_config({"quantize_config": {"quant_type": "nvfp4_per_row"}}).quant_type == "nvfp4_per_row"


def test_four_bit_linears_are_selected_by_their_own_shapes(monkeypatch):
  seen = []
  monkeypatch.setattr(float4.Float4Linear, "from_linear", classmethod(lambda cls, lin, fmt: seen.append((tuple(lin.weight.shape), fmt)) or torch.nn.Identity()))
  m = torch.nn.Sequential(torch.nn.Linear(64, 32), torch.nn.Linear(48, 32), torch.nn.Linear(64, 20)).to(torch.bfloat16)
  cd.quantize(m, cd.QuantizeConfig(quant_type="mxfp4", regional_quantize=False))
  assert seen == [((32, 64), "mxfp4")]  # 48 columns are no whole block of 32, 20 rows no multiple of 8


def test_encoder_attention_with_a_prompt_mask_on_cpu():
  from cache_dit_b200.synthetic.layers import encoder_attention
  g = torch.Generator().manual_seed(0)
  q, k, v = (torch.randn(3, n, 2, 16, generator=g) for n in (5, 7, 7))
  mask = torch.arange(7)[None] < torch.tensor([7, 3, 0])[:, None]
  v[~mask] = float("nan")
  got = encoder_attention(q, k, v, mask)
  for i, n in ((0, 7), (1, 3)):
    alone = encoder_attention(q[i:i + 1], k[i:i + 1, :n], v[i:i + 1, :n])
    assert torch.allclose(got[i], alone[0], atol=1e-6)
  assert (got[2] == 0).all()


def test_latched_codes_name_the_operator():
  for code, name in ((24, "4-bit product"), (36, "cross attention"), (13, "FP8 GEMM")):
    with pytest.raises(nat.DeviceTimeoutError, match=name):
      nat.raise_on_device_status(code, 0)
