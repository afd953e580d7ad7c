"""4-bit linears and padded prompts under the cache engine, with and without CUDA-graph replay of the block segments."""
import pytest
import torch

import cache_dit_b200 as cd
from cache_dit_b200 import _native

pytestmark = pytest.mark.gpu


def _build(shape):
  from cache_dit_b200 import synthetic as sy
  torch.manual_seed(0)
  if shape == "wan":
    model = sy.WanTransformer3DModel(num_layers=4, dim=256, heads=2, ffn_dim=512, in_channels=16, text_dim=64, axes_dims_rope=(44, 42, 42),
                                     time_scale=1.0, modulation_init_std=0.02)
    inputs = sy.WanTransformer3DModel.example_inputs(batch=3, frames=3, height=7, width=13, text_tokens=40, in_channels=16, text_dim=64)
    pipe = sy.WanDenoisePipeline
  else:
    kw = dict(dim=256, heads=4, in_channels=16, joint_attention_dim=64, axes_dims_rope=(8, 28, 28), time_scale=1.0, modulation_init_std=0.02)
    sizes = dict(batch=2, height=208, width=208, text_tokens=17, in_channels=16, joint_attention_dim=64)
    if shape == "flux":
      model = sy.FluxTransformer2DModel(num_layers=2, num_single_layers=2, pooled_projection_dim=32, **kw)
      inputs, pipe = sy.FluxTransformer2DModel.example_inputs(pooled_projection_dim=32, **sizes), sy.FluxDenoisePipeline
    else:
      model = sy.QwenImageTransformer2DModel(num_layers=3, **kw)
      inputs, pipe = sy.QwenImageTransformer2DModel.example_inputs(**sizes), sy.QwenImageDenoisePipeline
  return pipe(model.to("cuda", torch.bfloat16).eval().requires_grad_(False), inputs)


def _masks():
  at = torch.arange(40, device="cuda")[None]
  return [at < torch.tensor(n, device="cuda")[:, None] for n in ((40, 13, 1), (5, 40, 0))]


def _generations(shape, quant_type, masked, graphs, steps=8):
  """Latents and cached steps of three generations; with masks, the last one's prompts are padded otherwise."""
  pipe = _build(shape)
  quantize = None if quant_type is None else cd.QuantizeConfig(quant_type=quant_type)
  cd.enable_cache(pipe, cache_config=cd.DBCacheConfig(Fn_compute_blocks=1, max_warmup_steps=2, residual_diff_threshold=0.3),
                  quantize_config=quantize)
  if graphs:
    assert cd.enable_cuda_graphs(pipe, warmup_calls=1) >= 1
  out = []
  try:
    for i in range(3):
      if masked:
        pipe.inputs = dict(pipe.inputs, encoder_attention_mask=_masks()[i // 2])
      out.append((pipe(num_inference_steps=steps).clone(), list(pipe.transformer._cached_steps)))
    torch.cuda.synchronize()
    replays = sum(r.replays for r in cd.graph_runners(pipe))
    assert (replays > 0) == graphs
  finally:
    cd.disable_cache(pipe)
  assert _native.gemm_device_status(torch.device("cuda")) == 0
  return out


@pytest.mark.parametrize("shape,quant_type,masked", [("wan", None, True), ("wan", "float8_per_row", True), ("wan", "nvfp4_per_row", True),
                                                     ("wan", "mxfp4", True), ("wan", "nvfp4_per_row", False), ("flux", "nvfp4_per_row", False),
                                                     ("flux", "mxfp4", False), ("qwen_image", "mxfp4", False)])
def test_replayed_segments_equal_eager_ones(shape, quant_type, masked):
  eager, replayed = (_generations(shape, quant_type, masked, graphs) for graphs in (False, True))
  for (a, steps_a), (b, steps_b) in zip(eager, replayed):
    assert torch.isfinite(a).all() and steps_a == steps_b and steps_a
    assert torch.equal(a, b)
  assert torch.equal(eager[0][0], eager[1][0])  # a second generation starts afresh
  if masked:
    assert not torch.equal(eager[1][0], eager[2][0])


@pytest.mark.parametrize("quant_type", [None, "nvfp4_per_row", "mxfp4"])
def test_what_lies_in_the_padding_has_no_effect(quant_type):
  """NaN prompt tokens behind each prompt's end pass through the text embedding and the key and value projections, and end
  at the mask."""
  model = _build("wan").transformer
  if quant_type is not None:
    cd.quantize(model, cd.QuantizeConfig(quant_type=quant_type))
  inputs = dict(_build("wan").inputs, timestep=torch.full((3, ), 0.5, device="cuda"))
  for mask in _masks():
    dirty = torch.where(mask[:, :, None], inputs["encoder_hidden_states"], float("nan"))
    with torch.no_grad():
      want = model(**inputs, encoder_attention_mask=mask)
      got = model(**dict(inputs, encoder_hidden_states=dirty), encoder_attention_mask=mask)
    assert torch.isfinite(got).all() and torch.equal(got, want)
