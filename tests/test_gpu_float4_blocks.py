"""The 4-bit linears, the fused norms and the cross attention together: as a module, in a Wan-shape transformer, captured into
a graph, on streams of their own."""
import copy

import pytest
import torch
import torch.nn.functional as F

import cache_dit_b200 as cd
from cache_dit_b200 import _native
from cache_dit_b200.quantization import float4
from cache_dit_b200.synthetic.wan import WanTransformer3DModel

pytestmark = pytest.mark.gpu
FORMATS = ["nvfp4", "mxfp4"]


def _dense(linear4):
  """A linear with the values the 4-bit weight stands for."""
  w = cd.float4_dequantize_rows(linear4.weight_rows, torch.float32)
  return w, None if linear4.bias is None else linear4.bias.float()


@pytest.mark.parametrize("fmt", FORMATS)
def test_linear_module(fmt, tmp_path):
  torch.manual_seed(0)
  lin = torch.nn.Linear(320, 264).to("cuda", torch.bfloat16)
  m = cd.Float4Linear.from_linear(lin, fmt)
  x = torch.randn(2, 37, 320, device="cuda").to(torch.bfloat16)
  with torch.no_grad():
    y = m(x)
    w, b = _dense(m)
    xq = cd.float4_dequantize_rows(cd.float4_quantize_rows(x, fmt), torch.float32)
    want = F.linear(xq.double(), w.double(), b.double())
    # fp32 accumulation of 320 products (20 blocks), one rounding to bf16
    assert ((y.double() - want).abs() <= 2.0**-8 * want.abs() + 24 * 2.0**-23 * F.linear(xq.abs().double(), w.abs().double()) + 1e-6).all()
    assert torch.equal(m.forward_quantized(cd.float4_quantize_rows(x, fmt)), y)
    torch.save(m.state_dict(), tmp_path / "m.pt")
    other = cd.Float4Linear.from_linear(torch.nn.Linear(320, 264).to("cuda", torch.bfloat16), fmt)
    other.load_state_dict(torch.load(tmp_path / "m.pt"))
    assert torch.equal(other(x), y)
    assert torch.equal(copy.deepcopy(m)(x), y)
  with pytest.raises(RuntimeError, match="no backward pass"):
    m(x.requires_grad_())


def _wan(seed=0, **kw):
  torch.manual_seed(seed)
  m = WanTransformer3DModel(num_layers=2, dim=256, heads=4, ffn_dim=512, text_dim=64, axes_dims_rope=(24, 20, 20), **kw)
  return m.to("cuda", torch.bfloat16).eval()


def _inputs(batch=2, text=24):
  d = WanTransformer3DModel.example_inputs(batch=batch, frames=3, height=5, width=7, text_tokens=text, text_dim=64)
  d["timestep"] = torch.full((batch, ), 0.5, device="cuda", dtype=torch.bfloat16)
  return d


class _Reference(torch.nn.Module):
  """A 4-bit linear through dequantised operands and a dense product."""

  def __init__(self, lin4):
    super().__init__()
    self.lin4 = lin4

  def forward(self, x):
    w, b = _dense(self.lin4)
    xq = cd.float4_dequantize_rows(cd.float4_quantize_rows(x.contiguous(), self.lin4.format), torch.float32)
    return F.linear(xq, w, b).to(torch.bfloat16)


def _swap(module, make):
  for name, child in list(module.named_children()):
    if isinstance(child, cd.Float4Linear):
      setattr(module, name, make(child))
    else:
      _swap(child, make)
  return module


@pytest.mark.parametrize("fmt,quant_type", [("nvfp4", "nvfp4_per_row"), ("mxfp4", "mxfp4")])
@torch.no_grad()
def test_wan_shape_in_four_bits(fmt, quant_type):
  """The fused path (norms writing 4 bits, GELU in the product) against the same 4-bit linears one by one around eager norms."""
  model = _wan()
  cd.quantize(model, cd.QuantizeConfig(quant_type=quant_type))
  assert sum(isinstance(m, cd.Float4Linear) for m in model.modules()) == 2 * 10
  inputs = _inputs()
  fused = model(**inputs)
  plain = _swap(copy.deepcopy(model), _Reference)(**inputs)
  # the same quantised weights; activations differ by bf16 roundings of eager intermediates, which move a code now and then
  # (a step of a code is up to a sixth of its block's largest): 20 linears, a few per mille each
  assert (fused.float() - plain.float()).norm() <= 0.05 * plain.float().norm()
  assert _native.gemm_device_status(torch.device("cuda")) == 0


@pytest.mark.parametrize("quant_type", ["nvfp4_per_row", "mxfp4"])
@pytest.mark.parametrize("shape", ["flux", "qwen_image"])
@torch.no_grad()
def test_joint_attention_shapes_in_four_bits(shape, quant_type):
  """Blocks that the fused residual norms do not reach: modulation rows, joint attention and concatenated inputs, against
  the same 4-bit linears one by one, and under the cache engine."""
  from cache_dit_b200.synthetic import FluxDenoisePipeline, FluxTransformer2DModel, QwenImageDenoisePipeline, QwenImageTransformer2DModel
  torch.manual_seed(0)
  kw = dict(dim=256, heads=4, in_channels=16, joint_attention_dim=64, axes_dims_rope=(8, 28, 28), time_scale=1.0,
            modulation_init_std=0.02)
  sizes = dict(batch=2, height=208, width=208, text_tokens=17, in_channels=16, joint_attention_dim=64)
  if shape == "flux":
    model = FluxTransformer2DModel(num_layers=2, num_single_layers=2, pooled_projection_dim=32, **kw).cuda()
    inputs, pipe_cls = FluxTransformer2DModel.example_inputs(pooled_projection_dim=32, **sizes), FluxDenoisePipeline
  else:
    model = QwenImageTransformer2DModel(num_layers=3, **kw).cuda()
    inputs, pipe_cls = QwenImageTransformer2DModel.example_inputs(**sizes), QwenImageDenoisePipeline
  model = model.to(torch.bfloat16).eval().requires_grad_(False)
  cd.quantize(model, cd.QuantizeConfig(quant_type=quant_type))
  assert any(isinstance(m, cd.Float4Linear) for m in model.modules())
  t = torch.full((2, ), 0.5, device="cuda")
  fused = model(**inputs, timestep=t)
  plain = _swap(copy.deepcopy(model), _Reference)(**inputs, timestep=t)
  # as in the Wan shape: the same weights, a code of an activation moved now and then
  assert (fused.float() - plain.float()).norm() <= 0.05 * plain.float().norm()
  pipe = pipe_cls(model, inputs)
  cd.enable_cache(pipe, cache_config=cd.DBCacheConfig(Fn_compute_blocks=1, max_warmup_steps=3, residual_diff_threshold=0.15))
  try:
    assert torch.isfinite(pipe(num_inference_steps=6)).all()
  finally:
    cd.disable_cache(pipe)
  assert _native.gemm_device_status(torch.device("cuda")) == 0


@torch.no_grad()
def test_wan_shape_with_padded_prompts():
  """Each prompt of a padded batch gives what it gives alone, whatever lies in the padding."""
  model = _wan(1)
  inputs = _inputs(batch=3, text=40)
  lengths = torch.tensor([40, 13, 1], device="cuda")
  mask = torch.arange(40, device="cuda")[None] < lengths[:, None]
  noisy = dict(inputs)
  noisy["encoder_hidden_states"] = torch.where(mask[:, :, None], inputs["encoder_hidden_states"], 100.0).to(torch.bfloat16)
  got = model(**noisy, encoder_attention_mask=mask)
  assert torch.equal(got, model(**inputs, encoder_attention_mask=mask))
  for i, n in enumerate(lengths.tolist()):
    one = dict(hidden_states=inputs["hidden_states"][i:i + 1], encoder_hidden_states=inputs["encoder_hidden_states"][i:i + 1, :n],
               timestep=inputs["timestep"][i:i + 1], video_ids=inputs["video_ids"])
    alone = model(**one)
    # library attention on one side, this package's on the other, both bf16: a few roundings through two blocks
    assert (got[i].float() - alone[0].float()).norm() <= 0.02 * alone[0].float().norm()


@torch.no_grad()
def test_unquantised_and_fp8_blocks_keep_their_results():
  """Without 4-bit linears the block is the sequence it always was."""
  model = _wan(2)
  block, inputs = model.blocks[0], _inputs(batch=1)
  x = torch.randn(1, 105, 256, device="cuda").to(torch.bfloat16)
  enc = torch.randn(1, 24, 256, device="cuda").to(torch.bfloat16)
  temb = torch.randn(1, 6, 256, device="cuda").to(torch.bfloat16)
  from cache_dit_b200.synthetic import layers as ly
  rope = ly.RopeCache().get((inputs["video_ids"], ), model.axes_dims_rope, torch.bfloat16)

  def sequence():
    mod = block.scale_shift_table.to(temb.dtype) + temb
    s1, c1, g1, s2, c2, g2 = mod.unbind(dim=1)
    a = block.attn1
    q, k, v = ly.norm_modulate_linears(x, s1, c1, (a.to_q, a.to_k, a.to_v))
    o = ly.joint_attention(((q, a.norm_q), ), ((k, a.norm_k), ), (v, ), rope, a.heads, None, across_heads=True)
    h = ly.gated_add(x, g1, a.to_out[0](o))
    a = block.attn2
    heads = lambda t: t.unflatten(-1, (a.heads, a.head_dim)).transpose(1, 2)
    q, k, v = heads(a.norm_q(a.to_q(block.norm2(h)))), heads(a.norm_k(a.to_k(enc))), heads(a.to_v(enc))
    h = h + a.to_out[0](F.scaled_dot_product_attention(q, k, v).transpose(1, 2).flatten(2))
    act = ly.gelu_in_product()
    (f, ) = ly.norm_modulate_linears(h, s2, c2, (block.ffn.net[0].proj, ), gelu_last=act)
    return ly.gated_add(h, g2, ly.gelu_linear(f, block.ffn.net[2], activated=act))

  assert torch.equal(block(x, enc, temb, rope), sequence())
  cd.quantize(model, cd.QuantizeConfig(quant_type="float8_per_row"))
  assert torch.equal(block(x, enc, temb, rope), sequence())


def _chain(x, y, gate, w, q, k, mask):
  x2, h = cd.gated_residual_norm(x, y, gate, norm="rms", quantize="nvfp4")
  out = cd.float4_scaled_mm(h, w)
  return x2, out, cd.cross_attention(q, k, k, mask), cd.float4_linear(out, w)


@torch.no_grad()
def test_captured_replayed_and_beside_each_other():
  """A chain of the operators captured twice, the graphs replayed in turn and on two streams at once, equals the eager calls:
  no workspace is shared between captures."""
  torch.manual_seed(3)
  r = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
  w = cd.float4_quantize_rows(r(512, 512))
  sets = [(r(1, 300, 512), r(1, 300, 512), r(1, 512), w, r(2, 3, 8, 64), r(2, 3000, 2, 64), torch.rand(2, 3000, device="cuda") < 0.5)
          for _ in range(2)]
  want = [_chain(*s) for s in sets]
  graphs, outs = [], []
  for s in sets:
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
      _chain(*s)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
      outs.append(_chain(*s))
    graphs.append(g)
  streams = [torch.cuda.Stream(), torch.cuda.Stream()]
  for _ in range(3):
    for out in outs:
      for t in out:
        t.fill_(float("nan"))
    torch.cuda.synchronize()
    for g, st in zip(graphs, streams):
      with torch.cuda.stream(st):
        for _ in range(4):
          g.replay()
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
      assert all(torch.equal(a, b) for a, b in zip(got, ref))


@torch.no_grad()
def test_on_a_stream_of_its_own():
  torch.manual_seed(4)
  x = torch.randn(1, 700, 1024, device="cuda").to(torch.bfloat16)
  w = cd.float4_quantize_rows(torch.randn(1024, 1024, device="cuda").to(torch.bfloat16))
  want = cd.float4_linear(cd.gated_residual_norm(x, x)[1], w)
  st = torch.cuda.Stream()
  with torch.cuda.stream(st):
    torch.cuda._sleep(20_000_000)  # whatever ran on another stream would be ahead of the copy below
    y = x * 1
    got = cd.float4_linear(cd.gated_residual_norm(y, y)[1], w)
  st.synchronize()
  assert torch.equal(got, want)


@torch.no_grad()
def test_repeated_calls_are_bitwise_equal():
  torch.manual_seed(5)
  r = lambda *s: torch.randn(*s, device="cuda").to(torch.bfloat16)
  args = (r(2, 500, 640), r(2, 500, 640), r(2, 640), cd.float4_quantize_rows(r(640, 640)), r(2, 2, 16, 128), r(2, 5000, 4, 128),
          torch.rand(2, 5000, device="cuda") < 0.9)
  first = _chain(*args)
  for _ in range(5):
    assert all(torch.equal(a, b) for a, b in zip(first, _chain(*args)))
