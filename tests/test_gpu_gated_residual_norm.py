"""`gated_residual_norm` against its formula in 64 bits."""
import pytest
import torch

import cache_dit_b200 as cd

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _formula(x, y, gate, residual_scale, post, pw, pb, norm, w, b, scale, shift, eps=1e-6):
  d = lambda t: None if t is None else t.double()
  row = lambda t: d(t).unsqueeze(1) if t.dim() == 2 else d(t)

  def normed(v, kind):
    if kind == "layer":
      v = v - v.mean(-1, keepdim=True)
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + eps)

  x2 = d(x)
  if y is not None:
    v = d(y)
    if post is not None:
      v = normed(v, post) * (1 if pw is None else d(pw)) + (0 if pb is None else d(pb))
    x2 = x2 + residual_scale * (1 if gate is None else row(gate)) * v
  if norm is None:
    return x2, None
  h = normed(x2, norm) * (1 if w is None else d(w)) + (0 if b is None else d(b))
  if scale is not None:
    h = h * (1 + row(scale)) + row(shift)
  return x2, h


def _within(got, want, dtype, dim):
  """One rounding to the output type (half a step), over fp32 work: sums of `dim` terms in registers and trees of at
  most 64 + 13 additions (2^-24 each, on sums of squares and of magnitudes), a reciprocal root within 2^-22, and a dozen
  further operations on values no larger than the largest of the row."""
  top = want.abs().amax(-1, keepdim=True).clamp(min=1.0)
  fp32 = (77 + 24) * 2.0**-24 * top * 4
  tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
  bad = (got.double() - want).abs() > torch.finfo(dtype).eps / 2 * want.abs() * (1 + 2.0**-10) + fp32 + tiny
  assert not bad.any(), ((got.double() - want).abs() / want.abs().clamp(min=1e-3)).max().item()


def _case(batch, tokens, dim, dtype, seed=0):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s, std=1.0, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to("cuda", dtype)
  return dict(x=r(batch, tokens, dim, std=2.0, mean=0.3), y=r(batch, tokens, dim), gate=r(batch, dim, std=0.5), pw=r(dim, std=0.1, mean=1.0),
              pb=r(dim, std=0.1), w=r(dim, std=0.1, mean=1.0), b=r(dim, std=0.1), scale=r(batch, dim, std=0.3), shift=r(batch, dim, std=0.3))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("norm", [None, "rms", "layer"])
@pytest.mark.parametrize("batch,tokens,dim", [(1, 1, 8), (2, 3, 264), (1, 5, 1000), (3, 7, 1536), (1, 130, 2304), (2, 33, 5120)])
def test_against_the_formula(batch, tokens, dim, norm, post, dtype):
  c = _case(batch, tokens, dim, dtype)
  affine = dim != 1000
  pw, pb = (c["pw"], c["pb"]) if post is not None and affine else (None, None)
  w, b, scale, shift = (c["w"], c["b"], c["scale"], c["shift"]) if norm is not None and affine else (None, ) * 4
  got_x, got_h = cd.gated_residual_norm(c["x"], c["y"], c["gate"], residual_scale=0.7, post_norm=post, post_weight=pw, post_bias=pb,
                                        norm=norm, weight=w, bias=b, scale=scale, shift=shift)
  want_x, want_h = _formula(c["x"], c["y"], c["gate"], 0.7, post, pw, pb, norm, w, b, scale, shift)
  _within(got_x, want_x, dtype, dim)
  if norm is None:
    assert got_h is None
  else:
    _within(got_h, want_h, dtype, dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [1, 2, 7, 31, 63, 255, 777, 1023, 1025, 4099, 8192, 12288, 16383, 16384])
def test_every_width(dim, dtype):
  c = _case(2, 5, dim, dtype, seed=dim)
  got = cd.gated_residual_norm(c["x"], c["y"], c["gate"], post_norm="rms", post_weight=c["pw"], norm="layer", weight=c["w"], bias=c["b"])
  want = _formula(c["x"], c["y"], c["gate"], 1.0, "rms", c["pw"], None, "layer", c["w"], c["b"], None, None)
  for a, b in zip(got, want):
    _within(a, b, dtype, dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_norm_alone_returns_x_itself(norm, dtype):
  c = _case(2, 9, 640, dtype)
  x2, h = cd.gated_residual_norm(c["x"], norm=norm, scale=c["scale"], shift=c["shift"])
  assert x2 is c["x"]
  _within(h, _formula(c["x"], None, None, 1.0, None, None, None, norm, None, None, c["scale"], c["shift"])[1], dtype, 640)


def test_strides_slices_and_shared_vectors():
  c = _case(3, 20, 512, torch.bfloat16)
  wide = torch.randn(3, 40, 2048, device="cuda").to(torch.bfloat16)
  mod = torch.randn(3, 3 * 512, device="cuda").to(torch.bfloat16)
  for x, y in ((wide[:, :20, 512:1024], c["y"]), (c["x"], wide[:, 20:, 1024:1536]), (wide[:, ::2, 1:513], wide[:, 1::2, 3:515]),
               (c["x"].transpose(1, 2).contiguous().transpose(1, 2), c["y"])):
    args = dict(gate=mod[:, :512], scale=mod[:, 512:1024], shift=mod[:, 1024:])
    got = cd.gated_residual_norm(x, y, norm="layer", **args)
    want = _formula(x, y, args["gate"], 1.0, None, None, None, "layer", None, None, args["scale"], args["shift"])
    for a, b in zip(got, want):
      assert a.is_contiguous()
      _within(a, b, torch.bfloat16, 512)
  one = cd.gated_residual_norm(c["x"], c["y"], mod[0, :512], norm="rms")  # one gate for all batches
  each = cd.gated_residual_norm(c["x"], c["y"], mod[:1, :512].expand(3, 512).contiguous(), norm="rms")
  flat = cd.gated_residual_norm(c["x"].view(60, 512), c["y"].view(60, 512), mod[:1, :512], norm="rms")
  for a, b, f in zip(one, each, flat):
    assert torch.equal(a, b) and torch.equal(a.view(60, 512), f)


@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens,dim", [(1, 1, 32), (2, 65, 96), (1, 300, 1056), (2, 70, 2304), (1, 129, 5120), (1, 3, 16384)])
def test_four_bit_output_is_the_quantisation_of_h(batch, tokens, dim, dtype, fmt):
  c = _case(batch, tokens, dim, dtype)
  args = dict(post_norm="rms", norm="layer", scale=c["scale"], shift=c["shift"])
  x2, h = cd.gated_residual_norm(c["x"], c["y"], c["gate"], **args)
  x2q, q = cd.gated_residual_norm(c["x"], c["y"], c["gate"], quantize=fmt, **args)
  want = cd.float4_quantize_rows(h, fmt)
  assert torch.equal(x2, x2q) and q.shape == h.shape and q.format == fmt
  assert torch.equal(q.codes, want.codes) and torch.equal(q.block_scales, want.block_scales)
  assert q.row_scale is None or torch.equal(q.row_scale, want.row_scale)
  assert torch.equal(q.codes, cd.gated_residual_norm(c["x"], c["y"], c["gate"], quantize=fmt, **args)[1].codes)


def test_rows_with_infinities_and_nan_stay_to_themselves():
  c = _case(1, 12, 512, torch.bfloat16)
  clean = cd.gated_residual_norm(c["x"], c["y"], c["gate"], norm="layer")
  c["x"][0, 3, 7] = float("inf")
  c["y"][0, 8, 500] = float("nan")
  got = cd.gated_residual_norm(c["x"], c["y"], c["gate"], norm="layer")
  rest = [i for i in range(12) if i not in (3, 8)]
  for a, b in zip(got, clean):
    assert torch.equal(a[0, rest], b[0, rest])
  assert torch.isnan(got[1][0, [3, 8]]).all()


def test_large_mean_loses_nothing():
  """A row whose mean is thousands of standard deviations: two-pass statistics keep the variance."""
  g = torch.Generator().manual_seed(0)
  x = (4096.0 + torch.randn(1, 8, 1024, generator=g)).cuda()
  got = cd.gated_residual_norm(x, norm="layer")[1]
  want = _formula(x, None, None, 1.0, None, None, None, "layer", None, None, None, None)[1]
  # the mean itself is off by at most 77 * 2^-24 * 4096 = 0.019 and shifts every element of the row alike
  assert ((got.double() - want) - (got.double() - want).mean(-1, keepdim=True)).abs().max() < 1e-4
  assert (got.double() - want).abs().max() < 0.02
