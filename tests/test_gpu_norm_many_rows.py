"""`gated_residual_norm` with many rows for every thread block: the rows after a block's first one, where the next row's loads,
the alternating reduction words and the padding of 4-bit scales come in."""
import pytest
import torch

import cache_dit_b200 as cd
from tests.test_gpu_gated_residual_norm import DTYPES, _case, _formula, _within

pytestmark = pytest.mark.gpu

# A B200 holds at most 8 blocks of 256 threads per SM, 1184 in all, of 8 rows (up to 1024 elements), 4, 2 or 1 row each.
SHAPES = [(3, 6007, 640), (2, 5501, 1536), (1, 4099, 2304), (2, 2503, 5120), (1, 2411, 8192), (1, 2400, 16384), (3, 20011, 24), (5, 4001, 64),
          (3, 5003, 1001), (2, 1709, 4097)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("post", [None, "rms", "layer"])
@pytest.mark.parametrize("batch,tokens,dim", SHAPES)
def test_every_row(batch, tokens, dim, post, norm, dtype):
  c = _case(batch, tokens, dim, dtype, seed=dim)
  pw, pb = (None, None) if post is None else (c["pw"], c["pb"])
  got = cd.gated_residual_norm(c["x"], c["y"], c["gate"], residual_scale=0.7, post_norm=post, post_weight=pw, post_bias=pb, norm=norm,
                               weight=c["w"], bias=c["b"], scale=c["scale"], shift=c["shift"])
  for b in range(batch):  # one batch entry at a time: its own gate, scale and shift
    one = {k: v[b:b + 1] if k in ("x", "y", "gate", "scale", "shift") else v for k, v in c.items()}
    want = _formula(one["x"], one["y"], one["gate"], 0.7, post, pw, pb, norm, one["w"], one["b"], one["scale"], one["shift"])
    for a, w in zip(got, want):
      _within(a[b:b + 1], w, dtype, dim)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt", ["nvfp4", "mxfp4"])
@pytest.mark.parametrize("post", [None, "layer"])
@pytest.mark.parametrize("batch,tokens,dim", [(3, 6007, 640), (2, 5501, 1536), (1, 4099, 2304), (2, 2503, 5120), (1, 2400, 16384),
                                              (3, 20011, 32)])
def test_four_bits_of_every_row(batch, tokens, dim, post, fmt, dtype):
  c = _case(batch, tokens, dim, dtype, seed=dim)
  args = dict(post_norm=post, norm="layer", weight=c["w"], scale=c["scale"], shift=c["shift"])
  x2, h = cd.gated_residual_norm(c["x"], c["y"], c["gate"], **args)
  x2q, q = cd.gated_residual_norm(c["x"], c["y"], c["gate"], quantize=fmt, **args)
  want = cd.float4_quantize_rows(h, fmt)
  assert torch.equal(x2, x2q)
  assert torch.equal(q.codes, want.codes) and torch.equal(q.block_scales, want.block_scales)
  assert q.row_scale is None or torch.equal(q.row_scale, want.row_scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens,dim", [(3, 6007, 640), (2, 2503, 5120), (3, 5003, 1001)])
def test_the_norm_alone_and_the_sum_alone(batch, tokens, dim, dtype):
  c = _case(batch, tokens, dim, dtype, seed=1)
  _within(cd.gated_residual_norm(c["x"], norm="layer", weight=c["w"])[1],
          _formula(c["x"], None, None, 1.0, None, None, None, "layer", c["w"], None, None, None)[1], dtype, dim)
  x2, h = cd.gated_residual_norm(c["x"], c["y"], c["gate"], norm=None)
  assert h is None
  _within(x2, _formula(c["x"], c["y"], c["gate"], 1.0, None, None, None, None, None, None, None, None)[0], dtype, dim)
