"""`cross_attention` against its formula in 64 bits."""
import math

import pytest
import torch

import cache_dit_b200 as cd
from cache_dit_b200 import _native

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16]


def _formula(q, k, v, mask=None, scale=None):
  b, sq, h, d = q.shape
  g = h // k.shape[2]
  qd, kd, vd = q.double(), k.double().repeat_interleave(g, 2), v.double().repeat_interleave(g, 2)
  if mask is not None:
    kd = torch.where(mask[:, :, None, None], kd, 0.0)
    vd = torch.where(mask[:, :, None, None], vd, 0.0)
  s = torch.einsum("bqhd,bkhd->bhqk", qd, kd) * (d**-0.5 if scale is None else scale)
  if mask is not None:
    s = s.masked_fill(~mask[:, None, None, :], -math.inf)
  p = torch.softmax(s, dim=-1).nan_to_num(0.0) if mask is not None else torch.softmax(s, dim=-1)
  return torch.einsum("bhqk,bkhd->bqhd", p, vd), torch.einsum("bhqk,bkhd->bqhd", p, vd.abs()), s


def _check(got, q, k, v, mask=None, scale=None):
  want, magnitude, s = _formula(q, k, v, mask, scale)
  # P is rounded to the type (half a step each, with l unrounded); the scores' fp32 products and the exponential's
  # argument are off by about (d + 4) 2^-24 of sum |q k| scale, ex2.approx by 2^-22; the sum over keys in fp32 (the tensor
  # core may truncate: a whole step each 16 keys); one rounding of the result
  d, keys = q.shape[-1], k.shape[1]
  eps = torch.finfo(q.dtype).eps / 2
  g = q.shape[2] // k.shape[2]
  kk = k if mask is None else torch.where(mask[:, :, None, None], k, torch.zeros_like(k))
  biggest = torch.einsum("bqhd,bkhd->bhqk", q.double().abs(), kk.double().abs().repeat_interleave(g, 2)).amax().item()
  rel = eps + (d + 4) * 2.0**-23 * biggest * (d**-0.5 if scale is None else scale) + 2.0**-20 + (keys / 16 + 8) * 2.0**-23
  # fp16 P below 2^-14 of the running maximum's 2^8 window is subnormal: absolute 2^-25 per key against l >= 1
  floor = keys * 2.0**-25 * v[torch.isfinite(v)].abs().max().double().item() if q.dtype == torch.float16 else 0.0
  tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
  err = (got.double() - want).abs()
  assert torch.isfinite(got).all()
  assert (err <= rel * magnitude + eps * want.abs() + floor + tiny).all(), (err / (rel * magnitude + eps * want.abs() + floor + tiny)).max().item()
  assert _native.gemm_device_status(torch.device("cuda")) == 0


def _qkv(b, sq, skv, h, hk, d, dtype, seed=0, std=1.0):
  g = torch.Generator().manual_seed(seed)
  r = lambda *s: (torch.randn(*s, generator=g) * std).to("cuda", dtype)
  return r(b, sq, h, d), r(b, skv, hk, d), torch.randn(b, skv, hk, d, generator=g).to("cuda", dtype)


SHAPES = [(1, 1, 1, 1, 1, 8), (1, 128, 128, 1, 1, 64), (1, 128, 128, 1, 1, 128), (1, 129, 127, 2, 2, 64), (2, 257, 333, 3, 3, 128),
          (1, 1000, 77, 4, 4, 96), (2, 640, 512, 2, 2, 128), (3, 40, 1, 2, 1, 72), (1, 256, 1024, 1, 1, 40), (2, 700, 226, 6, 2, 64),
          (1, 300, 260, 12, 4, 80), (1, 5, 700, 40, 8, 112), (2, 1, 4000, 8, 2, 128), (1, 1, 9000, 5, 1, 64), (4, 3, 129, 7, 7, 16),
          (1, 33, 2049, 24, 3, 128), (1, 2, 300, 192, 1, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("b,sq,skv,h,hk,d", SHAPES)
def test_against_the_formula(b, sq, skv, h, hk, d, dtype):
  q, k, v = _qkv(b, sq, skv, h, hk, d, dtype)
  _check(cd.cross_attention(q, k, v), q, k, v)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["padded", "holes", "one", "none_in_some", "middle"])
@pytest.mark.parametrize("b,sq,skv,h,hk,d", [(3, 200, 333, 2, 2, 64), (3, 1, 2500, 8, 2, 128), (3, 300, 128, 2, 1, 96), (3, 70, 1111, 1, 1, 128)])
def test_masks(b, sq, skv, h, hk, d, kind, dtype):
  q, k, v = _qkv(b, sq, skv, h, hk, d, dtype, seed=3)
  g = torch.Generator().manual_seed(1)
  at = torch.arange(skv)
  mask = {"padded": at[None] < torch.tensor([skv, skv // 2 + 1, 5])[:, None], "holes": torch.rand(b, skv, generator=g) < 0.6,
          "one": at[None] == torch.tensor([0, skv - 1, skv // 2])[:, None], "none_in_some": (at[None] < torch.tensor([0, 100, 0])[:, None]),
          "middle": (at[None] >= skv // 3) & (at[None] < torch.tensor([skv // 3 + 2, skv - 1, skv])[:, None])}[kind].cuda()
  dirty_k, dirty_v = k.clone(), v.clone()  # what lies in masked places has no effect
  dirty_k[~mask] = float("nan")
  dirty_v[~mask] = float("inf")
  dirty_v[:, :, :, 0][~mask] = float("nan")
  got = cd.cross_attention(q, dirty_k, dirty_v, mask)
  _check(got, q, k, v, mask)
  assert (got[~mask.any(dim=1)] == 0).all()
  assert torch.equal(got, cd.cross_attention(q, k, v, mask))


@pytest.mark.parametrize("dtype", DTYPES)
def test_growing_maxima_and_large_scores(dtype):
  """Scores that keep growing along the keys (every step rescales), and ones of hundreds."""
  q, k, v = _qkv(1, 200, 1500, 2, 2, 64, dtype, seed=5)
  k = (k.float() * torch.linspace(0.01, 4, 1500, device="cuda")[None, :, None, None]).to(dtype)
  _check(cd.cross_attention(q, k, v), q, k, v)
  _check(cd.cross_attention(q, k.flip(1).contiguous(), v), q, k.flip(1), v)
  _check(cd.cross_attention(q, k, v, scale=0.01), q, k, v, scale=0.01)


def test_strides_and_slices():
  b, sq, skv, h, d = 2, 150, 260, 3, 64
  g = torch.Generator().manual_seed(2)
  qkv = torch.randn(b, sq, 3 * h * d, generator=g).to("cuda", torch.bfloat16)
  enc = torch.randn(b, skv + 9, 2, h, d, generator=g).to("cuda", torch.bfloat16)
  q = qkv[..., h * d:2 * h * d].unflatten(-1, (h, d))
  k, v = enc[:, 9:, 0], enc[:, 9:, 1]
  for qq, kk, vv in ((q, k, v), (q.transpose(1, 2).contiguous().transpose(1, 2), k.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3), v),
                     (q[:, ::2], k[:, ::2], v[:, 1::2]),
                     (q[..., :56], k[..., :56], v[..., 8:])):
    _check(cd.cross_attention(qq, kk, vv), qq, kk, vv)
  odd = torch.randn(b, skv, h, d + 1, device="cuda").to(torch.bfloat16)[..., 1:]  # misaligned rows are copied
  _check(cd.cross_attention(q, odd, odd), q, odd, odd)


def test_many_items_per_cta():
  q, k, v = _qkv(1, 9000, 512, 8, 8, 128, torch.bfloat16, seed=9)
  for _ in range(3):
    got = cd.cross_attention(q, k, v)
  for h in range(8):
    _check(got[:, :, h:h + 1].contiguous(), q[:, :, h:h + 1], k[:, :, h:h + 1], v[:, :, h:h + 1])


def test_no_keys_and_no_queries():
  q, k, v = _qkv(2, 4, 0, 2, 2, 64, torch.bfloat16)
  assert (cd.cross_attention(q, k, v) == 0).all()
  q, k, v = _qkv(2, 0, 5, 2, 2, 64, torch.bfloat16)
  assert cd.cross_attention(q, k, v).shape == (2, 0, 2, 64)
