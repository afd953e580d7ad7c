"""`cross_attention` with several work items for every thread block, where one item hands its stages, accumulators and
output over to the next: full, short and empty prompts in turn, one-tile items, shared heads, split key ranges."""
import pytest
import torch

import cache_dit_b200 as cd
from cache_dit_b200 import _native
from tests.test_gpu_cross_attention import DTYPES, _check, _qkv

pytestmark = pytest.mark.gpu


def _mask(lengths, skv, kind):
  at, n = torch.arange(skv, device="cuda")[None], torch.tensor(lengths, device="cuda")[:, None]
  if kind == "padded":
    return at < n
  keep = (at >= skv - n)  # kept keys at the end, with holes
  return keep & ((at % 7 != 3) | (n <= 7))


def _items(b, sq, h, hk):
  """Work items before any split: two tiles of 128 / g queries of g heads each, g the power of two (up to 32) in the group."""
  g, group = 1, h // hk
  while g < 32 and group % (2 * g) == 0:
    g *= 2
  return b * hk * (group // g) * -(-sq // (2 * (128 // g)))


def _run(b, sq, skv, h, hk, d, lengths, kind, dtype):
  q, k, v = _qkv(b, sq, skv, h, hk, d, dtype, seed=sq + skv)
  mask = _mask(lengths, skv, kind)
  dirty_k, dirty_v = k.clone(), v.clone()  # what lies in masked places has no effect
  dirty_k[~mask] = float("nan")
  dirty_v[~mask] = float("inf")
  got = cd.cross_attention(q, dirty_k, dirty_v, mask)
  for _ in range(3):
    assert torch.equal(got, cd.cross_attention(q, dirty_k, dirty_v, mask))
  assert torch.equal(got, cd.cross_attention(q, k, v, mask))
  assert (got[~mask.any(dim=1)] == 0).all()
  g = h // hk
  for i in range(hk):  # a key head at a time: the 64-bit formula of all heads would be large
    _check(got[:, :, i * g:(i + 1) * g], q[:, :, i * g:(i + 1) * g], k[:, :, i:i + 1], v[:, :, i:i + 1], mask)


# (batch, queries, keys, heads, key heads, kept keys): 1100 queries end in a pair with one tile
SHAPES = [(4, 1100, 333, 24, 24, (333, 0, 5, 200)), (4, 1000, 333, 24, 24, (0, 0, 128, 129)), (3, 600, 700, 24, 6, (1, 700, 0)),
          (5, 120, 1000, 64, 2, (1000, 0, 0, 3, 640)), (6, 300, 130, 20, 20, (0, 130, 0, 128, 2, 0)), (2, 2400, 257, 10, 10, (257, 1))]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128, 40, 72])
@pytest.mark.parametrize("kind", ["padded", "holes"])
@pytest.mark.parametrize("b,sq,skv,h,hk,lengths", SHAPES)
def test_masked(b, sq, skv, h, hk, lengths, kind, d, dtype):
  _run(b, sq, skv, h, hk, d, lengths, kind, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b,sq,skv,h,hk", [(3, 1100, 333, 24, 24), (3, 600, 700, 24, 6), (2, 2400, 100, 20, 20)])
def test_unmasked(b, sq, skv, h, hk, d, dtype):
  assert _items(b, sq, h, hk) > 148
  q, k, v = _qkv(b, sq, skv, h, hk, d, dtype, seed=sq)
  got = cd.cross_attention(q, k, v)
  for _ in range(3):
    assert torch.equal(got, cd.cross_attention(q, k, v))
  g = h // hk
  for i in range(hk):
    _check(got[:, :, i * g:(i + 1) * g], q[:, :, i * g:(i + 1) * g], k[:, :, i:i + 1], v[:, :, i:i + 1])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths", [None, (8192, 0, 129), (4000, 8192, 1)])
def test_split_key_range_with_more_items_than_blocks(lengths, d, dtype):
  b, sq, skv, h = 3, 2500, 8192, 5
  assert _items(b, sq, h, h) > 148
  assert _native.lib().cdb_cross_attention_workspace_bytes(b, sq, skv, h, h, d, 0) > 0  # the partial results of a split
  if lengths is not None:
    return _run(b, sq, skv, h, h, d, lengths, "padded", dtype)
  q, k, v = _qkv(b, sq, skv, h, h, d, dtype, seed=4)
  got = cd.cross_attention(q, k, v)
  assert torch.equal(got, cd.cross_attention(q, k, v))
  for i in range(h):
    _check(got[:, :, i:i + 1], q[:, :, i:i + 1], k[:, :, i:i + 1], v[:, :, i:i + 1])
