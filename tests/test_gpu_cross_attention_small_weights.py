"""`cross_attention` in float16 where many keys of tiny weight stand beside one that dominates: together they count."""
import math

import pytest
import torch

import cache_dit_b200 as cd

pytestmark = pytest.mark.gpu


def _one_key_above_the_rest(queries, keys, at, nats, d=64):
  """q . k is `nats` for key `at` and 0 for all others; v is 0 there and 1 elsewhere.  Every product is exact."""
  q = torch.zeros(1, queries, 1, d)
  k = torch.zeros(1, keys, 1, d)
  v = torch.ones(1, keys, 1, d)
  q[..., 0] = 4.0
  k[0, at, 0, 0] = nats / 4.0
  v[0, at] = 0.0
  return [t.to("cuda", torch.float16) for t in (q, k, v)]


# (1, ..) splits the key range, 37888 queries are one item of 256 each for every SM of a B200 and do not
@pytest.mark.parametrize("queries", [1, 37888])
@pytest.mark.parametrize("keys,at", [(8192, 0), (8192, 8191), (20001, 5000)])
@pytest.mark.parametrize("nats", [12.0, 15.0, 18.0])
def test_weights_below_the_smallest_half_add_up(queries, keys, at, nats):
  q, k, v = _one_key_above_the_rest(queries, keys, at, nats)
  got = cd.cross_attention(q, k, v, scale=1.0).double()
  rest = (keys - 1) * math.exp(-nats)
  want = rest / (1.0 + rest)
  # A key's weight is held in float16 as 2^7 times its share of the largest (which may stand 2^8 higher still): half a step
  # of a subnormal is 2^-25, or 2^-32 of the largest weight, for every key at most; half a step where it is normal.  The
  # exponential (2^-22 relative, its argument 15 * 1.45 * 2^-23) and the fp32 sums (tensor core: a whole step each 16 keys)
  # are below 2^-11 of the result; and one rounding of the result, normal or not.
  bound = keys * 2.0**-32 + want * (2.0**-11 + 2.0**-18 + (keys / 16 + 8) * 2.0**-23) + want * 2.0**-11 + 2.0**-25
  assert ((got - want).abs() <= bound).all(), (got.flatten()[0].item(), want, bound)
