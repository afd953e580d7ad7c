"""Sizes that `cdb_cross_attention` refuses before it touches a tensor; no GPU is needed."""
import ctypes

import pytest

from cache_dit_b200 import _native as nat

TOO_LARGE = 7  # CDB_ERR_TOO_LARGE


def _call(batch, heads, sq=1, skv=1, d=8):
  t = nat.Heads(1 << 20, skv * heads * d, heads * d, d)
  q = nat.Heads(1 << 20, sq * heads * d, heads * d, d)
  return nat.lib().cdb_cross_attention(ctypes.byref(q), ctypes.byref(t), ctypes.byref(t), None, 0, 1 << 20, batch, sq, skv, heads, heads, d, 1.0,
                                       1, None, 0, None, None)


@pytest.mark.parametrize("batch,heads", [(33554432, 64), (33554431, 64), (2147483647, 1), (2147483500, 1)])
def test_work_items_stay_below_a_step_of_the_grid_from_the_largest_integer(batch, heads):
  """A block steps by the grid (at most the SMs of a B200, 148) past the last item: that sum is an integer, too."""
  assert batch * heads > 2147483647 - 148
  assert _call(batch, heads) == TOO_LARGE


def _parts(batch, sq, skv, heads, kv_heads, d):
  """How many parts the key range is split into: the workspace of an unmasked call holds their rows, (d + 2) words each."""
  rows = batch * sq * heads
  for n in range(2, 65):
    up = lambda b: -(-b // 256) * 256
    if nat.lib().cdb_cross_attention_workspace_bytes(batch, sq, skv, heads, kv_heads, d, 0) == up(n * rows * 8) + up(n * rows * d * 4):
      return n
  assert nat.lib().cdb_cross_attention_workspace_bytes(batch, sq, skv, heads, kv_heads, d, 0) == 0
  return 1


@pytest.mark.parametrize("shape,parts", [((1, 6400, 4096, 12, 12, 128), {1}), ((1, 6400, 4096, 12, 12, 64), {1}), ((1, 1024, 4096, 24, 24, 128), {1}),
                                         ((1, 256, 1024, 40, 40, 128), {1}), ((1, 512, 512, 24, 24, 128), {1}), ((64, 1, 2048, 32, 8, 128), {1}),
                                         ((1, 2560, 8192, 15, 15, 128), {2, 3, 4}), ((3, 2500, 8192, 5, 5, 64), {3, 4, 5, 6}),
                                         ((1, 300, 4096, 24, 24, 128), {3}), ((1, 4000, 16384, 10, 10, 128), {3, 4, 5}),
                                         ((1, 64, 4096, 24, 24, 64), {6}), ((4, 1, 16385, 32, 8, 128), {4}), ((1, 16, 65536, 8, 8, 128), {18})])
def test_key_range_is_split_where_that_is_faster(shape, parts):
  """On 148 SMs: what timing with every number of parts found fastest (or within 3 % of it)."""
  assert _parts(*shape) in parts
