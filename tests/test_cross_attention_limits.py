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
