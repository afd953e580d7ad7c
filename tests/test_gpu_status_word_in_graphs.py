"""Kernels of a captured graph have a status word even where the capture is their operator's first call in the process."""
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

PROGRAM = """
import torch
import cache_dit_b200 as cd
from cache_dit_b200 import _native
torch.manual_seed(0)
x = torch.randn(300, 256, device="cuda").to(torch.bfloat16)
q = torch.randn(1, 200, 2, 64, device="cuda").to(torch.bfloat16)
{first}
side = torch.cuda.Stream()
graph = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(graph, stream=side):
  assert _native._status_ptr(0) is not None
  y = cd.float4_linear(x, w) if {linear} else cd.cross_attention(q, q, q)
graph.replay()
torch.cuda.synchronize()
with torch.no_grad():
  assert torch.equal(y, cd.float4_linear(x, w) if {linear} else cd.cross_attention(q, q, q))
assert _native._status_ptr(0) == _native.gemm_status_word(torch.device("cuda", 0)).data_ptr()
_native.check_device_status(torch.device("cuda", 0))
print("fine")
"""


@pytest.mark.parametrize("first,linear", [("w = cd.float4_quantize_rows(x[:128])", True), ("cd.gated_residual_norm(x)", False),
                                          ("cd.float4_quantize_rows(x)", False)])
def test_made_by_the_first_call_of_any_operator(first, linear):
  r = subprocess.run([sys.executable, "-c", PROGRAM.format(first=first, linear=linear)], capture_output=True, text=True, timeout=300)
  assert r.returncode == 0 and "fine" in r.stdout, r.stdout + r.stderr
