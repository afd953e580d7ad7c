"""Masked attention to an encoder's states for heads of any size: what the kernel does not take, the plain form does."""
import pytest
import torch

from cache_dit_b200.synthetic.layers import encoder_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [8, 20, 64, 100, 128, 136, 256])
@torch.no_grad()
def test_prompts_of_different_lengths(d, dtype):
  g = torch.Generator().manual_seed(d)
  q, k, v = (torch.randn(3, n, 2, d, generator=g).to("cuda", dtype) for n in (33, 70, 70))
  mask = torch.arange(70, device="cuda")[None] < torch.tensor([70, 9, 0], device="cuda")[:, None]
  got = encoder_attention(q, k, torch.where(mask[:, :, None, None], v, float("nan")), mask)
  assert got.shape == q.shape and got.dtype == dtype
  for i, n in enumerate((70, 9)):
    s = torch.einsum("qhd,khd->hqk", q[i].double(), k[i, :n].double()) * d**-0.5
    p = torch.softmax(s, dim=-1)
    want = torch.einsum("hqk,khd->qhd", p, v[i, :n].double())
    magnitude = torch.einsum("hqk,khd->qhd", p, v[i, :n].double().abs())
    # weights and the result rounded to the type; scores: d products of at most max|q k|, each step of the sum a whole step
    # (2^-23); an error e of a score moves a weight by e and the row's sum by as much
    eps = torch.finfo(dtype).eps / 2
    score = (d + 4) * 2.0**-23 * torch.einsum("qhd,khd->hqk", q[i].double().abs(), k[i, :n].double().abs()).max().item() * d**-0.5
    assert ((got[i].double() - want).abs() <= (2 * eps + 2 * score + 2.0**-18) * magnitude + eps * want.abs() + 2.0**-24).all()
  assert (got[2] == 0).all()
