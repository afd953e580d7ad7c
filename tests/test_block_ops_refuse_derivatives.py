"""The 4-bit, norm and attention operators have no derivative: inputs that carry one are refused in both directions."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

import cache_dit_b200 as cd
from cache_dit_b200.quantization import float4


def _calls(device):
  """{name of the argument that carries the derivative: (operator, that argument's value, call with it)}."""
  bf = dict(device=device, dtype=torch.bfloat16)
  x, row, w1 = torch.ones(2, 4, 64, **bf), torch.ones(2, 64, **bf), torch.ones(64, **bf)
  q, k = torch.ones(2, 3, 2, 64, **bf), torch.ones(2, 5, 2, 64, **bf)
  w = float4.empty_rows((8, ), 64, "mxfp4", device)
  w.codes.fill_(0x22)
  w.block_scales.fill_(127)
  bias = torch.ones(8, **bf)
  norm, att = cd.gated_residual_norm, cd.cross_attention
  return {
    "quantised x": ("float4_quantize_rows", x, lambda t: cd.float4_quantize_rows(t)),
    "linear x": ("float4_linear", x, lambda t: cd.float4_linear(t, w)),
    "linear bias": ("float4_linear", bias, lambda t: cd.float4_linear(x, w, t)),
    "product bias": ("float4_scaled_mm", bias, lambda t: cd.float4_scaled_mm(w, w, t)),
    "norm x": ("gated_residual_norm", x, lambda t: norm(t)),
    "norm y": ("gated_residual_norm", x, lambda t: norm(x, t)),
    "norm gate": ("gated_residual_norm", row, lambda t: norm(x, x, t)),
    "norm weight": ("gated_residual_norm", w1, lambda t: norm(x, weight=t, bias=w1)),
    "norm bias": ("gated_residual_norm", w1, lambda t: norm(x, bias=t)),
    "norm scale": ("gated_residual_norm", row, lambda t: norm(x, scale=t, shift=row)),
    "norm shift": ("gated_residual_norm", row, lambda t: norm(x, scale=row, shift=t)),
    "norm post_weight": ("gated_residual_norm", w1, lambda t: norm(x, x, post_norm="rms", post_weight=t)),
    "norm post_bias": ("gated_residual_norm", w1, lambda t: norm(x, x, post_norm="rms", post_bias=t)),
    "attention q": ("cross_attention", q, lambda t: att(t, k, k)),
    "attention k": ("cross_attention", k, lambda t: att(q, t, k)),
    "attention v": ("cross_attention", k, lambda t: att(q, k, t)),
  }


NAMES = list(_calls("cpu"))


def _refuses(device, name):
  what, value, call = _calls(device)[name]
  for context in (torch.enable_grad, torch.no_grad):  # forward derivatives do not stop at no_grad
    with context(), forward_ad.dual_level():
      with pytest.raises(RuntimeError, match=f"{what} has no forward-mode derivative"):
        call(forward_ad.make_dual(value, torch.ones_like(value)))
  with pytest.raises(RuntimeError, match=f"{what} has no backward pass"):
    call(value.clone().requires_grad_())


@pytest.mark.parametrize("name", NAMES)
def test_refused_before_the_device_is_looked_at(name):
  _refuses("cpu", name)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_refused_and_taken_without(name):
  _refuses("cuda", name)
  what, value, call = _calls("cuda")[name]
  with torch.no_grad():
    call(value.clone().requires_grad_())
    with forward_ad.dual_level():
      call(value)  # others' dual numbers are not this call's
