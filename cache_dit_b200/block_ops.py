"""Operators of transformer blocks around the linears: a gated residual with norms on either side, and attention to an
encoder's states.

In the models the reference wraps these are eager PyTorch ops inside the diffusers blocks.  Inference only: inputs that
carry a derivative (backward or forward mode) are refused.  All tensors of a call lie on one CUDA device; results are new,
contiguous tensors on the current stream of that device.  A wait inside the attention that runs out leaves its output
incomplete and is latched in the device's status word: the cache engine raises it at its next step, a direct caller asks
`_native.check_device_status(device)`.
"""
from __future__ import annotations

import math
from typing import Optional, Tuple, Union

import torch

from . import _native
from .quantization.float4 import FORMATS, Float4Rows, empty_rows, refuse

_DTYPES = (torch.float32, torch.bfloat16, torch.float16)


def _rows_of(what: str, name: str, t: torch.Tensor, shape, dtype) -> torch.Tensor:
  if t.shape != shape or t.dtype != dtype:
    raise RuntimeError(f"{what}: {name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")
  t = t if t.dim() == 3 else t.reshape(1, -1, t.shape[-1])
  return t if t.stride(2) == 1 or t.shape[2] == 1 else t.contiguous()


def _vector_of(what: str, name: str, t: Optional[torch.Tensor], batch: int, dim: int, dtype, per_batch: bool):
  if t is None:
    return None
  if t.dtype == dtype and t.dim() == (2 if per_batch else 1) and t.shape[-1] == dim and t.stride(-1) == 1 and \
      (not per_batch or t.shape[0] == batch):
    return t  # the usual case: [batch, dim], or a [dim] weight
  shapes = [(dim, )] + ([(batch, dim), (1, dim)] if per_batch else [])
  if t.dtype != dtype or tuple(t.shape) not in shapes:
    raise RuntimeError(f"{what}: {name} must be {dtype} {' or '.join(map(str, shapes[:2]))}, got {t.dtype} {tuple(t.shape)}")
  if t.dim() == 2 and t.shape[0] == 1 and batch != 1:
    t = t[0]
  return t if t.stride(-1) == 1 or dim == 1 else t.contiguous()


def gated_residual_norm(x: torch.Tensor, y: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, *,
                        residual_scale: float = 1.0, post_norm: Optional[str] = None,
                        post_weight: Optional[torch.Tensor] = None, post_bias: Optional[torch.Tensor] = None,
                        post_eps: float = 1e-6, norm: Optional[str] = "layer", weight: Optional[torch.Tensor] = None,
                        bias: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                        shift: Optional[torch.Tensor] = None, eps: float = 1e-6,
                        quantize: Optional[str] = None) -> Tuple[torch.Tensor, Union[torch.Tensor, Float4Rows, None]]:
  """(x', h) in one pass over the rows:

      x' = x + residual_scale * gate * post_norm(y)
      h  = norm(x') * weight + bias, then * (1 + scale) + shift

  x, y [batch, tokens, dim] (or [rows, dim]: one batch) in float32, bfloat16 or float16; rows may be strided.  The norms
  are "rms", "layer" or None (post_norm: y as it is; norm: no h).  gate, scale and shift are [batch, dim] or [dim],
  weights and biases [dim], all in x's type.  Without y, x' is x itself and only the norm runs.
  quantize = "nvfp4" | "mxfp4": h comes back as `Float4Rows`, the 4-bit form of exactly the h that would be returned
  without it; dim must then be a multiple of 32.  The norm reads x' before its rounding to x's type."""
  what = "gated_residual_norm"
  if x.dtype not in _DTYPES or x.dim() not in (2, 3):
    raise RuntimeError(f"{what}: x must be [batch, tokens, dim] or [rows, dim] in float32, bfloat16 or float16, got "
                       f"{x.dtype} {tuple(x.shape)}")
  for name, kind in (("post_norm", post_norm), ("norm", norm)):
    if kind not in _native.NORM_KINDS:
      raise ValueError(f"{what}: {name} must be 'rms', 'layer' or None, not {kind!r}")
  if y is None and (gate is not None or post_norm is not None or residual_scale != 1.0):
    raise RuntimeError(f"{what}: gate, post_norm and residual_scale belong to y, which is missing")
  if post_norm is None and (post_weight is not None or post_bias is not None):
    raise RuntimeError(f"{what}: post_weight and post_bias belong to post_norm, which is None")
  if norm is None and (y is None or any(t is not None for t in (weight, bias, scale, shift)) or quantize is not None):
    raise RuntimeError(f"{what}: without norm there is nothing but x' to compute")
  if (scale is None) != (shift is None):
    raise RuntimeError(f"{what}: scale and shift go together")
  dim = x.shape[-1]
  if dim == 0 or dim > _native.NORM_MAX_DIM:
    raise RuntimeError(f"{what}: rows of 1 to {_native.NORM_MAX_DIM} elements, got {dim}")
  if quantize is not None:
    if quantize not in FORMATS:
      raise ValueError(f"{what}: unknown 4-bit format {quantize!r}; supported: {FORMATS}")
    if dim % 32 != 0:
      raise RuntimeError(f"{what}: 4-bit rows need a width that is a multiple of 32, got {dim}")
  refuse(what, x, y, gate, post_weight, post_bias, weight, bias, scale, shift)
  batch = x.shape[0] if x.dim() == 3 else 1
  x3 = _rows_of(what, "x", x, x.shape, x.dtype)
  y3 = None if y is None else _rows_of(what, "y", y, x.shape, x.dtype)
  dtype = x.dtype
  vectors = (_vector_of(what, "gate", gate, batch, dim, dtype, True), _vector_of(what, "post_weight", post_weight, batch, dim, dtype, False),
             _vector_of(what, "post_bias", post_bias, batch, dim, dtype, False), _vector_of(what, "weight", weight, batch, dim, dtype, False),
             _vector_of(what, "bias", bias, batch, dim, dtype, False), _vector_of(what, "scale", scale, batch, dim, dtype, True),
             _vector_of(what, "shift", shift, batch, dim, dtype, True))
  x_out = x if y is None else x.new_empty(x.shape)
  h = fp4 = None
  if quantize is not None:
    h4 = empty_rows(x.shape[:-1], dim, quantize, x.device)
    fp4 = (*h4._triple(), quantize)
    aligned = lambda t: t is None or (t.data_ptr() % 16 == 0 and all(s * t.element_size() % 16 == 0 for s in t.stride()[:-1]))
    x3, y3, *vectors = (t if aligned(t) else t.clone(memory_format=torch.contiguous_format) for t in (x3, y3, *vectors))
  elif norm is not None:
    h = x.new_empty(x.shape)
  if x.numel():
    _native.gated_residual_norm(x3, y3, *vectors, x_out, h, fp4, post_norm, norm, float(residual_scale), float(post_eps), float(eps))
  return x_out, h if quantize is None else h4


def _heads_of(t: torch.Tensor) -> torch.Tensor:
  """t [batch, tokens, heads, d] as the kernel's loads want it: unit stride within a head, every other stride positive and a
  multiple of 16 bytes, base 16-byte aligned; copied only where it is not."""
  if t.is_contiguous() and t.data_ptr() % 16 == 0:
    return t  # the head dimension is a multiple of 8
  ok = t.data_ptr() % 16 == 0 and (t.stride(3) == 1 or t.shape[3] == 1) and \
      all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:3], t.stride()[:3]))
  return t if ok else t.clone(memory_format=torch.contiguous_format)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, key_mask: Optional[torch.Tensor] = None,
                    scale: Optional[float] = None) -> torch.Tensor:
  """softmax(scale * q k^T) v for q [batch, tokens, heads, d] and an encoder's k, v [batch, keys, kv_heads, d], in bfloat16
  or float16; heads is a multiple of kv_heads, consecutive query heads share a key / value head; d a multiple of 8, at
  most 128.  key_mask bool [batch, keys]: True keeps the key; a batch entry that keeps none gives zeros, and what lies in
  masked places of k and v (infinities and NaN too) has no effect.  scale defaults to 1 / sqrt(d).
  Returns [batch, tokens, heads, d]."""
  what = "cross_attention"
  if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[3] != q.shape[3]:
    raise RuntimeError(f"{what}: q [batch, tokens, heads, d] and k, v [batch, keys, kv_heads, d], got {tuple(q.shape)}, "
                       f"{tuple(k.shape)}, {tuple(v.shape)}")
  if q.dtype not in (torch.bfloat16, torch.float16) or k.dtype != q.dtype or v.dtype != q.dtype:
    raise RuntimeError(f"{what}: q, k and v must all be bfloat16 or all float16, got {q.dtype}, {k.dtype}, {v.dtype}")
  b, sq, h, d = q.shape
  skv, kv_h = k.shape[1], k.shape[2]
  if h == 0 or kv_h == 0 or h % kv_h != 0:
    raise RuntimeError(f"{what}: the number of query heads ({h}) must be a multiple of the key heads ({kv_h})")
  if d == 0 or d % 8 != 0 or d > _native.CROSS_MAX_HEAD_DIM:
    raise RuntimeError(f"{what}: the head dimension must be a multiple of 8 and at most {_native.CROSS_MAX_HEAD_DIM}, got {d}")
  if key_mask is not None and (key_mask.dtype != torch.bool or tuple(key_mask.shape) != (b, skv)):
    raise RuntimeError(f"{what}: key_mask must be bool {(b, skv)}, got {key_mask.dtype} {tuple(key_mask.shape)}")
  scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
  if not (scale > 0.0 and math.isfinite(scale)):
    raise RuntimeError(f"{what}: scale must be positive and finite, got {scale}")
  refuse(what, q, k, v, key_mask)
  out = q.new_empty((b, sq, h, d))
  if out.numel() == 0:
    return out
  if skv == 0:
    return out.zero_()
  if key_mask is not None and key_mask.stride(1) != 1 and skv > 1:
    key_mask = key_mask.contiguous()
  _native.cross_attention(_heads_of(q), _heads_of(k), _heads_of(v), key_mask, scale, out)
  return out
