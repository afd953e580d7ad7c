"""4-bit microscaled matrices: quantisation, the product, and `Float4Linear`.

Two formats, both of e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign):
  "nvfp4"  blocks of 16 with an e4m3 scale, and per row a power of two in fp32.  The reference's `nvfp4` type
           (src/cache_dit/quantization/torchao/quantize_ao.py) has one fp32 scale per tensor instead: per row it needs
           no pass over the whole tensor before the first row can be written.
  "mxfp4"  blocks of 32 with a power-of-two scale (OCP microscaling).
The arithmetic and the layout of the scales are those of `cdb_fp4_quant_rows` in include/cache_dit_b200.h.

Inference only: none of these has a backward pass or a forward-mode derivative, and inputs that carry one are refused.
A wait inside the product that runs out leaves its output incomplete and is latched in the device's status word: the cache
engine raises it at its next step, a direct caller asks `_native.check_device_status(device)`.
"""
from __future__ import annotations

import dataclasses
from typing import Optional

import torch
from torch.autograd import forward_ad

from .. import _native

FORMATS = tuple(_native.FP4_FORMATS)
# names in QuantizeConfig -> format
QUANT_TYPES = {"nvfp4_per_row": "nvfp4", "mxfp4": "mxfp4"}
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_OUT_DTYPES = (torch.bfloat16, torch.float16)


@dataclasses.dataclass(frozen=True, eq=False)
class Float4Rows:
  """A [..., cols] matrix in 4 bits: codes uint8 [..., cols / 2] (even column in the low half), the tiled block scales
  (uint8, flat), and for nvfp4 one float32 per row."""
  codes: torch.Tensor
  block_scales: torch.Tensor
  row_scale: Optional[torch.Tensor]
  format: str
  cols: int

  @property
  def shape(self) -> torch.Size:
    return torch.Size((*self.codes.shape[:-1], self.cols))

  @property
  def rows(self) -> int:
    return self.codes.numel() * 2 // self.cols

  @property
  def device(self) -> torch.device:
    return self.codes.device

  def nbytes(self) -> int:
    return sum(t.numel() * t.element_size() for t in self._triple() if t is not None)

  def _triple(self):
    return self.codes, self.block_scales, self.row_scale


def _check_format(fmt: str) -> str:
  if fmt not in FORMATS:
    raise ValueError(f"unknown 4-bit format {fmt!r}; supported: {FORMATS}")
  return fmt


def _check_cols(cols: int) -> None:
  if cols <= 0 or cols % 32 != 0 or cols > _native.FP4_MAX_COLS:
    raise ValueError(f"4-bit rows need a width that is a multiple of 32 and at most {_native.FP4_MAX_COLS}, got {cols}")


def refuse(what: str, *tensors) -> None:
  """Checks every operator here makes of its tensors (None: absent): none that carries a derivative, which would be lost
  silently (there is no backward pass and no forward-mode rule), and all on one CUDA device."""
  forward = forward_ad._current_level >= 0  # no_grad does not end forward mode
  if forward or torch.is_grad_enabled():
    for t in tensors:
      if t is None:
        continue
      if t.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors")
      if forward and forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"{what} has no forward-mode derivative: call it on the primal tensors (forward_ad.unpack_dual)")
  device = None
  for t in tensors:
    if t is None:
      continue
    if device is None:
      device = t.device
      if device.type != "cuda":
        _native._need_cuda(t)
    elif t.device != device:
      _native._need_cuda(t)
      raise RuntimeError(f"{what}: all tensors must be on one device")


def _check_rows(t: Float4Rows, what: str) -> int:
  """Refuses what is no 4-bit matrix; the number of its rows."""
  codes, scales, row = t.codes, t.block_scales, t.row_scale
  cols = t.cols
  _check_format(t.format)
  _check_cols(cols)
  if codes.dtype != torch.uint8 or codes.dim() < 1 or codes.shape[-1] * 2 != cols or not codes.is_contiguous():
    raise RuntimeError(f"{what}: codes must be contiguous uint8 [..., {cols // 2}], got {codes.dtype} {tuple(codes.shape)}")
  rows = codes.numel() * 2 // cols
  need = _native.fp4_block_scale_bytes(rows, cols, t.format)
  if scales.dtype != torch.uint8 or scales.numel() != need or not scales.is_contiguous():
    raise RuntimeError(f"{what}: block scales must be {need} contiguous bytes in tiles of 128 rows x 4 scales, got "
                       f"{scales.dtype} {tuple(scales.shape)}")
  if t.format == "nvfp4":
    if row is None or row.dtype != torch.float32 or row.numel() != rows or not row.is_contiguous():
      raise RuntimeError(f"{what}: nvfp4 needs one contiguous float32 scale per row ({rows})")
  elif row is not None:
    raise RuntimeError(f"{what}: mxfp4 has no row scale")
  return rows


def empty_rows(lead, cols: int, fmt: str, device) -> Float4Rows:
  """Uninitialised 4-bit rows for a kernel to fill."""
  rows = 1
  for n in lead:
    rows *= int(n)
  return Float4Rows(torch.empty((*lead, cols // 2), dtype=torch.uint8, device=device),
                    torch.empty(_native.fp4_block_scale_bytes(rows, cols, fmt), dtype=torch.uint8, device=device),
                    torch.empty(lead, dtype=torch.float32, device=device) if fmt == "nvfp4" else None, fmt, cols)


def _as_matrix(x: torch.Tensor, rows: int, cols: int):
  """(x as rows of `cols` elements with unit column stride and 16-byte aligned rows, their distance); copied only where it
  is not that already."""
  if x.is_contiguous():
    ld = cols
  else:
    x = x.reshape(rows, cols)
    ld = x.stride(0) if rows > 1 else cols
    if x.stride(1) != 1 or ld < cols or ld * x.element_size() % 16 != 0:
      x = x.clone(memory_format=torch.contiguous_format)
      ld = cols
  if x.data_ptr() % 16 != 0:
    x = x.clone(memory_format=torch.contiguous_format)
    ld = cols
  return x, ld


def _rows_to_quantise(x: torch.Tensor, dtypes, what: str):
  if x.dtype not in dtypes or x.dim() < 1:
    raise RuntimeError(f"{what} takes rows of {', '.join(str(d)[6:] for d in dtypes)}, got {x.dtype} {tuple(x.shape)}")
  cols = x.shape[-1]
  _check_cols(cols)
  return x.numel() // cols, cols


def float4_quantize_rows(x: torch.Tensor, format: str = "nvfp4") -> Float4Rows:
  """Quantise the rows of x [..., cols] (float32, bfloat16 or float16) to 4 bits.  An infinity or NaN makes its row
  (nvfp4) or its block of 32 (mxfp4) stand for NaN."""
  what = "float4_quantize_rows"
  _check_format(format)
  rows, cols = _rows_to_quantise(x, _DTYPES, what)
  refuse(what, x)
  out = empty_rows(x.shape[:-1], cols, format, x.device)
  if rows:
    x2, ld = _as_matrix(x, rows, cols)
    _native.fp4_quant_rows(x2, ld, rows, cols, *out._triple(), format)
  return out


def float4_dequantize_rows(t: Float4Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
  """The values that 4-bit rows stand for, rounded once to `dtype`."""
  what = "float4_dequantize_rows"
  rows = _check_rows(t, what)
  refuse(what, *t._triple())
  if dtype not in _DTYPES:
    raise RuntimeError(f"{what} writes float32, bfloat16 or float16, not {dtype}")
  out = torch.empty(t.shape, dtype=dtype, device=t.device)
  if rows:
    t = _aligned(t)
    _native.fp4_dequant_rows(*t._triple(), rows, t.cols, t.format, out)
  return out


def _aligned(t: Float4Rows) -> Float4Rows:
  """t with 16-byte aligned codes and scales (copied only where a view starts elsewhere)."""
  if t.codes.data_ptr() % 16 == 0 and t.block_scales.data_ptr() % 16 == 0:
    return t
  return dataclasses.replace(t, codes=t.codes.clone(), block_scales=t.block_scales.clone())


def _check_weight(w: Float4Rows, bias: Optional[torch.Tensor], out_dtype: torch.dtype, what: str) -> int:
  n = _check_rows(w, what + " (w)")
  if w.codes.dim() != 2 or n == 0 or n % 8 != 0:
    raise RuntimeError(f"{what}: the weight must be [N, K] with N a multiple of 8, got {tuple(w.shape)}")
  if out_dtype not in _OUT_DTYPES:
    raise RuntimeError(f"{what} writes bfloat16 or float16, not {out_dtype}")
  if bias is not None and (bias.dtype != out_dtype or bias.dim() != 1 or bias.shape[0] != n or not bias.is_contiguous()):
    raise RuntimeError(f"{what}: bias must be contiguous {out_dtype} [{n}], got {bias.dtype} {tuple(bias.shape)}")
  return n


def float4_scaled_mm(a: Float4Rows, w: Float4Rows, bias: Optional[torch.Tensor] = None,
                     out_dtype: torch.dtype = torch.bfloat16, gelu: bool = False) -> torch.Tensor:
  """act(a [..., K] @ w [N, K]^T + bias [N]) -> [..., N]; `gelu`: act is the tanh-GELU of the fp32 value."""
  what = "float4_scaled_mm"
  rows = _check_rows(a, what + " (a)")
  n = _check_weight(w, bias, out_dtype, what)
  if a.format != w.format or a.cols != w.cols:
    raise RuntimeError(f"{what}: operands do not match: {a.format} {tuple(a.shape)} and {w.format} {tuple(w.shape)}")
  refuse(what, *a._triple(), *w._triple(), bias)
  out = torch.empty((*a.codes.shape[:-1], n), dtype=out_dtype, device=a.device)
  if rows:
    _native.fp4_gemm(_aligned(a)._triple(), _aligned(w)._triple(), bias, out, rows, a.cols, a.format, gelu)
  return out


def float4_linear(x: torch.Tensor, w: Float4Rows, bias: Optional[torch.Tensor] = None, gelu: bool = False) -> torch.Tensor:
  """act(x @ w^T + bias) with x quantised to w's format on the way; x bfloat16 or float16, and so is the result: the same
  numbers as float4_scaled_mm(float4_quantize_rows(x, w.format), w, bias, x.dtype, gelu)."""
  what = "float4_linear"
  rows, cols = _rows_to_quantise(x, _OUT_DTYPES, what)
  n = _check_weight(w, bias, x.dtype, what)
  if cols != w.cols:
    raise RuntimeError(f"{what}: x has {cols} columns, the weight {w.cols}")
  refuse(what, x, w.codes, w.block_scales, w.row_scale, bias)
  out = x.new_empty((*x.shape[:-1], n))
  if rows:
    x2, ld = _as_matrix(x, rows, cols)
    _native.fp4_linear(x2, ld, _aligned(w)._triple(), bias, out, rows, cols, w.format, gelu)
  return out


class Float4Linear(torch.nn.Module):
  """y = float4_linear(x, W): an nn.Linear replacement with 4-bit activations and weights, bfloat16 in and out.  The weight
  is quantised once; codes and scales are buffers, so they move and save with the module.  A cast of the module (`.half()`,
  `.to(dtype)`) leaves them and the bias in their types."""

  def __init__(self, weight: Float4Rows, bias: Optional[torch.Tensor]):
    super().__init__()
    self.out_features, self.in_features = weight.shape
    self.format = weight.format
    self.register_buffer("weight_codes", weight.codes)                # [N, K / 2] uint8
    self.register_buffer("weight_block_scales", weight.block_scales)  # tiled, uint8
    self.register_buffer("weight_row_scale", weight.row_scale)        # [N] float32, None for mxfp4
    self.register_buffer("bias", bias)                                # [N] bfloat16 or None

  @classmethod
  def from_linear(cls, linear: torch.nn.Linear, format: str = "nvfp4") -> "Float4Linear":
    w = linear.weight.detach()
    if not w.is_cuda:
      raise RuntimeError("4-bit quantization runs on the GPU: move the module to CUDA first")
    if not cls.supports(linear):
      raise RuntimeError("a 4-bit linear needs bfloat16 weights with in_features % 32 == 0, at most "
                         f"{_native.FP4_MAX_COLS}, and out_features % 8 == 0, got {w.dtype} {tuple(w.shape)}")
    bias = None if linear.bias is None else linear.bias.detach().to(torch.bfloat16).contiguous()
    return cls(float4_quantize_rows(w, format), bias)

  @staticmethod
  def supports(linear: torch.nn.Linear) -> bool:
    n, k = linear.weight.shape
    return linear.weight.dtype == torch.bfloat16 and k % 32 == 0 and 0 < k <= _native.FP4_MAX_COLS and n % 8 == 0 and n > 0

  def _apply(self, fn, recurse: bool = True):
    """`.to()`, `.half()` and the like: the buffers follow the device, their types are the kernels' and stay."""
    before = dict(self._buffers)
    super()._apply(fn, recurse)
    for name, old in before.items():
      new = self._buffers[name]
      if old is not None and new.dtype != old.dtype:
        self._buffers[name] = old.to(new.device)
    return self

  @property
  def weight_rows(self) -> Float4Rows:
    return Float4Rows(self.weight_codes, self.weight_block_scales, self.weight_row_scale, self.format, self.in_features)

  def forward_quantized(self, a: Float4Rows, gelu: bool = False) -> torch.Tensor:
    """Product for activations that a producer already wrote in 4 bits.  `gelu`: the tanh-GELU of the output."""
    return float4_scaled_mm(a, self.weight_rows, self.bias, torch.bfloat16, gelu)

  def forward(self, x: torch.Tensor, gelu: bool = False) -> torch.Tensor:
    if x.dtype != torch.bfloat16:
      x = x.to(torch.bfloat16)
    return float4_linear(x, self.weight_rows, self.bias, gelu)

  def extra_repr(self) -> str:
    return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}, 4-bit={self.format}"
