"""4-bit microscaled matrices: quantisation, the product, and `Float4Linear`.

Two formats, both of e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign):
  "nvfp4"  blocks of 16 with an e4m3 scale, and per row a power of two in fp32.  The reference's `nvfp4` type
           (src/cache_dit/quantization/torchao/quantize_ao.py) has one fp32 scale per tensor instead: per row it needs
           no pass over the whole tensor before the first row can be written.
  "mxfp4"  blocks of 32 with a power-of-two scale (OCP microscaling).
The arithmetic and the layout of the scales are those of `cdb_fp4_quant_rows` in include/cache_dit_b200.h.

Inference only: none of these has a backward pass, and inputs that ask for one are refused.
"""
from __future__ import annotations

import dataclasses
from typing import Optional

import torch

from .. import _native

FORMATS = tuple(_native.FP4_FORMATS)
# names in QuantizeConfig -> format
QUANT_TYPES = {"nvfp4_per_row": "nvfp4", "mxfp4": "mxfp4"}
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_OUT_DTYPES = (torch.bfloat16, torch.float16)


@dataclasses.dataclass(frozen=True)
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
    return self.codes.numel() * 2 // self.cols if self.cols else 0

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


def no_gradients(what: str, *tensors) -> None:
  """These operators have no backward pass: refuse inputs that would silently lose one."""
  if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
    raise RuntimeError(f"{what} has no backward pass: call it under torch.no_grad() or on detached tensors")


def one_device(what: str, *tensors) -> None:
  present = [t for t in tensors if t is not None]
  _native._need_cuda(*present)
  if any(t.device != present[0].device for t in present):
    raise RuntimeError(f"{what}: all tensors must be on one device")


def _check_rows(t: Float4Rows, what: str) -> None:
  _check_format(t.format)
  _check_cols(t.cols)
  one_device(what, *t._triple())
  _native._need_contig(*t._triple())
  if t.codes.dtype != torch.uint8 or t.codes.dim() < 1 or t.codes.shape[-1] * 2 != t.cols:
    raise RuntimeError(f"{what}: codes must be uint8 [..., {t.cols // 2}], got {t.codes.dtype} {tuple(t.codes.shape)}")
  need = _native.fp4_block_scale_bytes(t.rows, t.cols, t.format)
  if t.block_scales.dtype != torch.uint8 or t.block_scales.numel() != need:
    raise RuntimeError(f"{what}: block scales must be {need} bytes in tiles of 128 rows x 4 scales, got "
                       f"{t.block_scales.dtype} {tuple(t.block_scales.shape)}")
  if t.format == "nvfp4":
    if t.row_scale is None or t.row_scale.dtype != torch.float32 or t.row_scale.numel() != t.rows:
      raise RuntimeError(f"{what}: nvfp4 needs one float32 scale per row ({t.rows})")
  elif t.row_scale is not None:
    raise RuntimeError(f"{what}: mxfp4 has no row scale")


def empty_rows(lead, cols: int, fmt: str, device) -> Float4Rows:
  """Uninitialised 4-bit rows for a kernel to fill."""
  rows = 1
  for n in lead:
    rows *= int(n)
  return Float4Rows(torch.empty((*lead, cols // 2), dtype=torch.uint8, device=device),
                    torch.empty(_native.fp4_block_scale_bytes(rows, cols, fmt), dtype=torch.uint8, device=device),
                    torch.empty(lead, dtype=torch.float32, device=device) if fmt == "nvfp4" else None, fmt, cols)


def _as_matrix(x: torch.Tensor) -> torch.Tensor:
  """x as [rows, cols] with unit column stride, 16-byte aligned rows; copied only where it is not."""
  x2 = x.reshape(-1, x.shape[-1])
  if x2.stride(-1) != 1 or (x2.shape[0] > 1 and x2.stride(0) * x2.element_size() % 16 != 0) or x2.stride(0) < x2.shape[1] \
      or x2.data_ptr() % 16 != 0:
    x2 = x2.clone(memory_format=torch.contiguous_format)
  return x2


def float4_quantize_rows(x: torch.Tensor, format: str = "nvfp4") -> Float4Rows:
  """Quantise the rows of x [..., cols] (float32, bfloat16 or float16) to 4 bits.  An infinity or NaN makes its row
  (nvfp4) or its block of 32 (mxfp4) stand for NaN."""
  _check_format(format)
  if x.dtype not in _DTYPES or x.dim() < 1:
    raise RuntimeError(f"float4_quantize_rows takes rows of float32, bfloat16 or float16, got {x.dtype} {tuple(x.shape)}")
  _check_cols(x.shape[-1])
  one_device("float4_quantize_rows", x)
  no_gradients("float4_quantize_rows", x)
  out = empty_rows(x.shape[:-1], x.shape[-1], format, x.device)
  if out.rows:
    _native.fp4_quant_rows(_as_matrix(x), *out._triple(), format)
  return out


def float4_dequantize_rows(t: Float4Rows, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
  """The values that 4-bit rows stand for, rounded once to `dtype`."""
  _check_rows(t, "float4_dequantize_rows")
  if dtype not in _DTYPES:
    raise RuntimeError(f"float4_dequantize_rows writes float32, bfloat16 or float16, not {dtype}")
  out = torch.empty(t.shape, dtype=dtype, device=t.device)
  if t.rows:
    _native.fp4_dequant_rows(*t._triple(), t.cols, t.format, out.view(-1, t.cols))
  return out


def float4_scaled_mm(a: Float4Rows, w: Float4Rows, bias: Optional[torch.Tensor] = None,
                     out_dtype: torch.dtype = torch.bfloat16, gelu: bool = False) -> torch.Tensor:
  """act(a [..., K] @ w [N, K]^T + bias [N]) -> [..., N]; `gelu`: act is the tanh-GELU of the fp32 value."""
  _check_rows(a, "float4_scaled_mm (a)")
  _check_rows(w, "float4_scaled_mm (w)")
  if a.format != w.format or a.cols != w.cols or w.codes.dim() != 2:
    raise RuntimeError(f"float4_scaled_mm: operands do not match: {a.format} {tuple(a.shape)} and {w.format} {tuple(w.shape)}")
  n = w.rows
  if n == 0 or n % 8 != 0:
    raise RuntimeError(f"float4_scaled_mm: the number of weight rows must be a multiple of 8, got {n}")
  if out_dtype not in _OUT_DTYPES:
    raise RuntimeError(f"float4_scaled_mm writes bfloat16 or float16, not {out_dtype}")
  if bias is not None and (bias.dtype != out_dtype or tuple(bias.shape) != (n, ) or not bias.is_contiguous()):
    raise RuntimeError(f"float4_scaled_mm: bias must be contiguous {out_dtype} [{n}]")
  one_device("float4_scaled_mm", a.codes, w.codes, bias)
  no_gradients("float4_scaled_mm", bias)
  out = torch.empty((*a.shape[:-1], n), dtype=out_dtype, device=a.device)
  if a.rows:
    _native.fp4_gemm(a._triple(), w._triple(), bias, out.view(-1, n), a.cols, a.format, gelu)
  return out


def float4_linear(x: torch.Tensor, w: Float4Rows, bias: Optional[torch.Tensor] = None, gelu: bool = False) -> torch.Tensor:
  """act(x @ w^T + bias) with x quantised to w's format on the way; x bfloat16 or float16, and so is the result."""
  if x.dtype not in _OUT_DTYPES:
    raise RuntimeError(f"float4_linear takes bfloat16 or float16 activations, got {x.dtype}")
  if x.shape[-1] != w.cols:
    raise RuntimeError(f"float4_linear: x has {x.shape[-1]} columns, the weight {w.cols}")
  return float4_scaled_mm(float4_quantize_rows(x, w.format), w, bias, x.dtype, gelu)
