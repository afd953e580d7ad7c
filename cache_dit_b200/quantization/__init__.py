from .config import QuantizeBackend, QuantizeConfig
from .float4 import (Float4Linear, Float4Rows, float4_dequantize_rows, float4_linear, float4_quantize_rows, float4_scaled_mm)
from .linear import (Float8RowwiseLinear, FusedFloat8Linears, fused_group, grouped_forward_quantized,
                     quantize_rows_fused, quantize_rows_fused_pair)
from .quantize import quantize, remove_quantization_stats
from . import ops
