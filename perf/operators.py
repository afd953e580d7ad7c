"""Cases that measure the operators of a 4-bit, cross-attending transformer block, with their plain forms.

Operators
  round trip   4-bit microscaled quantisation of rows and back (`float4_quantize_rows`, `float4_dequantize_rows`)
  linear       a linear layer with 4-bit activations and weights (`float4_linear`)
  norm         x + residual_scale * gate * post_norm(y), and the next norm of it (`gated_residual_norm`)
  layer        the same norm written in 4 bits, and the linear layer that reads it
  attention    attention of tokens to an encoder's states of another length (`cross_attention`)

4-bit formats (magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6; even element in the low half of a byte)
  nvfp4  blocks of 16 with an e4m3 scale, and per row the smallest power of two (fp32) that keeps those scales
         within 448: row = 2^ceil(log2(max|row| / 2688)), scale = e4m3(max|block| / (6 row))
  mxfp4  blocks of 32 with a power-of-two scale (e8m0): 2^(floor(log2(max|block|)) - 2)
A code is the nearest magnitude to x / (scale * row), ties to the even code.
Block scales lie in tiles of 128 rows x 4 scales: byte (r % 32) * 16 + (r / 32) * 4 + k, tiles of a row panel one
after another, panels padded with zeros to whole 256-column steps.
"""
import math

import torch

own = False

BF16, F16, F32 = "bfloat16", "float16", "float32"
BLOCK = {"nvfp4": 16, "mxfp4": 32}


def listed():
  return [
    # the joint sequence of an image model (4096 image + 512 text tokens), hidden size of the video model
    dict(name="quant-nv-joint", op="quant", fmt="nvfp4", rows=4608, cols=5120, dtype=BF16),
    # a ragged batch of MLP activations
    dict(name="quant-mx-ragged", op="quant", fmt="mxfp4", rows=1001, cols=13824, dtype=F16),
    # one timestep embedding through a six-way modulation projection
    dict(name="linear-nv-one-row", op="linear", fmt="nvfp4", m=1, n=30720, k=5120, dtype=BF16, gelu=False),
    # a padded prompt through the key projection of a cross attention
    dict(name="linear-mx-prompt", op="linear", fmt="mxfp4", m=77, n=5120, k=4096, dtype=F16, gelu=False),
    # a context-parallel rank's image tokens through an MLP-in projection with its GELU
    dict(name="linear-nv-shard-gelu", op="linear", fmt="nvfp4", m=1153, n=12288, k=5120, dtype=BF16, gelu=True),
    # the largest product of the linear sweep
    dict(name="linear-nv-large", op="linear", fmt="nvfp4", m=16384, n=13824, k=5120, dtype=BF16, gelu=False),
    # one rank's video tokens after self-attention: gated residual and the LayerNorm in front of cross-attention
    dict(name="norm-video", op="norm", batch=1, tokens=9450, dim=5120, dtype=BF16, post="none", norm="layer", affine=True, mod=False),
    # a block with norms on both sides, RMS, two prompts, a width that is no power of two
    dict(name="norm-sandwich", op="norm", batch=2, tokens=257, dim=2304, dtype=F16, post="rms", norm="rms", affine=True, mod=True),
    # gated residual, modulated LayerNorm and the MLP-in projection that reads it in 4 bits
    dict(name="layer-nv-image", op="layer", fmt="nvfp4", batch=1, tokens=4096, dim=5120, n=13824, dtype=BF16),
    # half of a video's tokens attending to 512 text tokens
    dict(name="cross-video", op="attention", batch=1, sq=37800, skv=512, heads=40, kv_heads=40, d=128, dtype=BF16, mask="none"),
    # a batch of prompts of different lengths, padded
    dict(name="cross-padded", op="attention", batch=2, sq=4096, skv=333, heads=24, kv_heads=24, d=64, dtype=F16, mask="padded"),
    # one query token over a long context with shared key/value heads
    dict(name="cross-one-token", op="attention", batch=4, sq=1, skv=16385, heads=32, kv_heads=8, d=128, dtype=BF16, mask="padded"),
  ]


def _spread(rng, lo, hi):
  return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
  op = rng.choice(["quant", "linear", "norm", "layer", "attention"])
  dtype = rng.choice([BF16, F16])
  fmt = rng.choice(["nvfp4", "mxfp4"])
  if op == "quant":
    cols = 32 * _spread(rng, 1, 480)
    return dict(op=op, fmt=fmt, rows=_spread(rng, 1, max(1, 50_000_000 // cols)), cols=cols, dtype=rng.choice([BF16, F16, F32]))
  if op == "linear":
    k, n = 32 * _spread(rng, 2, 480), 8 * _spread(rng, 2, 2400)
    return dict(op=op, fmt=fmt, m=min(_spread(rng, 1, 16384), max(1, int(1.1e12 / (n * k)))), n=n, k=k, dtype=dtype, gelu=rng.random() < 0.3)
  if op == "norm":
    dim, batch = _spread(rng, 16, 8192), rng.randint(1, 3)
    if rng.random() < 0.7:
      dim = (dim + 7) // 8 * 8
    return dict(op=op, batch=batch, tokens=_spread(rng, 1, max(1, 45_000_000 // (dim * batch))), dim=dim, dtype=rng.choice([BF16, F16, F32]),
                post=rng.choice(["none", "rms", "layer"]), norm=rng.choice(["rms", "layer"]), affine=rng.random() < 0.5, mod=rng.random() < 0.5)
  if op == "layer":
    dim, n = 32 * _spread(rng, 4, 256), 8 * _spread(rng, 8, 1800)
    return dict(op=op, fmt=fmt, batch=rng.randint(1, 2), tokens=_spread(rng, 1, 4096), dim=dim, n=n, dtype=dtype)
  kv_heads, d = rng.choice([1, 2, 8, 12, 24]), 8 * rng.randint(4, 16)
  heads = kv_heads * rng.choice([1, 1, 1, 2, 4])
  batch, skv = rng.randint(1, 4), _spread(rng, 1, 8192)
  sq = _spread(rng, 1, 20000)
  sq = min(sq, max(1, int(7e8 / (batch * heads * skv))))
  return dict(op=op, batch=batch, sq=sq, skv=skv, heads=heads, kv_heads=kv_heads, d=d, dtype=dtype, mask=rng.choice(["none", "padded", "holes"]))


# ---- what a program has in hand -----------------------------------------------------------------------------


def _normal(g, shape, dtype, std=1.0, mean=0.0):
  return (torch.randn(shape, generator=g, device="cuda") * std + mean).to(getattr(torch, dtype))


def _activations(g, rows, cols, dtype):
  """Transformer activations: a few channels far louder than the rest."""
  x = torch.randn((rows, cols), generator=g, device="cuda")
  loud = torch.exp(0.7 * torch.randn((cols, ), generator=g, device="cuda"))
  return (x * loud).to(getattr(torch, dtype))


def _packed_weight(g, n, k, fmt):
  w = _normal(g, (n, k), BF16, std=k**-0.5)
  code, scale_byte, row = quantize_plain(w, fmt)
  return dict(codes=code[:, 0::2] | (code[:, 1::2] << 4), block_scales=tiled(scale_byte, fmt), row_scale=row)


def prepare(case, seed):
  g = torch.Generator(device="cuda").manual_seed(seed)
  op, dt = case["op"], case["dtype"]
  s = dict(case=case)
  if op == "quant":
    s["x"] = _activations(g, case["rows"], case["cols"], dt)
  elif op == "linear":
    s["x"] = _activations(g, case["m"], case["k"], dt)
    s["w"] = _packed_weight(g, case["n"], case["k"], case["fmt"])
    s["bias"] = _normal(g, (case["n"], ), dt, std=0.1)
  elif op in ("norm", "layer"):
    b, t, c = case["batch"], case["tokens"], case["dim"]
    s["x"] = _activations(g, b * t, c, dt).view(b, t, c)
    s["y"] = _normal(g, (b, t, c), dt, std=0.5)
    mod = _normal(g, (b, 3 * c), dt, std=0.3)  # gate, scale and shift are slices of one projection
    s["gate"] = mod[:, :c]
    if op == "layer" or case["mod"]:
      s["scale"], s["shift"] = mod[:, c:2 * c], mod[:, 2 * c:]
    if op == "norm" and case["affine"]:
      s["weight"] = _normal(g, (c, ), dt, std=0.1, mean=1.0)
      s["bias"] = _normal(g, (c, ), dt, std=0.1) if case["norm"] == "layer" else None
    if op == "norm" and case["post"] != "none":
      s["post_weight"] = _normal(g, (c, ), dt, std=0.1, mean=1.0)
    if op == "layer":
      s["w"] = _packed_weight(g, case["n"], c, case["fmt"])
      s["w_bias"] = _normal(g, (case["n"], ), dt, std=0.1)
  else:
    b, h, hk, d = case["batch"], case["heads"], case["kv_heads"], case["d"]
    s["q"] = _normal(g, (b, case["sq"], h, d), dt)
    s["k"] = _normal(g, (b, case["skv"], hk, d), dt)
    s["v"] = _normal(g, (b, case["skv"], hk, d), dt)
    s["mask"] = None
    if case["mask"] == "padded":
      share = torch.rand((b, 1), generator=g, device="cuda")
      s["mask"] = torch.arange(case["skv"], device="cuda")[None] < (share * (case["skv"] + 1)).floor()
    elif case["mask"] == "holes":
      s["mask"] = torch.rand((b, case["skv"]), generator=g, device="cuda") < 0.7
  return s


# ---- plain forms --------------------------------------------------------------------------------------------


def tiled(scale_byte, fmt):
  """Row-major block scales [rows, K / block] -> the tiled layout, one flat tensor."""
  rows, per_row = scale_byte.shape
  step = 256 // BLOCK[fmt]
  rt, kt = -(-rows // 128), -(-per_row // step) * step // 4
  full = scale_byte.new_zeros((rt * 128, kt * 4))
  full[:rows, :per_row] = scale_byte
  return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).reshape(-1)


def untiled(flat, rows, cols, fmt):
  per_row, rt = cols // BLOCK[fmt], -(-rows // 128)
  return flat.view(rt, -1, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, -1)[:rows, :per_row]


def scale_values(scale_byte, fmt):
  if fmt == "nvfp4":
    return scale_byte.contiguous().view(torch.float8_e4m3fn).float()
  return torch.tensor([2.0**(i - 127) for i in range(255)] + [math.nan], device=scale_byte.device)[scale_byte.long()]


def code_values(code):
  table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, 0, -0.5, -1, -1.5, -2, -3, -4, -6], device=code.device)
  return table[code.long()]


def power_of_two(exponent):
  return ((exponent + 127) << 23).to(torch.int32).view(torch.float32)


def quantize_plain(x, fmt):
  """x [rows, K] -> (codes 0..15 uint8 [rows, K], block scale bytes uint8 [rows, K / block], row scales f32 or None)."""
  rows, cols = x.shape
  xb = x.float().view(rows, cols // BLOCK[fmt], BLOCK[fmt])
  top = xb.abs().amax(dim=2)
  if fmt == "nvfp4":
    mantissa, exponent = torch.frexp(top.amax(dim=1))  # mantissa in [0.5, 1), 0 for 0
    exponent = torch.where(mantissa <= 0.65625, exponent - 12, exponent - 11)
    row = power_of_two(torch.where(mantissa > 0, exponent, -100).clamp(min=-100))
    scale = (top / (6 * row)[:, None]).to(torch.float8_e4m3fn)
    step = scale.float() * row[:, None]
    step = torch.where(step > 0, step, math.inf)
    byte = scale.view(torch.uint8)
  else:
    row = None
    exponent = torch.where(top > 0, torch.frexp(top)[1] - 3, -127).clamp(min=-127)
    byte = (exponent + 127).to(torch.uint8)
    step = scale_values(byte, fmt)
  y = xb / step[:, :, None]
  m = y.abs()
  index = sum(t.to(torch.uint8) for t in (m > 0.25, m >= 0.75, m > 1.25, m >= 1.75, m > 2.5, m >= 3.5, m > 5))
  code = index + 8 * (y < 0).to(torch.uint8)
  return code.view(rows, cols), byte, row


def dequantize_plain(code, byte, row, fmt):
  rows, cols = code.shape
  step = scale_values(byte, fmt)
  if row is not None:
    step = step * row[:, None]
  return (code_values(code).view(rows, -1, BLOCK[fmt]) * step[:, :, None]).view(rows, cols)


def linear_plain(x, w, bias, fmt, gelu):
  n, half = w["codes"].shape
  code = torch.stack([w["codes"] & 15, w["codes"] >> 4], dim=2).view(n, 2 * half)
  wf = dequantize_plain(code, untiled(w["block_scales"], n, 2 * half, fmt), w["row_scale"], fmt)
  y = dequantize_plain(*quantize_plain(x, fmt), fmt) @ wf.t() + bias.float()
  if gelu:
    y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y**3)))
  return y.to(x.dtype)


def normalise_plain(x, kind, eps=1e-6):
  if kind == "layer":
    x = x - x.mean(dim=-1, keepdim=True)
  return x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + eps)


def norm_plain(s, post, norm):
  """(x + gate * post(y), the norm of it), both in 32 bits."""
  y = s["y"].float()
  if post != "none":
    y = normalise_plain(y, post) * s["post_weight"].float()
  x = s["x"].float() + s["gate"].float()[:, None] * y
  h = normalise_plain(x, norm)
  if s.get("weight") is not None:
    h = h * s["weight"].float()
  if s.get("bias") is not None:
    h = h + s["bias"].float()
  if s.get("scale") is not None:
    h = h * (1 + s["scale"].float()[:, None]) + s["shift"].float()[:, None]
  return x, h


def attention_plain(q, k, v, mask):
  b, sq, h, d = q.shape
  hk = k.shape[2]
  qf = q.float().view(b, sq, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
  kf, vf = k.float().permute(0, 2, 3, 1), v.float().permute(0, 2, 1, 3)
  scores = (qf @ kf) * d**-0.5
  if mask is not None:
    vf = torch.where(mask[:, None, :, None], vf, 0.0)
    scores = torch.where(mask[:, None, None, :], scores, -math.inf)
  top = scores.amax(dim=-1, keepdim=True)
  p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))  # a prompt without any token: all zeros
  total = p.sum(dim=-1, keepdim=True)
  o = (p @ vf) / torch.where(total == 0, 1.0, total)
  return o.view(b, hk, h // hk, sq, d).permute(0, 3, 1, 2, 4).reshape(b, sq, h, d).to(q.dtype)


# ---- one pass -----------------------------------------------------------------------------------------------


def run(state):
  return (run_own if own else run_plain)(state)


def run_plain(s):
  case = s["case"]
  op = case["op"]
  if op == "quant":
    return dequantize_plain(*quantize_plain(s["x"], case["fmt"]), case["fmt"]).to(torch.bfloat16)
  if op == "linear":
    return linear_plain(s["x"], s["w"], s["bias"], case["fmt"], case["gelu"])
  if op == "norm":
    x, h = norm_plain(s, case["post"], case["norm"])
    return x.to(s["x"].dtype), h.to(s["x"].dtype)
  if op == "layer":
    x, h = norm_plain(s, "none", "layer")
    h = h.to(s["x"].dtype)  # what is quantised is the layer's activation in its own type
    out = linear_plain(h.view(-1, case["dim"]), s["w"], s["w_bias"], case["fmt"], False)
    return x.to(s["x"].dtype), out.view(*h.shape[:2], case["n"])
  return attention_plain(s["q"], s["k"], s["v"], s["mask"])


def run_own(s):
  import cache_dit_b200 as cache_dit
  case = s["case"]
  op = case["op"]
  if op == "quant":
    return cache_dit.float4_dequantize_rows(cache_dit.float4_quantize_rows(s["x"], case["fmt"]), torch.bfloat16)
  if op in ("linear", "layer"):
    k = case["k"] if op == "linear" else case["dim"]
    w = cache_dit.Float4Rows(s["w"]["codes"], s["w"]["block_scales"], s["w"]["row_scale"], case["fmt"], k)
  if op == "linear":
    return cache_dit.float4_linear(s["x"], w, s["bias"], gelu=case["gelu"])
  if op == "norm":
    post = None if case["post"] == "none" else case["post"]
    return cache_dit.gated_residual_norm(s["x"], s["y"], s["gate"], post_norm=post, post_weight=s.get("post_weight"), norm=case["norm"],
                                         weight=s.get("weight"), bias=s.get("bias"), scale=s.get("scale"), shift=s.get("shift"))
  if op == "layer":
    x, h = cache_dit.gated_residual_norm(s["x"], s["y"], s["gate"], norm="layer", scale=s["scale"], shift=s["shift"], quantize=case["fmt"])
    return x, cache_dit.float4_scaled_mm(h, w, s["w_bias"], out_dtype=s["x"].dtype)
  return cache_dit.cross_attention(s["q"], s["k"], s["v"], s["mask"])


# ---- what a pass cannot do without --------------------------------------------------------------------------


def _size(dtype):
  return 4 if dtype == F32 else 2


def _packed_bytes(rows, cols, fmt):
  return rows * cols // 2 + rows * cols // BLOCK[fmt] + (4 * rows if fmt == "nvfp4" else 0)


def work(case):
  op, e = case["op"], _size(case["dtype"])
  if op == "quant":
    n = case["rows"] * case["cols"]
    return dict(bytes=n * (e + 2) + 2 * _packed_bytes(case["rows"], case["cols"], case["fmt"]), flops=4 * n)
  if op == "linear":
    m, n, k = case["m"], case["n"], case["k"]
    return dict(bytes=m * k * e + _packed_bytes(n, k, case["fmt"]) + n * e + m * n * e, flops=2 * m * n * k)
  if op == "norm":
    n, extra = case["batch"] * case["tokens"] * case["dim"], (3 * case["batch"] + 3) * case["dim"]
    return dict(bytes=(4 * n + extra) * e, flops=14 * n)
  if op == "layer":
    m, k, n = case["batch"] * case["tokens"], case["dim"], case["n"]
    return dict(bytes=(3 * m * k + m * n + n) * e + _packed_bytes(n, k, case["fmt"]), flops=2 * m * n * k)
  b, sq, skv, h, hk, d = (case[i] for i in ("batch", "sq", "skv", "heads", "kv_heads", "d"))
  return dict(bytes=(2 * b * sq * h * d + 2 * b * skv * hk * d) * e + (b * skv if case["mask"] != "none" else 0), flops=4 * b * h * sq * skv * d)


# ---- the definitions in 64 bits -----------------------------------------------------------------------------


def _two_to(exponent):
  return ((exponent.long() + 1023) << 52).view(torch.float64)


def _floor_log2(x):
  return torch.frexp(x)[1] - 1


def _quantized64(x, fmt):
  """The values that the 4-bit form of x [rows, K] stands for."""
  x = x.double()
  blocks = x.unflatten(1, (-1, BLOCK[fmt]))
  top = blocks.abs().max(dim=2).values
  if fmt == "nvfp4":
    least = (top.max(dim=1).values / 2688).clamp(min=2.0**-100)
    row = _two_to(_floor_log2(least))
    row = torch.where(row < least, 2 * row, row)
    t = top / (6 * row[:, None])
    grid = _two_to(_floor_log2(t.clamp(min=2.0**-6)) - 3)  # e4m3: three bits behind the first, 2^-9 at least
    step = torch.round(t / grid) * grid * row[:, None]
  else:
    step = _two_to((_floor_log2(top.clamp(min=2.0**-140)) - 2).clamp(min=-127))
  y = blocks / torch.where(step > 0, step, math.inf)[:, :, None]
  m = y.abs()
  m = torch.where(m < 2, torch.round(2 * m) / 2, torch.where(m < 4, torch.round(m), 2 * torch.round(m / 2))).clamp(max=6)
  return (torch.sign(y) * m * step[:, :, None]).view(x.shape)


def _weight64(w, k, fmt):
  n = w["codes"].shape[0]
  low, high = w["codes"] % 16, w["codes"] // 16
  code = torch.empty((n, k), dtype=torch.uint8, device=low.device)
  code[:, 0::2], code[:, 1::2] = low, high
  r, c = torch.meshgrid(torch.arange(n, device=low.device), torch.arange(k // BLOCK[fmt], device=low.device), indexing="ij")
  step = 256 // BLOCK[fmt]
  tiles = -(-k // 256) * step // 4
  at = ((r // 128) * tiles + c // 4) * 512 + (r % 32) * 16 + (r % 128) // 32 * 4 + c % 4
  scale = scale_values(w["block_scales"][at], fmt).double()
  if w["row_scale"] is not None:
    scale = scale * w["row_scale"].double()[:, None]
  return code_values(code).double() * scale.repeat_interleave(BLOCK[fmt], dim=1)


def _norm64(x, kind):
  if kind == "rms":
    return x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
  return (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-6)


def exact(case, seed):
  s = prepare(case, seed)
  op = case["op"]
  d64 = {name: t.double() for name, t in s.items() if torch.is_tensor(t)}
  if op == "quant":
    return _quantized64(s["x"], case["fmt"])
  if op == "linear":
    y = _quantized64(s["x"], case["fmt"]) @ _weight64(s["w"], case["k"], case["fmt"]).t() + d64["bias"]
    if case["gelu"]:
      y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * y * (1 + 0.044715 * y * y)))
    return y
  if op in ("norm", "layer"):
    y = d64["y"]
    if case.get("post", "none") != "none":
      y = _norm64(y, case["post"]) * d64["post_weight"]
    x = d64["x"] + d64["gate"].unsqueeze(1) * y
    h = _norm64(x, case.get("norm", "layer")) * d64.get("weight", 1.0) + d64.get("bias", 0.0)
    if "scale" in d64:
      h = h * (1 + d64["scale"].unsqueeze(1)) + d64["shift"].unsqueeze(1)
    if op == "norm":
      return x, h
    h = h.to(s["x"].dtype).view(-1, case["dim"])
    out = _quantized64(h, case["fmt"]) @ _weight64(s["w"], case["dim"], case["fmt"]).t() + d64["w_bias"]
    return x, out.view(*x.shape[:2], case["n"])
  out = torch.zeros_like(s["q"], dtype=torch.float64)
  group = case["heads"] // case["kv_heads"]
  for b in range(case["batch"]):
    keep = slice(None) if s["mask"] is None else s["mask"][b].nonzero()[:, 0]
    k, v = s["k"][b, keep].double(), s["v"][b, keep].double()
    if not len(k):
      continue
    for h in range(case["heads"]):
      p = torch.softmax(s["q"][b, :, h].double() @ k[:, h // group].t() / math.sqrt(case["d"]), dim=-1)
      out[b, :, h] = p @ v[:, h // group]
  return out
