"""What the 8-bit operators are timed on: dense layers and experts whose operands are
8-bit floating point numbers (e4m3) with a scale for each block of 128, and the passes
that make such operands.

Blocks run along the reduction index of the product an operand is made for: 128
consecutive values of a row share the power of two 2^e with the smallest e for which
their largest magnitude is at most 448 * 2^e (not below -117), and stand for q * 2^e.
A block with an infinity or a NaN is NaN as a whole.  A row is filled up with zeros to
whole blocks; its exponents are bytes (e + 127), as many as whole groups of four blocks
have.

A case is a dict of plain values:

  kind       "quantize": a tensor's rows and its columns as 8-bit operands
             "norm": residual sum, RMS norm and padding mask, the result in 8 bits
             "product": y[e] = act(a[e] . w[e]^T) of 8-bit operands
             "backward": the gradients of such a product from the gradient of its
             output, which is made an 8-bit operand both ways first
             "mlp": norm, wi (relu, hidden tensor in 8 bits) and wo of a dense block
  dtype      "bf16" or "f32": of the tensors that are not 8-bit operands
  experts, rows, width, columns   sizes: a [experts, rows, width], w [experts,
             columns, width]
  activation, eight_bit   of the product: its activation, and whether the result is an
             8-bit operand (of the next product) or bf16
  ragged     experts hold between none and all of their rows
  masked     norm: padding rows; quantize, backward: a ReLU's mask
"""

import math

import torch

own = False

BLOCK = 128
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(name, kind, rows, width, columns=0, experts=1, dtype="bf16",
          activation="linear", eight_bit=False, ragged=False, masked=False):
  case = dict(kind=kind, dtype=dtype, experts=experts, rows=rows, width=width,
              columns=columns, activation=activation, eight_bit=eight_bit,
              ragged=ragged, masked=masked)
  if name:
    case["name"] = name
  return case


def listed():
  return [
      # Pre-training: the tokens of a step as operands of the forward product and of
      # the weight gradient.
      _case("quantize_64k", "quantize", 65536, 4096),
      # Fine-tuning on texts of odd lengths: the gradient of a hidden tensor behind a
      # ReLU.
      _case("quantize_ragged", "quantize", 6 * 1500, 2050, masked=True),
      # A decoding step of 32 sequences: the norm in front of a layer.
      _case("norm_decode", "norm", 32, 1024),
      # The same over packed rows of texts, with padding.
      _case("norm_packed", "norm", 32 * 1000, 4096, masked=True),
      # One token through a dense layer: a stream over its weights.
      _case("dense_decode", "product", 1, 4096, 16384, activation="relu",
            eight_bit=True),
      # The experts of a decoding step: few rows each.
      _case("experts_decode", "product", 6, 4096, 1024, experts=64),
      # Skewed routing: 64 experts with unequal shares of a padded buffer.
      _case("experts_ragged", "product", 705, 1024, 4096, experts=64,
            activation="relu", ragged=True),
      # A dense layer over whole prompts: one large product.
      _case("dense_32k", "product", 32768, 4096, 16384),
      # Training on texts of odd lengths: gradients of a dense layer behind a ReLU.
      _case("dense_backward", "backward", 8 * 1385, 1024, 4096, masked=True),
      # Training of experts with unequal shares.
      _case("experts_backward", "backward", 640, 4096, 1024, experts=32,
            ragged=True),
      # A dense block for one token of each of 8 sequences, and over whole prompts.
      _case("mlp_decode", "mlp", 8, 1024, 4096),
      _case("mlp_prefill", "mlp", 16384, 1024, 4096),
  ]


def _log_int(rng, low, high):
  return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
  """Mostly widths of models, which are multiples of 64; odd ones among them."""
  n = _log_int(rng, low, high)
  return n if rng.random() < 0.3 else max(64, 64 * int(round(n / 64.0)))


def _draw(rng):
  kind = rng.choice(["quantize", "norm", "product", "product", "product", "backward",
                     "mlp"])
  dtype = "f32" if kind in ("quantize", "norm") and rng.random() < 0.25 else "bf16"
  if kind in ("quantize", "norm"):
    return _case(None, kind, _log_int(rng, 1, 65536), _width(rng, 64, 8192),
                 dtype=dtype, masked=rng.random() < 0.5)
  if kind == "mlp":
    width = _width(rng, 256, 4096)
    return _case(None, kind, _log_int(rng, 1, 16384), width, 4 * width)
  experts = rng.choice([1, 1, _log_int(rng, 2, 64)])
  return _case(
      None, kind, _log_int(rng, 1 if kind == "product" else 64, 32768),
      _width(rng, 128, 8192), _width(rng, 64, 16384), experts=experts,
      activation=rng.choice(["linear", "relu", "gelu"]) if kind == "product"
      else "linear",
      eight_bit=kind == "product" and rng.random() < 0.3,
      ragged=experts > 1 and rng.random() < 0.5,
      masked=kind == "backward" and rng.random() < 0.5)


def draw(rng):
  """One more case of the same ranges, without a name; never more work than the
  largest of the listed ones."""
  cost = [work(c) for c in listed()]
  flops, moved = (max(w[k] for w in cost) for k in ("flops", "bytes"))
  while True:
    case = _draw(rng)
    # (and no more than 2 GB of weights)
    if (work(case)["flops"] <= flops and work(case)["bytes"] <= moved and
        case["experts"] * case["width"] * case["columns"] <= 1 << 31):
      return case


def work(case):
  """A pass reads its inputs once and writes its outputs once; 8-bit outputs of
  quantize, norm and eight_bit products leave it as the bf16 values they stand for."""
  e, r, k, n = (case[x] for x in ("experts", "rows", "width", "columns"))
  b = 4 if case["dtype"] == "f32" else 2
  if case["kind"] == "quantize":
    return {"bytes": r * k * (b * (2 if case["masked"] else 1) + 2 + 2),
            "flops": 4 * r * k}
  if case["kind"] == "norm":
    return {"bytes": r * k * (3 * b + 2) + k * b, "flops": 8 * r * k}
  # (ragged: half of the rows on average)
  live = r / 2.0 if case["ragged"] else r
  eight = 1 + 1.0 / BLOCK
  if case["kind"] == "product":
    return {"bytes": e * (live * k * eight + n * k * eight + live * n * 2),
            "flops": 2.0 * e * live * k * n}
  if case["kind"] == "backward":
    return {"bytes": e * (live * k * eight + n * k * eight +
                          live * n * 2 * (2 if case["masked"] else 1) +
                          live * k * 2 + k * n * 2),
            "flops": 4.0 * e * live * k * n}
  return {"bytes": r * k * 2 * 4 + 2 * n * k * eight, "flops": 4.0 * r * k * n}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _padded(n):
  return (n + BLOCK - 1) // BLOCK * BLOCK


def _power_of_two(e):
  """2^e in float32, of whole numbers from -126 to 127."""
  return ((e.int() + 127) << 23).view(torch.float32)


def _exponents(blocks):
  """The exponents of float32 blocks [..., 128], and which hold an infinity or a NaN."""
  top = blocks.abs().amax(-1)
  bad = ~torch.isfinite(top)
  mantissa, e = torch.frexp(torch.where(bad, torch.zeros_like(top), top))
  # top = mantissa * 2^e with mantissa in [1/2, 1); 448 = 7/8 * 2^9
  e = e - 9 + (mantissa > 0.875).int()
  return torch.where(top == 0, torch.full_like(e, -117), e).clamp_min(-117), bad


def _quantize(x):
  """float32 [..., n] -> e4m3 values [..., padded n], exponent bytes [..., blocks]."""
  n = x.shape[-1]
  x = torch.nn.functional.pad(x, (0, _padded(n) - n))
  blocks = x.reshape(x.shape[:-1] + (-1, BLOCK))
  e, bad = _exponents(blocks)
  scaled = blocks * _power_of_two(-e).unsqueeze(-1)
  scaled = torch.where(bad.unsqueeze(-1), torch.full_like(scaled, float("nan")), scaled)
  values = scaled.to(torch.float8_e4m3fn).reshape(x.shape)
  e = torch.where(bad, torch.zeros_like(e), e)
  bytes_ = (e + 127).to(torch.uint8)
  return values, torch.nn.functional.pad(bytes_, (0, -bytes_.shape[-1] % 4), value=127)


def _stands_for(values, scales, n):
  """What 8-bit operands stand for, float32 [..., n]."""
  blocks = values.float().reshape(values.shape[:-1] + (-1, BLOCK))
  unit = _power_of_two(scales[..., :blocks.shape[-2]].int() - 127)
  return (blocks * unit.unsqueeze(-1)).reshape(values.shape)[..., :n]


def _act(y, activation):
  if activation == "relu":
    return torch.relu(y)
  if activation == "gelu":
    return y * 0.5 * (1 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
  return y


def _rounded(x):
  """What x's 8-bit form stands for, as bf16 (which holds all such values)."""
  return _stands_for(*_quantize(x), x.shape[-1]).bfloat16()


def _live(state, t):
  """t [experts, rows, ...] with zeros behind the experts' last rows."""
  if state["count"] is None:
    return t
  at = torch.arange(t.shape[1], device=t.device)
  return torch.where((at[None] < state["count"][:, None])[..., None], t,
                     torch.zeros((), dtype=t.dtype, device=t.device))


def _plain(state):
  case = state["case"]
  kind = case["kind"]
  if kind == "quantize":
    x = state["x"].float()
    if case["masked"]:
      x = torch.where(state["mask"] > 0, x, torch.zeros_like(x))
    return _rounded(x), _rounded(x.t().contiguous())
  if kind in ("norm", "mlp"):
    dtype = state["x"].dtype
    total = (state["x"].float() + state["residual"].float()).to(dtype)
    t = total.float()
    y = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * state["scale"].float()
    if case["masked"]:
      y = y * state["mask"].float()[:, None]
    if kind == "norm":
      return total, _rounded(y)
    a = _stands_for(*_quantize(y), y.shape[-1])
    h = torch.relu(a @ _stands_for(*state["wi"], case["width"])[0].t())
    h = _stands_for(*_quantize(h), case["columns"])
    return total, (h @ _stands_for(*state["wo"], case["columns"])[0].t()).bfloat16()
  if kind == "product":
    a = _stands_for(*state["a"], case["width"])
    w = _stands_for(*state["w"], case["width"])
    y = _act(torch.matmul(a, w.transpose(1, 2)), case["activation"])
    return _live(state, _rounded(y) if case["eight_bit"] else y.bfloat16())
  dy = state["dy"].float()
  if case["masked"]:
    dy = torch.where(state["mask"] > 0, dy, torch.zeros_like(dy))
  dy = _live(state, dy)
  by_row = _stands_for(*_quantize(dy), case["columns"])
  da = torch.matmul(by_row, _stands_for(*state["w_rows"], case["columns"])
                    .transpose(1, 2))
  by_column = _stands_for(*_quantize(dy.transpose(1, 2).contiguous()), case["rows"])
  dw = torch.matmul(_stands_for(*state["a_columns"], case["rows"]),
                    by_column.transpose(1, 2))
  return _live(state, da.bfloat16()), dw.bfloat16()


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(state):
  from mesh_amd import fp8_hip
  case = state["case"]
  kind = case["kind"]

  def operand(name, n):
    return fp8_hip.Fp8Blocks(state[name][0], state[name][1], n)

  if kind == "quantize":
    rows, columns = fp8_hip.quantize(
        state["x"], rows=True, columns=True,
        relu_mask=state["mask"] if case["masked"] else None)
    return fp8_hip.dequantize(rows), fp8_hip.dequantize(columns)
  if kind in ("norm", "mlp"):
    total, y = fp8_hip.residual_rms_norm(
        state["x"], state["residual"], state["scale"],
        row_mask=state["mask"] if case["masked"] else None)
    if kind == "norm":
      return total, fp8_hip.dequantize(y)
    h = fp8_hip.dense(y, operand("wi", case["width"]), "relu", eight_bit=True)
    return total, fp8_hip.dense(h, operand("wo", case["columns"]))
  if kind == "product":
    out = state["out"]
    if isinstance(out, tuple):
      out = operand("out", case["columns"])
    y = fp8_hip.expert_linear(
        operand("a", case["width"]), operand("w", case["width"]), case["activation"],
        eight_bit=case["eight_bit"], row_count=state["count"], out=out)
    return fp8_hip.dequantize(y) if case["eight_bit"] else y
  return fp8_hip.expert_linear_backward(
      operand("a_columns", case["rows"]), state["dy"], operand("w_rows", case["columns"]),
      relu_mask=state["mask"] if case["masked"] else None, row_count=state["count"],
      da=state["da"])


def run(state):
  return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the program around the pass
# ---------------------------------------------------------------------------
def _normal(gen, sizes, std=1.0):
  return torch.randn(sizes, generator=gen, device="cuda") * std


def _tokens(gen, sizes):
  """What flows between layers: some features are much larger than the others, and
  tokens differ in size."""
  features = torch.exp(_normal(gen, sizes[-1:], 0.7))
  tokens = torch.exp(_normal(gen, sizes[:-1] + (1,), 0.3))
  return _normal(gen, sizes) * features * tokens


def _operand(gen, sizes, std):
  """Random 8-bit operands, made an expert at a time."""
  made = [_quantize(_normal(gen, sizes[1:], std)) for _ in range(sizes[0])]
  return torch.stack([m[0].view(torch.uint8) for m in made]).view(
      torch.float8_e4m3fn), torch.stack([m[1] for m in made])


def prepare(case, seed):
  """What the program has before the pass: tokens or gradients as the layers around
  leave them, weights as 8-bit operands laid out once, and the buffers that hold an
  expert's rows from step to step."""
  gen = torch.Generator(device="cuda").manual_seed(seed)
  dtype = DTYPES[case["dtype"]]
  e, r, k, n = (case[x] for x in ("experts", "rows", "width", "columns"))
  state = {"case": case, "count": None, "out": None, "da": None}
  if case["ragged"]:
    state["count"] = torch.randint(0, r + 1, (e,), generator=gen, device="cuda",
                                   dtype=torch.int32)
  kind = case["kind"]
  if kind == "quantize":
    state["x"] = _tokens(gen, (r, k)).to(dtype)
    if case["masked"]:
      state["mask"] = torch.relu(_normal(gen, (r, k))).to(dtype)
  elif kind in ("norm", "mlp"):
    state["x"] = _tokens(gen, (r, k)).to(dtype)
    state["residual"] = _tokens(gen, (r, k)).to(dtype)
    state["scale"] = (1 + _normal(gen, (k,), 0.1)).to(dtype)
    if case["masked"]:
      state["mask"] = (torch.rand((r,), generator=gen, device="cuda") < 0.8).to(dtype)
    if kind == "mlp":
      state["wi"] = _operand(gen, (1, n, k), k ** -0.5)
      state["wo"] = _operand(gen, (1, k, n), n ** -0.5)
  elif kind == "product":
    made = [_quantize(_tokens(gen, (r, k))) for _ in range(e)]
    state["a"] = (torch.stack([m[0].view(torch.uint8) for m in made]).view(
        torch.float8_e4m3fn), torch.stack([m[1] for m in made]))
    state["w"] = _operand(gen, (e, n, k), k ** -0.5)
    if case["ragged"]:
      if case["eight_bit"]:
        blocks = -(-n // BLOCK)
        state["out"] = (
            torch.zeros((e, r, _padded(n)), dtype=torch.uint8, device="cuda").view(
                torch.float8_e4m3fn),
            torch.full((e, r, (blocks + 3) // 4 * 4), 127, dtype=torch.uint8,
                       device="cuda"))
      else:
        state["out"] = torch.zeros((e, r, n), dtype=dtype, device="cuda")
  else:
    # (the forward pass left the columns of its input; rows behind an expert's last
    # one are zeros there)
    made = []
    for i in range(e):
      a = _tokens(gen, (r, k))
      if case["ragged"]:
        a[int(state["count"][i]):] = 0
      made.append(_quantize(a.t().contiguous()))
    state["a_columns"] = (torch.stack([m[0].view(torch.uint8) for m in made]).view(
        torch.float8_e4m3fn), torch.stack([m[1] for m in made]))
    state["w_rows"] = _operand(gen, (e, k, n), k ** -0.5)
    state["dy"] = (_tokens(gen, (e, r, n)) * 1e-3).to(dtype)
    if case["masked"]:
      state["mask"] = torch.relu(_normal(gen, (e, r, n))).to(dtype)
    if case["ragged"]:
      state["da"] = torch.zeros((e, r, k), dtype=dtype, device="cuda")
  return state


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _eight_bit_64(x):
  """float64 [..., n] -> what its 8-bit form stands for, float64.  Normal numbers of
  e4m3 have three bits behind the first, the steps below 2^-6 are 2^-9."""
  out = torch.empty_like(x)
  for at in range(0, x.shape[-1], BLOCK):
    part = x[..., at:at + BLOCK]
    top = part.abs().max(-1, keepdim=True).values
    e = torch.ceil(torch.log2(torch.clamp(top, min=2.0 ** -130) / 448.0))
    # (log2 rounds: settle the neighbours by comparison)
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e)
    unit = torch.exp2(torch.clamp(e, min=-117.0))
    q = part / unit
    binade = torch.floor(torch.log2(torch.clamp(q.abs(), min=2.0 ** -6)))
    binade = torch.where(torch.exp2(binade) > torch.clamp(q.abs(), min=2.0 ** -6),
                         binade - 1, binade)
    binade = torch.where(torch.exp2(binade + 1) <= q.abs(), binade + 1, binade)
    step = torch.exp2(binade - 3)
    out[..., at:at + BLOCK] = torch.round(q / step) * step * unit
  return out


def _value_64(operand, n):
  values, scales = operand
  factor = torch.exp2(scales.double() - 127)
  factor = factor.repeat_interleave(BLOCK, dim=-1)[..., :values.shape[-1]]
  return (values.float().double() * factor)[..., :n]


def exact(case, seed):
  state = prepare(case, seed)
  kind = case["kind"]
  live = None
  if case["ragged"]:
    live = (torch.arange(case["rows"], device="cuda") <
            state["count"].unsqueeze(1)).double().unsqueeze(2)
  if kind == "quantize":
    x = state["x"].double()
    if case["masked"]:
      x = x * (state["mask"] > 0)
    return _eight_bit_64(x), _eight_bit_64(x.t()).contiguous()
  if kind in ("norm", "mlp"):
    # (the sum is a tensor of its own, rounded to its type: the norm is of that one)
    total = state["x"].double() + state["residual"].double()
    t = total.to(state["x"].dtype).double()
    y = t / torch.sqrt(t.square().sum(-1, keepdim=True) / case["width"] + 1e-6)
    y = y * state["scale"].double()
    if case["masked"]:
      y = y * state["mask"].double().unsqueeze(1)
    y = _eight_bit_64(y)
    if kind == "norm":
      return total, y
    h = y @ _value_64(state["wi"], case["width"])[0].t()
    h = _eight_bit_64(h.clamp_min(0))
    return total, h @ _value_64(state["wo"], case["columns"])[0].t()
  if kind == "product":
    y = torch.stack([
        _act(a @ w.t(), case["activation"])
        for a, w in zip(_value_64(state["a"], case["width"]),
                        _value_64(state["w"], case["width"]))])
    if case["eight_bit"]:
      y = _eight_bit_64(y)
    return y if live is None else y * live
  dy = state["dy"].double()
  if case["masked"]:
    dy = dy * (state["mask"] > 0)
  if live is not None:
    dy = dy * live
  w = _value_64(state["w_rows"], case["columns"])
  a = _value_64(state["a_columns"], case["rows"])
  da = torch.stack([_eight_bit_64(d) @ v.t() for d, v in zip(dy, w)])
  dw = torch.stack([u @ _eight_bit_64(d.t()).t() for d, u in zip(dy, a)])
  return da if live is None else da * live, dw
