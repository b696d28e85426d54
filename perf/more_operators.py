"""What the paged cache is timed on: writing keys and values into pages (in the
activations' type, or in 8 bits), reading them back, and attention of one new token over
them, with and without the write of the token's own row.

A cache is two buffers of pages, [pages, kv_heads, page, width]; a sequence's position p
lies in page table[b, p // page], row p % page.  8-bit caches hold e4m3 values; each 128
consecutive values of a row (the last block of a row may be shorter) share the power of
two 2^e with the smallest e >= -117 for which their largest magnitude is at most
448 * 2^e, kept as the byte e + 127.

A case is a dict of plain values:

  kind       "write": rows of keys and values go into the pages, and are read back
             "read": the pages of sequences as dense tensors
             "attention": one query per sequence over what the cache holds of it
             "step": the same, the token's own key and value written first; the written
             rows are read back
  dtype      "bf16" or "f32": of the queries, of rows and results
  eight_bit  whether the cache holds e4m3 values (else values of `dtype`)
  batch      sequences
  length     positions of the longest sequence (write: rows of the longest)
  heads, kv_heads, width   query heads, key/value heads, values per head
  page       rows of a page
  ragged     sequences differ in length, from a few positions up to `length`
  bias       a learned relative position bias by buckets
"""

import math

import torch

own = False

BLOCK = 128
BUCKETS = 32
DISTANCE = 128                    # farther positions share the last bucket
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def _case(name, kind, batch, length, heads, kv_heads, width, page, dtype="bf16",
          eight_bit=False, ragged=False, bias=False):
  case = dict(kind=kind, dtype=dtype, eight_bit=eight_bit, batch=batch, length=length,
              heads=heads, kv_heads=kv_heads, width=width, page=page, ragged=ragged,
              bias=bias)
  if name:
    case["name"] = name
  return case


def listed():
  return [
      # Prompts of different lengths enter an 8-bit cache.
      _case("write_prompts", "write", 16, 4096, 16, 16, 64, 64, eight_bit=True,
            ragged=True),
      # The rows of one decoding step of 64 sequences.
      _case("write_rows", "write", 64, 1, 8, 8, 128, 16),
      # What an 8-bit cache holds of four long texts, for a pass over more of them.
      _case("read_texts", "read", 4, 16384, 32, 8, 128, 64, eight_bit=True),
      # The same of short sequences with heads of an odd size.
      _case("read_odd", "read", 23, 1000, 6, 6, 80, 32, ragged=True),
      # One sequence of a small model: latency.
      _case("attend_one", "attention", 1, 700, 16, 16, 64, 16),
      # A decoding step of 32 sequences through a layer with a relative position bias.
      _case("attend_biased", "attention", 32, 1024, 16, 16, 64, 32, ragged=True,
            bias=True),
      # One very long text in 8 bits, query heads in groups.
      _case("attend_long", "attention", 1, 131072, 32, 8, 128, 128, eight_bit=True),
      # A full server: many sequences of all lengths.
      _case("attend_many", "attention", 128, 16384, 32, 8, 128, 64, ragged=True),
      # In float32, with heads of an odd size.
      _case("attend_f32", "attention", 9, 2500, 12, 4, 96, 16, dtype="f32", ragged=True),
      # A layer's step with its own row, in the sizes of a transformer block.
      _case("step_block", "step", 32, 1024, 16, 16, 64, 32, bias=True),
      # The same for a server's sequences in 8 bits.
      _case("step_server", "step", 64, 8192, 32, 8, 128, 64, eight_bit=True, ragged=True),
      # One sequence whose query heads share one wide key and value head.
      _case("step_shared", "step", 1, 2001, 8, 1, 256, 16, eight_bit=True),
  ]


def _log_int(rng, low, high):
  return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw(rng):
  kind = rng.choice(["write", "read", "attention", "attention", "step"])
  kv_heads = rng.choice([1, 2, 4, 6, 8, 8, 12, 16, 16, 32])
  group = rng.choice([1, 1, 1, 2, 3, 4, 4, 7, 8, 16])
  width = rng.choice([64, 64, 128, 128, 128, 32, 80, 96, 112, 192, 256, 36, 100])
  if kind == "write":
    batch, length = rng.choice([(_log_int(rng, 1, 256), 1),
                                (_log_int(rng, 1, 32), _log_int(rng, 2, 8192))])
  else:
    batch, length = _log_int(rng, 1, 256), _log_int(rng, 1, 131072)
  return _case(
      None, kind, batch, length, kv_heads * group, kv_heads, width,
      rng.choice([8, 16, 16, 32, 64, 128, 256]),
      dtype="f32" if rng.random() < 0.2 else "bf16", eight_bit=rng.random() < 0.5,
      ragged=batch > 1 and rng.random() < 0.6,
      bias=kind in ("attention", "step") and rng.random() < 0.3)


def draw(rng):
  """One more case of the same ranges, without a name; never more work than the largest
  listed one of its kind or of attention."""
  cost = [work(c) for c in listed()]
  most = {k: max(w[k] for w in cost) for k in ("bytes", "flops")}
  copied = 1 << 28               # values that a write or read moves at most
  while True:
    case = _draw(rng)
    if case["kind"] in ("write", "read") and (
        sum(_lengths(case)) * case["kv_heads"] * case["width"] > copied):
      continue
    if all(v <= most[k] for k, v in work(case).items()):
      return case


def _lengths(case):
  """The sequences' lengths, in rising order."""
  b, n = case["batch"], case["length"]
  if not case["ragged"]:
    return [n] * b
  return [max(1, n * (i + 1) // b) for i in range(b)]


def _value_bytes(case):
  """Of a stored value, its part of a scale included."""
  if case["eight_bit"]:
    return 1 + -(-case["width"] // BLOCK) / case["width"]
  return 4 if case["dtype"] == "f32" else 2


def work(case):
  """A pass reads its inputs once and writes its outputs once."""
  b = 4 if case["dtype"] == "f32" else 2
  row = 2 * case["kv_heads"] * case["width"]       # values of a position
  rows, stored = sum(_lengths(case)), _value_bytes(case)
  dense = case["batch"] * case["length"]           # rows of a dense result
  if case["kind"] == "write":
    # (the rows, the pages, and the way back)
    return {"bytes": row * (rows * (b + 2 * stored) + dense * b), "flops": 2 * rows * row}
  if case["kind"] == "read":
    return {"bytes": row * (rows * stored + dense * b), "flops": rows * row}
  q = case["batch"] * case["heads"] * case["width"]
  moved = rows * row * stored + 2 * q * b
  if case["kind"] == "step":
    moved += case["batch"] * row * (2 * b + stored)
  return {"bytes": moved, "flops": 4 * rows * case["heads"] * case["width"]}


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------
def _power_of_two(e):
  """2^e in float32, of whole numbers from -126 to 127."""
  return ((e.int() + 127) << 23).view(torch.float32)


def _to_eight_bits(x):
  """float32 [..., width] -> e4m3 values of the same shape, exponent bytes
  [..., blocks]."""
  values, scales = [], []
  for part in x.split(BLOCK, dim=-1):
    top = part.abs().amax(-1)
    bad = ~torch.isfinite(top)
    mantissa, e = torch.frexp(torch.where(bad, torch.zeros_like(top), top))
    # top = mantissa * 2^e with mantissa in [1/2, 1); 448 = 7/8 * 2^9
    e = (e - 9 + (mantissa > 0.875).int()).clamp_min(-117)
    e = torch.where(top == 0, torch.full_like(e, -117), e)
    q = part * _power_of_two(-e).unsqueeze(-1)
    q = torch.where(bad.unsqueeze(-1), torch.full_like(q, float("nan")), q)
    values.append(q.to(torch.float8_e4m3fn).view(torch.uint8))
    scales.append((torch.where(bad, torch.zeros_like(e), e) + 127).to(torch.uint8))
  return torch.cat(values, -1).view(torch.float8_e4m3fn), torch.stack(scales, -1)


def _from_eight_bits(values, scales):
  unit = _power_of_two(scales.int() - 127)
  unit = unit.repeat_interleave(BLOCK, dim=-1)[..., :values.shape[-1]]
  return values.float() * unit


def _slots(state, positions):
  """Page and row of positions [batch, n]."""
  page = state["case"]["page"]
  return state["table"].gather(1, positions // page).long(), positions % page


def _store(state, rows, positions, there):
  """rows: keys and values, [batch, n, kv_heads * width]; only where `there` [batch, n]
  is set."""
  case = state["case"]
  pages, at = _slots(state, positions)
  pages, at = pages[there], at[there]
  for name, x in zip("kv", rows):
    x = x[there].reshape(-1, case["kv_heads"], case["width"])
    if case["eight_bit"]:
      values, scales = _to_eight_bits(x.float())
      state[name + "_pages"].view(torch.uint8)[pages, :, at] = values.view(torch.uint8)
      state[name + "_scales"][pages, :, at] = scales
    else:
      state[name + "_pages"][pages, :, at] = x


def _load(state, name, table, positions):
  """float32 [batch, n, kv_heads, width] of positions [batch, n] or [n]."""
  page = state["case"]["page"]
  positions = positions.expand(table.shape[0], -1)
  pages, at = table.gather(1, positions // page).long(), positions % page
  if not state["case"]["eight_bit"]:
    return state[name + "_pages"][pages, :, at].float()
  values = state[name + "_pages"].view(torch.uint8)[pages, :, at]
  return _from_eight_bits(values.view(torch.float8_e4m3fn),
                          state[name + "_scales"][pages, :, at])


def _dense(state, positions, there):
  """Keys and values [batch, n, kv_heads * width] in the case's type, zeros where
  nothing is."""
  dtype = DTYPES[state["case"]["dtype"]]
  out = []
  for name in "kv":
    x = _load(state, name, state["table"], positions).flatten(2)
    out.append(torch.where(there.unsqueeze(-1), x, torch.zeros_like(x)).to(dtype))
  return out


def _attend(state):
  case = state["case"]
  b, heads, kv, width = (case[x] for x in ("batch", "heads", "kv_heads", "width"))
  n, group = case["length"], case["heads"] // case["kv_heads"]
  outs = []
  at_once = max(1, (1 << 28) // (n * kv * width))     # sequences
  positions = torch.arange(n, device="cuda")
  for first in range(0, b, at_once):
    part = slice(first, first + at_once)
    table, last = state["table"][part], state["position"][part].long()
    # (positions behind a sequence have no page: any page there is, masked below)
    pages = table.clamp_min(0)
    k = _load(state, "k", pages, positions).permute(0, 2, 3, 1).contiguous()
    q = state["q"][part].float().reshape(-1, kv, group, width)
    logits = torch.matmul(q, k)
    del k
    if case["bias"]:
      distance = (positions[None] - last[:, None]).clamp(1 - state["reach"], 0)
      bucket = state["bucket"].long()[distance + state["reach"] - 1]
      bias = state["values"].float()[:, bucket]       # [heads, sequences, n]
      logits = logits + bias.permute(1, 0, 2).reshape(-1, kv, group, n)
    seen = (positions[None] <= last[:, None])[:, None, None]
    logits = torch.where(seen, logits, torch.full_like(logits, -math.inf))
    top = logits.amax(-1, keepdim=True)
    w = torch.exp(logits - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    v = _load(state, "v", pages, positions)
    v = torch.where(seen.squeeze(1).squeeze(1)[..., None, None], v, torch.zeros_like(v))
    o = torch.matmul(w, v.transpose(1, 2).contiguous()) / w.sum(-1, keepdim=True)
    outs.append(o.reshape(-1, heads * width).to(DTYPES[case["dtype"]]))
  return torch.cat(outs)


def _rows(state):
  """Positions of a call's rows, and which of them there are: [batch, n]."""
  n = torch.arange(state["rows"], device="cuda")
  positions = state["start"].long()[:, None] + n
  there = n < state["count"].long()[:, None]
  return torch.where(there, positions, torch.zeros_like(positions)), there


def _plain(state):
  kind = state["case"]["kind"]
  if kind in ("write", "step"):
    positions, there = _rows(state)
    _store(state, (state["k"], state["v"]), positions, there)
  if kind == "write":
    return tuple(_dense(state, positions, there))
  if kind == "read":
    return tuple(_dense(state, *_rows(state)))
  if kind == "attention":
    return _attend(state)
  k, v = _dense(state, positions, there)
  return _attend(state), k[:, 0], v[:, 0]


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
def _own(state):
  from mesh_amd import cache_hip
  case = state["case"]
  kind = case["kind"]
  cache = cache_hip.PagedCache(state["k_pages"], state["v_pages"],
                               state.get("k_scales"), state.get("v_scales"))
  table, dtype = state["table"], DTYPES[case["dtype"]]
  if kind == "write":
    cache_hip.write(cache, state["k"], state["v"], table, state["start"],
                    count=state["count"])
  if kind in ("write", "read"):
    return cache_hip.read(cache, table, state["start"], state["rows"],
                          count=state["count"], dtype=dtype)
  bias = (state["values"], state["bucket"]) if case["bias"] else None
  if kind == "attention":
    return cache_hip.attention(state["q"], cache, table, state["position"],
                               relative_bias=bias)
  out = cache_hip.attention(state["q"], cache, table, state["position"],
                            k_new=state["k"][:, 0], v_new=state["v"][:, 0],
                            relative_bias=bias)
  k, v = cache_hip.read(cache, table, state["position"], 1, dtype=dtype)
  return out, k[:, 0], v[:, 0]


def run(state):
  return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the program around the pass
# ---------------------------------------------------------------------------
def _normal(gen, sizes, std=1.0):
  return torch.randn(sizes, generator=gen, device="cuda") * std


def _projected(gen, sizes):
  """Keys or values as projections leave them: some of a head's values are much larger
  than the others, and tokens differ in size."""
  channels = torch.exp(_normal(gen, sizes[-1:], 0.5))
  tokens = torch.exp(_normal(gen, sizes[:-1] + (1,), 0.3))
  return _normal(gen, sizes) * channels * tokens


def _buckets(n):
  """Bucket of the distances 1 - n .. n - 1 of memory to query: half of them hold one
  distance each, the others grow with its logarithm; what lies ahead is in the first."""
  back = torch.arange(n - 1, -n, -1).clamp_min(0).double()
  exact_ones = BUCKETS // 2
  far = exact_ones + torch.floor(
      torch.log(back.clamp_min(1) / exact_ones) / math.log(DISTANCE / exact_ones)
      * (BUCKETS - exact_ones))
  return torch.where(back < exact_ones, back, far.clamp_max(BUCKETS - 1)).int().cuda()


def prepare(case, seed):
  """What the program has before the pass: the cache's pages, which lie in no order, the
  sequences' table of them, and the projections of the step or the prompts."""
  gen = torch.Generator(device="cuda").manual_seed(seed)
  cpu = torch.Generator().manual_seed(seed)
  dtype = DTYPES[case["dtype"]]
  b, heads, kv, width, page = (case[x] for x in (
      "batch", "heads", "kv_heads", "width", "page"))
  lengths = torch.tensor(_lengths(case))[torch.randperm(b, generator=cpu)]
  # (written rows follow others, in the middle of a page)
  start = (torch.randint(0, 2 * page, (b,), generator=cpu)
           if case["kind"] == "write" else torch.zeros(b, dtype=torch.long))
  used = (start + lengths + page - 1) // page
  columns = int(used.max())
  pages = int(used.sum()) + 3                          # (some are free)
  order = torch.randperm(pages, generator=cpu)
  table = torch.full((b, columns), -1, dtype=torch.int32)
  first = 0
  for i, n in enumerate(used.tolist()):
    table[i, :n] = order[first:first + n].int()
    first += n
  state = {"case": case, "table": table.cuda(), "start": start.int().cuda(),
           "count": lengths.int().cuda(), "rows": case["length"]}
  full = case["kind"] != "write"
  for name in "kv":
    shape = (pages, kv, page, width)
    stored = torch.zeros(shape, dtype=torch.uint8 if case["eight_bit"] else dtype,
                         device="cuda")
    scales = torch.full(shape[:-1] + (-(-width // BLOCK),), 127, dtype=torch.uint8,
                        device="cuda")
    many = max(1, (1 << 26) // (kv * page * width))
    for at in range(0, pages if full else 0, many):
      x = _projected(gen, (min(many, pages - at),) + shape[1:])
      if case["eight_bit"]:
        values, scales[at:at + many] = _to_eight_bits(x)
        stored[at:at + many] = values.view(torch.uint8)
      else:
        stored[at:at + many] = x.to(dtype)
    if case["eight_bit"]:
      state[name + "_pages"] = stored.view(torch.float8_e4m3fn)
      state[name + "_scales"] = scales
    else:
      state[name + "_pages"] = stored
  if case["kind"] == "write":
    for name in "kv":
      state[name] = _projected(gen, (b, case["length"], kv, width)).flatten(2).to(dtype)
  if case["kind"] in ("attention", "step"):
    # (the scaling by width ** -0.5 is part of the query projection)
    state["q"] = (_normal(gen, (b, heads, width), 2 * width ** -0.5)
                  .flatten(1).to(dtype))
    state["position"] = state["count"] - 1
  if case["kind"] == "step":
    for name in "kv":
      state[name] = _projected(gen, (b, 1, kv, width)).flatten(2).to(dtype)
    state.update(start=state["position"], rows=1, count=torch.ones_like(state["count"]))
  if case["bias"]:
    state["reach"] = 2 * DISTANCE
    state["values"] = _normal(gen, (heads, BUCKETS)).to(dtype)
    state["bucket"] = _buckets(state["reach"])
  return state


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _eight_bit_64(x):
  """float64 [..., width] -> what its 8-bit form stands for.  Normal numbers of e4m3
  have three bits behind the first, the steps below 2^-6 are 2^-9."""
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
    size = torch.clamp(q.abs(), min=2.0 ** -6)
    binade = torch.floor(torch.log2(size))
    binade = torch.where(torch.exp2(binade) > size, binade - 1, binade)
    binade = torch.where(torch.exp2(binade + 1) <= size, binade + 1, binade)
    step = torch.exp2(binade - 3)
    out[..., at:at + BLOCK] = torch.round(q / step) * step * unit
  return out


def _sequence_64(state, name, i, n):
  """float64 [n, kv_heads, width]: the first n positions of sequence i."""
  case = state["case"]
  pages = state["table"][i, :-(-n // case["page"])].long()
  if case["eight_bit"]:
    x = state[name + "_pages"].view(torch.uint8)[pages].view(torch.float8_e4m3fn)
    scales = state[name + "_scales"][pages].double()
    x = x.float().double()
    for block in range(scales.shape[-1]):
      x[..., block * BLOCK:(block + 1) * BLOCK] *= torch.exp2(
          scales[..., block:block + 1] - 127)
  else:
    x = state[name + "_pages"][pages].double()
  return x.transpose(1, 2).flatten(0, 1)[:n]


def exact(case, seed):
  state = prepare(case, seed)
  b, kv, width = case["batch"], case["kv_heads"], case["width"]
  written = {}
  if case["kind"] in ("write", "step"):
    for name in "kv":
      x = state[name].double().reshape(b, -1, kv, width)
      written[name] = _eight_bit_64(x) if case["eight_bit"] else x
  if case["kind"] == "write":
    there = torch.arange(case["length"], device="cuda") < state["count"][:, None]
    return tuple(written[name].flatten(2) * there[..., None] for name in "kv")
  lengths = state["count"] if case["kind"] == "read" else state["position"] + 1
  lengths = lengths.tolist()
  if case["kind"] == "read":
    out = []
    for name in "kv":
      dense = torch.zeros((b, case["length"], kv * width), dtype=torch.float64,
                          device="cuda")
      for i, n in enumerate(lengths):
        dense[i, :n] = _sequence_64(state, name, i, n).flatten(1)
      out.append(dense)
    return tuple(out)
  outs = []
  for i, n in enumerate(lengths):
    k, v = (_sequence_64(state, name, i, n) for name in "kv")
    if case["kind"] == "step":
      k[n - 1], v[n - 1] = written["k"][i, 0], written["v"][i, 0]
    q = state["q"][i].double().reshape(kv, -1, width)
    logits = torch.bmm(q, k.permute(1, 2, 0).contiguous())
    if case["bias"]:
      back = torch.arange(n - 1, -1, -1, device="cuda").clamp(max=state["reach"] - 1)
      bucket = state["bucket"].long()[state["reach"] - 1 - back]
      logits = logits + state["values"].double()[:, bucket].reshape(kv, -1, n)
    weights = torch.softmax(logits, -1)
    outs.append(torch.bmm(weights, v.transpose(0, 1).contiguous()).flatten())
  out = torch.stack(outs)
  if case["kind"] == "attention":
    return out
  return (out,) + tuple(written[name][:, 0].flatten(1) for name in "kv")
