"""The paged cache in float64 on the CPU (test infrastructure): what pages hold, position
by position, attention over them by its definition, and how far float32 arithmetic and
roundings can take a result from it."""

import numpy as np
import torch

from tests import fp8_reference as F

BLOCK = 128


def stored(x, eight_bit):
  """What rows x [..., width] (already of the activations' type) are kept as."""
  if not eight_bit:
    return x
  flat = x.reshape(-1, x.shape[-1])
  codes, scales = F.quantize(flat)
  return F.value(codes, scales)[:, :x.shape[-1]].reshape(x.shape)


def values_of(pages, scales):
  """float64 [pages, heads, page, width] of a cache's buffer (any device)."""
  if scales is None:
    return pages.double().cpu().numpy()
  codes = pages.view(torch.uint8).cpu().numpy()
  width = codes.shape[-1]
  padded = np.zeros(codes.shape[:-1] + (-(-width // BLOCK) * BLOCK,), np.uint8)
  padded[..., :width] = codes
  return F.value(padded, scales.cpu().numpy())[..., :width]


def page_at(table, pages, page, b, p):
  """(page, row) of position p of sequence b, or None."""
  if p < 0 or p // page >= table.shape[1]:
    return None
  n = int(table[b, p // page])
  return (n, p % page) if 0 <= n < pages else None


def write(held, rows, table, position, count, page):
  """held [pages, heads, page, width] with rows [B, T, heads, width] written."""
  held = held.copy()
  for b in range(rows.shape[0]):
    for t in range(rows.shape[1] if count is None else min(rows.shape[1], count[b])):
      at = page_at(table, held.shape[0], page, b, int(position[b]) + t)
      if at is not None:
        held[at[0], :, at[1]] = rows[b, t]
  return held


def read(held, table, position, length, count, page):
  """[B, length, heads, width], zeros where nothing is."""
  b = table.shape[0]
  out = np.zeros((b, length, held.shape[1], held.shape[3]))
  for i in range(b):
    for t in range(length if count is None else min(length, count[i])):
      at = page_at(table, held.shape[0], page, i, int(position[i]) + t)
      if at is not None:
        out[i, t] = held[at[0], :, at[1]]
  return out


def attention(q, k, v, table, position, page, eps, values=None, bucket=None):
  """q [B, heads, width] over pages k, v [pages, kv heads, page, width] -> (out [B, heads,
  width], how far a result may be off).  eps: the half step of the results' type (2^-8 for
  bfloat16, whose weights are rounded too, 2^-24 for float32).

  The bound, with u = 2^-24 and, over the positions that are seen, S the largest sum of
  |q k|, R the logits' largest magnitude, n their number and A = sum w |v|: a logit's
  products and additions are off by (width + 1) u S, the bias's addition by u R, the
  difference to the maximum and its exponential by 4 u R + 8 u, relatively to the weight;
  the weight's own rounding by eps, the sums by n u.  Numerator and denominator both take
  that, and the result is rounded once."""
  b, heads, width = q.shape
  group = heads // k.shape[1]
  out, bound = np.zeros(q.shape), np.zeros(q.shape)
  u = 2.0 ** -24
  for i in range(b):
    last = int(position[i])
    at = [(p, page_at(table, k.shape[0], page, i, p)) for p in range(
        min(last + 1, table.shape[1] * page))]
    at = [(p, a) for p, a in at if a is not None]
    if not at:
      continue
    pages, rows = (np.array([a[x] for _, a in at]) for x in (0, 1))
    for h in range(heads):
      keys, vals = k[pages, h // group, rows], v[pages, h // group, rows]
      logits = keys @ q[i, h]
      if values is not None:
        reach = (len(bucket) + 1) // 2
        back = np.maximum([p - last for p, _ in at], 1 - reach)
        logits = logits + values[h][bucket[back + reach - 1]]
      if (logits == -np.inf).all():
        continue
      w = np.exp(logits - logits.max())
      w /= w.sum()
      out[i, h] = w @ vals
      finite = np.abs(logits[np.isfinite(logits)])
      s = (np.abs(keys) @ np.abs(q[i, h])).max()
      off = u * ((width + 1) * s + 5 * finite.max() * 2 + 8 + len(at))
      if eps > u:
        off += eps
      bound[i, h] = eps * np.abs(out[i, h]) + 2 * off * (1 + 2 * off) * (w @ np.abs(vals))
  return out, bound + 1e-37
