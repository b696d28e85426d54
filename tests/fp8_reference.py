"""What 8-bit operands stand for, in float64 on the CPU (test infrastructure): e4m3 by its
definition, an exponent per block of 128 by search."""

import numpy as np
import torch

BLOCK = 128


def e4m3_table():
  """The 256 numbers of e4m3, NaN at 0x7f and 0xff."""
  out = np.zeros(256)
  for i in range(256):
    exponent, mantissa = (i >> 3) & 15, i & 7
    value = (mantissa / 8.0 * 2.0 ** -6 if exponent == 0
             else (1 + mantissa / 8.0) * 2.0 ** (exponent - 7))
    out[i] = -value if i & 128 else value
  out[0x7f] = out[0xff] = np.nan
  return out


_POSITIVE = e4m3_table()[:0x7f]


def _codes(x):
  """Magnitudes up to 448 -> the codes of the nearest numbers, ties to the even code."""
  above = np.searchsorted(_POSITIVE, x)            # first number >= x
  above = np.minimum(above, 0x7e)
  below = np.maximum(above - 1, 0)
  up, down = _POSITIVE[above] - x, x - _POSITIVE[below]
  return np.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)


def quantize(x):
  """float64 [rows, n] -> codes [rows, padded n] uint8, scale bytes [rows, blocks]."""
  x = np.asarray(x, np.float64)
  rows, n = x.shape
  blocks = (n + BLOCK - 1) // BLOCK
  full = np.zeros((rows, blocks * BLOCK))
  full[:, :n] = x
  full = full.reshape(rows, blocks, BLOCK)
  with np.errstate(invalid="ignore"):
    top = np.abs(full).max(-1)
  bad = ~np.isfinite(top)
  exponent = np.full(top.shape, -117)
  for e in range(-117, 121):      # the smallest that is enough
    exponent = np.where(np.where(bad, 0, top) > 448 * 2.0 ** e, e + 1, exponent)
  exponent = np.where(bad, 0, exponent)
  unit = 2.0 ** exponent[..., None]
  clean = np.where(bad[..., None], 0, full)
  codes = _codes(np.abs(clean) / unit) | np.where(np.signbit(clean), 128, 0)
  codes = np.where(bad[..., None], 0x7f, codes)
  return (codes.reshape(rows, blocks * BLOCK).astype(np.uint8),
          (exponent + 127).astype(np.uint8))


def value(codes, scales):
  """What codes [..., padded n] with scale bytes [..., >= blocks] stand for."""
  table = e4m3_table()
  v = table[codes]
  unit = 2.0 ** (scales[..., :v.shape[-1] // BLOCK].astype(np.int64) - 127)
  return v * np.repeat(unit, BLOCK, axis=-1)


def operand_value(q):
  """float64 array of what an Fp8Blocks stands for."""
  codes = q.values.view(torch.uint8).cpu().numpy()
  return value(codes, q.scales.cpu().numpy())[..., :q.n]


def random_operand(rng, shape, std, device="cuda"):
  """An Fp8Blocks of normal numbers, quantized here."""
  from mesh_amd import fp8_hip
  x = rng.standard_normal(shape) * std
  x *= np.exp(0.5 * rng.standard_normal(shape[-1:]))
  codes, scales = quantize(x.reshape(-1, shape[-1]))
  ks = fp8_hip.scale_bytes(shape[-1])
  # (bytes of blocks that a row does not have may hold anything)
  padded = rng.integers(0, 256, (codes.shape[0], ks)).astype(np.uint8)
  padded[:, :scales.shape[1]] = scales
  lead = tuple(shape[:-1])
  return fp8_hip.Fp8Blocks(
      torch.from_numpy(codes.reshape(lead + (-1,))).view(torch.float8_e4m3fn).to(device),
      torch.from_numpy(padded.reshape(lead + (-1,))).to(device), shape[-1])
