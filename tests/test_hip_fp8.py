"""The 8-bit operators on the GPU against float64 (tests/fp8_reference.py).

Tolerances.  Operands: the exponent is settled by comparisons and values are rounded to
nearest, so that both are equal bit for bit.  Results that become operands: half a step of
e4m3 (2^-4 relative, or 2^-10 of the block's unit below its normal numbers), the unit
being the smallest that holds the block's largest value up to float32 rounding.  bfloat16
results: half a step (2^-8) plus what the matrix instructions drop.  They keep the sum of
a group of 8 products to 2^-14 of the largest one at least, so at most 8 * 2^-14 of the
sum of the products' magnitudes over 8, 2^-14 of it on the whole; 2^-13 with the float32
additions behind."""

import numpy as np
import pytest
import torch

from tests import fp8_reference as F

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


@pytest.fixture(scope="module")
def hip():
  from mesh_amd import fp8_hip
  fp8_hip.load_library()
  return fp8_hip


def _f64(t):
  return t.detach().double().cpu().numpy()


def _tensor(rng, shape, dtype, spread=2.0):
  x = rng.standard_normal(shape) * np.exp(spread * rng.standard_normal(shape[-1:]))
  return torch.from_numpy(x.astype(np.float32)).to(TYPES[dtype]).cuda()


def _assert_operand(q, want):
  """q holds the codes and scale bytes of the 8-bit form of `want` [..., n]."""
  n = want.shape[-1]
  codes, scales = F.quantize(want.reshape(-1, n))
  got = q.values.view(torch.uint8).cpu().numpy().reshape(codes.shape)
  got_scales = q.scales.cpu().numpy().reshape(codes.shape[0], -1)
  np.testing.assert_array_equal(got_scales[:, :scales.shape[1]], scales)
  # (either NaN is one)
  np.testing.assert_array_equal(np.where(got == 0xff, 0x7f, got), codes)


def _assert_rounded(q, want, slack=2.0 ** -18):
  """q stands for `want` up to a rounding to e4m3."""
  n = want.shape[-1]
  want = want.reshape(-1, n)
  got = F.operand_value(q).reshape(-1, n)
  blocks = (n + 127) // 128
  scales = q.scales.cpu().numpy().reshape(want.shape[0], -1)[:, :blocks]
  unit = 2.0 ** (scales.astype(np.float64) - 127)
  full = np.zeros((want.shape[0], blocks * 128))
  full[:, :n] = np.abs(want)
  top = full.reshape(-1, blocks, 128).max(-1)
  assert (top <= 448 * unit * (1 + slack)).all()
  smaller = (unit > 2.0 ** -117) & (top <= 224 * unit * (1 - slack))
  assert not smaller.any()
  unit = np.repeat(unit, 128, axis=-1)[:, :n]
  step = np.maximum(np.abs(want) * 2.0 ** -4, unit * 2.0 ** -10)
  assert (np.abs(got - want) <= step * (1 + 2.0 ** -8) + np.abs(want) * slack).all()
  codes = q.values.view(torch.uint8).cpu().numpy().reshape(want.shape[0], -1)
  assert (codes[:, n:] == 0).all()


def _assert_product(got, want, magnitudes):
  error = np.abs(_f64(got) - want)
  assert (error <= np.abs(want) * 2.0 ** -8 + magnitudes * 2.0 ** -13).all()


# --- operands ---------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 1, 128), (1, 128, 1), (2, 129, 127), (3, 5, 1000),
          (1, 300, 264), (2, 64, 513), (1, 700, 1032), (5, 130, 8)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", SHAPES)
def test_quantize(hip, shape, dtype):
  rng = np.random.default_rng(sum(shape))
  x = _tensor(rng, shape, dtype)
  rows, columns = hip.quantize(x, rows=True, columns=True)
  _assert_operand(rows, _f64(x))
  _assert_operand(columns, _f64(x).transpose(0, 2, 1))
  only = hip.quantize(x)
  assert torch.equal(only.values.view(torch.uint8), rows.values.view(torch.uint8))
  only = hip.quantize(x, rows=False, columns=True)
  assert torch.equal(only.values.view(torch.uint8), columns.values.view(torch.uint8))
  flat = hip.quantize(x[0], rows=False, columns=True)
  assert flat.shape == (shape[2], shape[1])
  assert torch.equal(flat.values.view(torch.uint8),
                     columns.values[0].view(torch.uint8))


def test_quantize_into_given_operands(hip):
  rng = np.random.default_rng(4)
  x = _tensor(rng, (2, 70, 300), "bf16")
  want = hip.quantize(x, rows=True, columns=True)
  out = hip.Fp8Blocks.empty((2, 70, 300), "cuda"), hip.Fp8Blocks.empty((2, 300, 70), "cuda")
  for rows, columns, given in ((True, True, out), (True, False, out[0]),
                               (False, True, out[1])):
    for q in out:
      q.values.view(torch.uint8).fill_(0x55)
    got = hip.quantize(x, rows, columns, out=given)
    for g, o, w in zip(got if rows and columns else (got,),
                       out if rows and columns else (given,),
                       want if rows and columns else want[:1] if rows else want[1:]):
      assert g is o
      assert torch.equal(hip.dequantize(g, torch.float32), hip.dequantize(w, torch.float32))
  for rows, columns, given in ((True, False, out[1]), (False, True, out[0]),
                               (True, True, out[::-1])):
    with pytest.raises(hip.MoeHipError, match="shape"):
      hip.quantize(x, rows, columns, out=given)


def test_quantize_of_many_tiles(hip):
  """Blocks of the grid in the order that keeps an XCD's tiles together."""
  rng = np.random.default_rng(0)
  x = _tensor(rng, (1, 2055, 5000), "bf16")
  rows, columns = hip.quantize(x, rows=True, columns=True)
  _assert_operand(rows, _f64(x))
  _assert_operand(columns, _f64(x).transpose(0, 2, 1))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_of_borders(hip, dtype):
  """Ties, values next to a unit's limit, zeros, the smallest and the largest numbers,
  infinities and NaN."""
  x = np.zeros((40, 128), np.float32)
  for i in range(20):
    x[i] = np.linspace(-17, 17, 128) * 2.0 ** (7 * i - 70)
    x[i, 0] = [448, 449, 447, 450, 452, 224, 225, 1, 1.75, 1.7578125][i % 10] * 2.0 ** (
        7 * i - 70)
  x[20, 5] = 1e-45
  x[21] = np.float32(2.0 ** -126) * np.linspace(-1, 1, 128)
  x[22] = np.float32(3.3e38) * np.linspace(-1, 1, 128)
  x[23, 1], x[24, 2], x[25, 3] = np.inf, -np.inf, np.nan
  x[26, 1:3] = 448, 0.5 * 2.0 ** -9          # a tie with zero
  x[27, 1:4] = 448, 1.5 * 2.0 ** -9, 2.5 * 2.0 ** -9
  x[28] = -0.0
  x[29, :2] = 2.0 ** -109 * 1.75, 2.0 ** -126
  x[30, :2] = 2.0 ** -120, 2.0 ** -127
  t = torch.from_numpy(x).to(TYPES[dtype]).cuda()
  for rows, want in ((hip.quantize(t), _f64(t)),
                     (hip.quantize(t.t().contiguous(), rows=False, columns=True),
                      _f64(t))):
    _assert_operand(rows, want)
    for to in (torch.bfloat16, torch.float32):
      # (numbers from 248 * 2^120 on round to 2^128, which neither type has: there the
      # 8-bit value is read as an infinity)
      want = F.operand_value(rows)
      want = np.where(np.abs(want) == 2.0 ** 128, np.copysign(np.inf, want), want)
      np.testing.assert_array_equal(_f64(hip.dequantize(rows, to)), want)


@pytest.mark.parametrize("shape", [(3, 140, 200), (2, 70, 131)])
def test_quantize_masks_and_counts(hip, shape):
  """What is masked or behind the count does not reach the operands, whatever it is."""
  rng = np.random.default_rng(7)
  x = _tensor(rng, shape, "bf16")
  mask = torch.from_numpy(np.maximum(rng.standard_normal(shape), 0)).to(x).contiguous()
  mask[0, 3, 5], mask[1, 2, 2], mask[0, 0, 0] = float("nan"), -1, -float("inf")
  x = torch.where(mask > 0, x, torch.full_like(x, float("inf")))
  count = torch.tensor([0, shape[1] + 9, 129][:shape[0]], dtype=torch.int32).cuda()
  x[2:, 129:] = float("nan")
  want = np.where(_f64(mask) > 0, _f64(x), 0)
  for e, c in enumerate(count.tolist()):
    want[e, c:] = 0
  rows, columns = hip.quantize(x, rows=True, columns=True, relu_mask=mask,
                               row_count=count)
  _assert_operand(rows, want)
  _assert_operand(columns, want.transpose(0, 2, 1))


@pytest.mark.parametrize("shape", [(1, 1), (7, 130), (300, 1024), (2, 3, 77)])
def test_dequantize(hip, shape):
  q = F.random_operand(np.random.default_rng(1), shape, 3.0)
  for dtype in (torch.bfloat16, torch.float32):
    y = hip.dequantize(q, dtype)
    assert y.dtype == dtype and tuple(y.shape) == shape
    np.testing.assert_array_equal(_f64(y), F.operand_value(q))


def test_dequantize_every_scale_byte(hip):
  """Every code under every scale byte, 255 being NaN; numbers that are not normal are
  kept, in bfloat16 to its last bit, 2^-133."""
  codes = torch.arange(256, dtype=torch.uint8).repeat(256, 1)
  scales = torch.arange(256, dtype=torch.uint8)[:, None].repeat(1, 4)
  q = hip.Fp8Blocks(codes.view(torch.float8_e4m3fn).cuda(), scales.cuda(), 256)
  want = F.value(codes.numpy(), scales.numpy())
  want[255] = np.nan
  want = np.where(np.abs(want) >= 2.0 ** 128, np.copysign(np.inf, want), want)
  np.testing.assert_array_equal(_f64(hip.dequantize(q, torch.float32)), want)
  with np.errstate(invalid="ignore"):
    rounded = np.where(np.abs(want) < 2.0 ** -126,
                       np.round(want * 2.0 ** 133) * 2.0 ** -133, want)
  assert (rounded[3:255] == want[3:255])[~np.isnan(want[3:255])].all()
  np.testing.assert_array_equal(_f64(hip.dequantize(q)), rounded)


# --- the norm ---------------------------------------------------------------
def _norm_64(total, scale, mask, epsilon):
  t = _f64(total)
  y = t / np.sqrt((t * t).mean(-1, keepdims=True) + epsilon) * _f64(scale)
  return y if mask is None else np.where(_f64(mask)[..., None] != 0, y, 0) * np.where(
      _f64(mask) != 0, _f64(mask), 0)[..., None]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,m", [(1, 1), (5, 100), (3, 128), (33, 1024), (2, 1025),
                                    (7, 2048), (3, 4096), (4, 4099), (2, 8192),
                                    (3, 9000), (1, 16385), (2, 20000)])
def test_residual_rms_norm(hip, rows, m, dtype):
  rng = np.random.default_rng(m + rows)
  x, residual = (_tensor(rng, (rows, m), dtype, 1.0) for _ in range(2))
  scale = (1 + 0.2 * torch.randn(m, generator=torch.Generator().manual_seed(m))).to(
      x).contiguous()
  mask = torch.tensor([1.0, 0.0, 0.5, 1.0])[torch.arange(rows) % 4].to(x)
  want_sum = (x.float() + residual.float()).to(x.dtype)
  total, y, norm = hip.residual_rms_norm(x, residual, scale, want_norm=True)
  assert torch.equal(total, want_sum)
  want = _norm_64(total, scale, None, 1e-6)
  _assert_rounded(y, want)
  eps = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -19
  assert (np.abs(_f64(norm) - want) <= eps * np.abs(want) * (1 + 2.0 ** -8)).all()
  total, y = hip.residual_rms_norm(x, residual, scale, 1e-3, row_mask=mask)
  assert torch.equal(total, want_sum)
  _assert_rounded(y, _norm_64(total, scale, mask, 1e-3))
  total, y = hip.residual_rms_norm(x, None, scale)
  assert total is x
  _assert_rounded(y, _norm_64(x, scale, None, 1e-6))


def test_residual_rms_norm_of_odd_rows(hip):
  """Zeros, rows that are masked out with an infinity in them, rows with one, more
  leading dimensions, operands that do not start on 16 bytes."""
  rng = np.random.default_rng(0)
  x = _tensor(rng, (2, 3, 640), "bf16", 1.0)
  x[0, 0] = 0
  x[0, 1, 7], x[1, 0, 600] = float("inf"), float("nan")
  scale = torch.ones(640, dtype=torch.bfloat16, device="cuda")
  mask = torch.ones(2, 3, dtype=torch.bfloat16, device="cuda")
  mask[0, 1] = 0
  total, y = hip.residual_rms_norm(x, torch.zeros_like(x), scale, row_mask=mask)
  got = F.operand_value(y)
  assert y.shape == (2, 3, 640) and total.shape == (2, 3, 640)
  assert (got[0, :2] == 0).all() and np.isnan(got[1, 0]).all()
  for at in ((0, 2), (1, 1), (1, 2)):
    assert np.isfinite(got[at]).all() and np.abs(got[at]).max() > 0.5
  flat = _tensor(rng, (5 * 640 + 3,), "bf16", 1.0)
  odd = flat[3:].view(5, 640)
  assert odd.data_ptr() % 16
  total, y = hip.residual_rms_norm(odd, odd, scale)
  again = hip.residual_rms_norm(odd.clone(), odd.clone(), scale)
  assert torch.equal(total, again[0])
  assert torch.equal(y.values.view(torch.uint8), again[1].values.view(torch.uint8))


@pytest.mark.parametrize("rows,m", [(67108860 + 7, 1), (16777215 + 5, 2049)])
def test_residual_rms_norm_of_more_rows_than_a_launch_has(hip, rows, m):
  """Rows around the first launch's end are what the call makes of those alone."""
  at = torch.arange(rows, device="cuda")
  mask = (at % 5 != 0).bfloat16()
  x = ((at % 7).bfloat16() + 1)[:, None].expand(rows, m).contiguous()
  del at
  residual = -0.5 * x if m == 1 else None
  scale = torch.linspace(0.5, 2, m, device="cuda").bfloat16()
  total, y, *norm = hip.residual_rms_norm(x, residual, scale, row_mask=mask,
                                          want_norm=m == 1)
  edge = rows - (7 if m == 1 else 5)
  for sl in (slice(0, 9), slice(edge - 9, edge + 1), slice(edge, rows)):
    part = (x[sl].contiguous(), None if residual is None else residual[sl].contiguous())
    t, q, *n = hip.residual_rms_norm(*part, scale, row_mask=mask[sl].contiguous(),
                                     want_norm=m == 1)
    assert torch.equal(total[sl], t)
    assert torch.equal(y.values[sl].view(torch.uint8), q.values.view(torch.uint8))
    assert torch.equal(y.scales[sl], q.scales)
    for whole, alone in zip(norm, n):
      assert torch.equal(whole[sl], alone)
  del x, y, total, residual, norm
  torch.cuda.empty_cache()                     # (up to 105 GB)


def test_residual_rms_norm_of_the_widest_row(hip):
  """A row whose last step's columns reach 2^31: what lies behind it is not read.  Every
  sum is 1 and the norm of ones is one, whose code is 256 under the unit 2^-8."""
  m = 0x7ffffefd
  x, residual = (torch.full((m + 300,), 0.5, dtype=torch.bfloat16, device="cuda")
                 for _ in range(2))
  x[m:], residual[m:] = float("nan"), float("nan")
  scale = torch.ones(m, dtype=torch.bfloat16, device="cuda")
  total, y = hip.residual_rms_norm(x[:m].view(1, m), residual[:m].view(1, m), scale, 0.0)
  assert (total == 1).all()
  del x, residual, scale, total
  codes = y.values.view(torch.uint8)[0]
  assert (codes[:m] == 0x78).all() and (codes[m:] == 0).all()
  assert (y.scales[0, :hip.row_bytes(m) // 128] == 127 - 8).all()


# --- products ---------------------------------------------------------------
def _act(y, activation):
  if activation == "relu":
    return np.maximum(y, 0)
  if activation == "gelu":
    return y * 0.5 * (1 + np.tanh(0.7978845608028654 * (y + 0.044715 * y ** 3)))
  if activation == "sigmoid":
    return 1 / (1 + np.exp(-y))
  if activation == "swish":
    return y / (1 + np.exp(-y))
  return np.tanh(y) if activation == "tanh" else y


# rows from one to several tiles, reductions of one block and of many, odd columns
PRODUCTS = [(1, 1, 1, 1), (1, 1, 128, 32), (1, 1, 4096, 1000), (1, 3, 300, 17),
            (2, 33, 130, 129), (1, 64, 1024, 256), (5, 40, 256, 64), (1, 65, 640, 385),
            (1, 129, 2000, 130), (3, 200, 384, 300), (1, 257, 512, 513),
            (2, 300, 1100, 256), (1, 1000, 256, 1024), (4, 520, 896, 640),
            (1, 2050, 384, 1537), (1, 512, 4224, 512), (64, 6, 512, 256),
            (1, 8, 1024, 4096), (1, 1100, 128, 8), (1, 384, 129, 4000),
            (1, 700, 128, 520), (3, 400, 65, 1000)]


@pytest.mark.parametrize("e,r,k,n", PRODUCTS)
def test_expert_linear(hip, e, r, k, n):
  rng = np.random.default_rng(e + r + k + n)
  a = F.random_operand(rng, (e, r, k), 1.0)
  w = F.random_operand(rng, (e, n, k), k ** -0.5)
  av, wv = F.operand_value(a), F.operand_value(w).transpose(0, 2, 1)
  want, magnitudes = av @ wv, np.abs(av) @ np.abs(wv)
  _assert_product(hip.expert_linear(a, w), want, magnitudes)
  for activation in ("relu", "gelu"):
    # (their slopes are at most 1.13)
    _assert_product(hip.expert_linear(a, w, activation), _act(want, activation),
                    1.13 * magnitudes)
  q = hip.expert_linear(a, w, "relu", eight_bit=True)
  y = hip.dequantize(hip.quantize(torch.from_numpy(
      np.maximum(want, 0)).float().cuda()), torch.float32)
  # the 8-bit result against the 8-bit form of the exact one: the same but where the
  # sums' error crosses a rounding border, there a step apart
  got, ref = F.operand_value(q), _f64(y)
  assert np.abs(got - np.maximum(want, 0)).max() <= (
      2.0 ** -4 * np.abs(want).max() + 2.0 ** -13 * magnitudes.max())
  assert (got == ref).mean() > 0.98
  codes = q.values.view(torch.uint8).cpu().numpy()
  assert (codes[..., n:] == 0).all()


# sizes that fill the GPU with tiles of each kind, some more than once, with rows that
# are and are not whole pieces of 16 bytes, and ones that split the reduction
MANY = [(16, 1100, 300, 1030), (8, 2000, 400, 1032), (40, 300, 384, 520),
        (64, 200, 256, 1000), (16, 300, 256, 1030), (32, 260, 256, 1032),
        (4, 500, 3100, 300), (1, 200, 2300, 640), (1, 1000, 8192, 520),
        (1, 40, 4096, 300), (32, 24, 1024, 1030), (1, 24, 11080, 1500),
        (16, 1100, 128, 1030), (16, 300, 100, 1032), (64, 60, 77, 520),
        (16, 1100, 4200, 1030), (8, 1100, 8192, 2056), (8, 1100, 8200, 1030),
        (16, 600, 8300, 1032)]


def _random(hip, shape, std, seed):
  """A random operand and its value in float64, on the GPU."""
  gen = torch.Generator(device="cuda").manual_seed(seed)
  x = torch.randn(shape, generator=gen, device="cuda") * std
  q = hip.quantize(x * torch.exp(0.5 * torch.randn(shape[-1:], generator=gen,
                                                   device="cuda")))
  return q, hip.dequantize(q, torch.float32).double()


def _near(got, want, magnitudes):
  return ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 +
          magnitudes * 2.0 ** -13).all()


@pytest.mark.parametrize("e,r,k,n", MANY)
def test_expert_linear_of_many_tiles(hip, e, r, k, n):
  a, av = _random(hip, (e, r, k), 1.0, 1)
  w, wv = _random(hip, (e, n, k), k ** -0.5, 2)
  wt = wv.transpose(1, 2).contiguous()
  want, magnitudes = av @ wt, av.abs() @ wt.abs()
  assert _near(hip.expert_linear(a, w), want, magnitudes)
  act = torch.nn.functional.gelu(want, approximate="tanh")
  assert _near(hip.expert_linear(a, w, "gelu"), act, 1.13 * magnitudes)
  count = torch.randint(0, r + 1, (e,), dtype=torch.int32, device="cuda")
  count[0], count[e // 2] = r // 2 + 1, 0 if e > 1 else 1
  live = torch.arange(r, device="cuda") < count.unsqueeze(1)
  out = torch.full((e, r, n), 7.0, dtype=torch.bfloat16, device="cuda")
  hip.expert_linear(a, w, row_count=count, out=out)
  assert (out[~live] == 7).all() and _near(out[live], want[live], magnitudes[live])
  for activation, exact in (("relu", want.clamp_min(0)), ("gelu", act)):
    exact = hip.dequantize(hip.quantize(exact.float()), torch.float32)
    for counts in (None, count):
      q = hip.Fp8Blocks.empty((e, r, n), "cuda")
      q.values.view(torch.uint8).fill_(0x55)
      q.scales.fill_(99)
      hip.expert_linear(a, w, activation, True, row_count=counts, out=q)
      codes, got = q.values.view(torch.uint8), hip.dequantize(q, torch.float32)
      rows = torch.ones_like(live) if counts is None else live
      assert (codes[~rows] == 0x55).all() and (q.scales[~rows] == 99).all()
      assert (codes[rows][:, n:] == 0).all()
      # (a step apart where the sums' error crosses a rounding border, see above)
      assert (got[rows] == exact[rows]).double().mean() > 0.98
      assert (got[rows] - exact[rows]).abs().max() <= (
          2.0 ** -4 * exact.abs().max() + 2.0 ** -13 * 1.13 * magnitudes.max())


@pytest.mark.parametrize("e,r,k,n", [(40, 384, 300, 520), (16, 384, 300, 1030),
                                     (24, 900, 300, 1030), (6, 700, 1300, 256),
                                     (2, 1000, 520, 1024), (24, 100, 600, 1030),
                                     (8, 128, 300, 100), (16, 4400, 600, 1030),
                                     (8, 8200, 1100, 1030)])
def test_gradients_of_counted_rows(hip, e, r, k, n):
  """Experts with none, one, a block, a block and one, and all of their rows."""
  count = torch.tensor([(0, 1, 128, 129, r, r - 1, 257)[i % 7] for i in range(e)],
                       dtype=torch.int32, device="cuda")
  live = (torch.arange(r, device="cuda") < count.unsqueeze(1)).unsqueeze(2)
  gen = torch.Generator(device="cuda").manual_seed(3)
  dy = torch.randn((e, r, n), generator=gen, device="cuda").bfloat16()
  x = torch.randn((e, r, k), generator=gen, device="cuda") * live
  a_columns = hip.quantize(x, rows=False, columns=True)
  w_rows, wv = _random(hip, (e, k, n), 0.05, 4)
  da = torch.full((e, r, k), 3.0, dtype=torch.bfloat16, device="cuda")
  hip.expert_linear_backward(a_columns, dy, w_rows, row_count=count, da=da)
  _, dw = hip.expert_linear_backward(a_columns, dy, row_count=count)
  by_row, by_column = hip.quantize((dy * live).contiguous(), rows=True, columns=True)
  by_row, by_column, av = (hip.dequantize(q, torch.float32).double()
                           for q in (by_row, by_column, a_columns))
  wt, yt = wv.transpose(1, 2).contiguous(), by_column.transpose(1, 2).contiguous()
  want, magnitudes = by_row @ wt, by_row.abs() @ wt.abs()
  dead = ~live.squeeze(2)
  assert (da[dead] == 3).all() and _near(da[~dead], want[~dead], magnitudes[~dead])
  assert _near(dw, av @ yt, av.abs() @ yt.abs())


@pytest.mark.parametrize("e,r,k,n", [(1, 1, 4096, 1000), (1, 16, 1024, 4096),
                                     (2, 100, 700, 130), (30, 16, 100, 40),
                                     (3, 200, 384, 300), (8, 1100, 256, 520)])
def test_products_that_are_exact(hip, e, r, k, n):
  """Seven products of 2^-15 beside each of 1 or -1, which cancel out: the instructions
  for 8 bits lose them.  Where the call says that products are exact, so are these sums
  (multiples of 2^-15 below 2^9 in any order), and the result is the nearest bfloat16.
  Elsewhere seven products of eight lose 2^-13 of the largest at most, so sums less than
  2^-10 of their products' magnitudes."""
  x = torch.full((e, r, k), 2.0 ** -7, device="cuda")
  w = torch.full((e, n, k), 2.0 ** -8, device="cuda")
  x[..., ::16], x[..., 8::16], w[..., ::8] = 1.0, -1.0, 1.0
  x *= (torch.arange(r, device="cuda")[:, None] % 3 - 1.0)      # rows of -1, 0, 1 of it
  a, b = hip.quantize(x), hip.quantize(w)
  assert torch.equal(hip.dequantize(a, torch.float32), x)
  wt = w.double().transpose(1, 2).contiguous()
  want, magnitudes = x.double() @ wt, x.double().abs() @ wt
  for counts in (None, torch.full((e,), r, dtype=torch.int32, device="cuda")):
    exact = hip.multiplies_exactly(e, r, k, n, counted=counts is not None)
    assert exact == (r <= 100)
    got = hip.expert_linear(a, b, row_count=counts)
    if exact:
      assert torch.equal(got, want.to(torch.bfloat16))
    else:
      assert ((got.double() - want).abs() <= want.abs() * 2.0 ** -8 +
              magnitudes * 2.0 ** -10).all()


@pytest.mark.parametrize("activation", [None, "linear", "sigmoid", "tanh", "swish"])
@pytest.mark.parametrize("r", [2, 300])
def test_activations(hip, activation, r):
  rng = np.random.default_rng(3)
  a, w = F.random_operand(rng, (1, r, 256), 1.0), F.random_operand(rng, (1, 264, 256),
                                                                  0.06)
  av, wv = F.operand_value(a), F.operand_value(w).transpose(0, 2, 1)
  _assert_product(hip.expert_linear(a, w, activation), _act(av @ wv, activation),
                  1.13 * (np.abs(av) @ np.abs(wv)))


# of the few rows' kernel, of the one for one block, of 64-row tiles with and without a
# split reduction, of 128- and 256-row tiles
@pytest.mark.parametrize("e,r,k,n", [(30, 16, 256, 40), (480, 1, 64, 200),
                                     (1, 480, 256, 40), (1, 480, 4096, 200),
                                     (1, 480, 512, 16384), (8, 60, 512, 40000)])
@pytest.mark.parametrize("activation", ["relu", "gelu", "sigmoid", "tanh", "swish"])
def test_activations_of_all_magnitudes(hip, activation, e, r, k, n):
  """Sums from 2^-110 to 2^127, of either sign, and infinite ones: every row has one
  value, which every column takes as it is.  The sums are exact here; results are off by
  half a step, by 2^-13 from the exponential, and by 2^-118 where they are next to
  nothing."""
  p = np.arange(480) // 2 - 110
  codes, scales = np.zeros((480, hip.row_bytes(k)), np.uint8), np.full(
      (480, hip.scale_bytes(k)), 127, np.uint8)
  # 1.5 in e4m3 is 0x3c; units go up to 2^120
  codes[:, 0] = 0x3c + 8 * np.clip(p - 120, 0, 7) + 128 * (np.arange(480) % 2)
  codes[:, 1] = np.where(p > 127, codes[:, 0], 0)         # twice 1.5 * 2^127
  scales[:, 0] = np.minimum(p, 120) + 127
  v = F.value(codes, scales)[:, :2].sum(-1, keepdims=True)
  v = np.where(np.abs(v) < 2.0 ** 128, v, np.copysign(np.inf, v))
  assert np.isinf(v).sum() == 4
  a = hip.Fp8Blocks(
      torch.from_numpy(codes).view(torch.float8_e4m3fn).cuda().reshape(e, r, -1),
      torch.from_numpy(scales).cuda().reshape(e, r, -1), k)
  w = hip.Fp8Blocks.empty((e, n, k), "cuda")
  w.values.view(torch.uint8).zero_()
  w.values.view(torch.uint8)[..., :2] = 0x38              # 1.0
  w.scales.fill_(127)
  with np.errstate(all="ignore"):
    want = _act(v, activation)                            # [480, 1]
  ends = np.isfinite(want[:, 0])
  got = hip.expert_linear(a, w, activation).reshape(480, n)
  assert torch.equal(got.isnan(), got[:, :1].isnan().expand_as(got))
  assert torch.equal(got.nan_to_num(0.5), got[:, :1].nan_to_num(0.5).expand_as(got))
  got = _f64(got[:, :1])
  np.testing.assert_array_equal(got[~ends], want[~ends])
  assert (np.abs(got[ends] - want[ends]) <= np.abs(want[ends]) * (2.0 ** -8 + 2.0 ** -13) +
          2.0 ** -118).all()
  q = hip.expert_linear(a, w, activation, eight_bit=True).reshape(480)
  # (columns are alike: the first block, rows with an infinity being NaN)
  first = [t.view(torch.uint8)[:, :m] for t, m in ((q.values, 128), (q.scales, 4))]
  def rows(which):
    values, scales = (t[torch.from_numpy(which).cuda()] for t in first)
    return hip.Fp8Blocks(values.view(torch.float8_e4m3fn), scales, min(n, 128))
  assert np.isnan(F.operand_value(rows(~ends))).all()
  finite = rows(ends)
  _assert_rounded(finite, np.broadcast_to(want[ends], finite.shape), 2.0 ** -12)


@pytest.mark.parametrize("eight_bit", [False, True])
@pytest.mark.parametrize("r,n", [(6, 200), (70, 128), (300, 256), (600, 392)])
def test_row_counts(hip, r, n, eight_bit):
  """Rows behind an expert's count are left as they were; infinities in them go
  nowhere."""
  rng = np.random.default_rng(r)
  e, k = 5, 320
  a, w = F.random_operand(rng, (e, r, k), 1.0), F.random_operand(rng, (e, n, k), 0.05)
  count = [0, 1, r // 2 + 1, r, r + 100]
  for i, c in enumerate(count):
    a.values[i, c:].view(torch.uint8).fill_(0x7f)
  counts = torch.tensor(count, dtype=torch.int32, device="cuda")
  whole = hip.expert_linear(a, w, "relu", eight_bit)
  if eight_bit:
    out = hip.Fp8Blocks.empty((e, r, n), "cuda")
    out.values.view(torch.uint8).fill_(0x55)
    out.scales.fill_(99)
  else:
    out = torch.full((e, r, n), 7.0, dtype=torch.bfloat16, device="cuda")
  got = hip.expert_linear(a, w, "relu", eight_bit, row_count=counts, out=out)
  assert got is out
  for i, c in enumerate(count):
    if eight_bit:
      assert torch.equal(got.values[i, :c].view(torch.uint8),
                         whole.values[i, :c].view(torch.uint8))
      assert (got.values[i, c:].view(torch.uint8) == 0x55).all()
      assert (got.scales[i, c:] == 99).all()
    else:
      assert torch.equal(got[i, :c], whole[i, :c]) and (got[i, c:] == 7).all()
  counts.fill_(-3)
  hip.expert_linear(a, w, "relu", eight_bit, row_count=counts, out=out)
  assert ((got.values[0].view(torch.uint8) == 0x55) if eight_bit else got[0] == 7).all()


@pytest.mark.parametrize("r", [1, 40, 300])
def test_infinities_stay_in_their_rows(hip, r):
  """A block that is NaN makes its row of the result NaN, and no other one."""
  rng = np.random.default_rng(r)
  x = _tensor(rng, (1, r, 300), "bf16", 0.5)
  x[0, r // 2, 200] = float("inf")
  w = F.random_operand(rng, (1, 256, 300), 0.05)
  y = hip.expert_linear(hip.quantize(x), w)
  bad = torch.isnan(y[0]).all(-1)
  assert bad[r // 2] and bad.sum() == 1 and torch.isnan(y).sum() == 256
  q = hip.expert_linear(hip.quantize(x), w, eight_bit=True)
  assert np.isnan(F.operand_value(q)[0, r // 2]).all()
  assert np.isnan(F.operand_value(q)).sum() == 256


@pytest.mark.parametrize("r", [1, 40, 300])
def test_scale_byte_of_nan(hip, r):
  rng = np.random.default_rng(r)
  a = F.random_operand(rng, (1, r, 640), 1.0)
  w = F.random_operand(rng, (1, 200, 640), 0.05)
  want = hip.expert_linear(a, w)
  a.scales[0, r // 2, 4], w.scales[0, 77, 0] = 255, 255
  got = hip.expert_linear(a, w)
  nan = torch.zeros_like(got, dtype=torch.bool)
  nan[0, r // 2], nan[0, :, 77] = True, True
  assert got[nan].isnan().all() and torch.equal(got[~nan], want[~nan])


def test_scales_of_all_sizes(hip):
  """Every unit an operand can have, on both sides."""
  rng = np.random.default_rng(0)
  a, w = F.random_operand(rng, (1, 235, 512), 1.0), F.random_operand(rng, (1, 16, 512),
                                                                    1.0)
  a.scales[0, :, :] = torch.arange(10, 245, dtype=torch.uint8, device="cuda")[:, None]
  w.scales.fill_(120)
  w.scales[..., 1] = 130
  av, wv = F.operand_value(a), F.operand_value(w).transpose(0, 2, 1)
  want, magnitudes = (av @ wv)[0], (np.abs(av) @ np.abs(wv))[0]
  got = _f64(hip.expert_linear(a, w))[0]
  # (where neither the results nor their parts leave float32's normal numbers)
  inside = (magnitudes < 2.0 ** 126) & (np.arange(235)[:, None] > 25)
  error = np.abs(got - want)
  assert inside.any(-1).sum() > 180
  assert (error <= np.abs(want) * 2.0 ** -8 + magnitudes * 2.0 ** -13)[inside].all()


def test_dense(hip):
  rng = np.random.default_rng(5)
  x, w = F.random_operand(rng, (3, 5, 384), 1.0), F.random_operand(rng, (1, 250, 384),
                                                                  0.05)
  flat = hip.expert_linear(x.reshape(1, 15), w, "relu")
  y = hip.dense(x, w, "relu")
  assert tuple(y.shape) == (3, 5, 250) and torch.equal(y.view(1, 15, 250), flat)
  q = hip.dense(x, w, "relu", eight_bit=True)
  assert q.shape == (3, 5, 250)


def test_refusals(hip):
  rng = np.random.default_rng(5)
  a, w = F.random_operand(rng, (2, 4, 256), 1.0), F.random_operand(rng, (2, 8, 256), 1.0)
  Error = hip.MoeHipError
  other = F.random_operand(rng, (2, 8, 255), 1.0)
  bf16 = torch.zeros(2, 4, 8, dtype=torch.bfloat16, device="cuda")
  count = torch.zeros(2, dtype=torch.int32, device="cuda")
  strided = hip.Fp8Blocks(a.values.transpose(0, 1), a.scales.transpose(0, 1), 256)
  for call in (
      lambda: hip.expert_linear(a, other), lambda: hip.expert_linear(a, w.reshape(16)),
      lambda: hip.expert_linear(strided, w),
      lambda: hip.expert_linear(a, w, out=bf16.float()),
      lambda: hip.expert_linear(a, w, out=bf16[..., :7]),
      lambda: hip.expert_linear(a, w, eight_bit=True, out=bf16),
      lambda: hip.expert_linear(a, w, row_count=count.long()),
      lambda: hip.expert_linear(a, w, row_count=count[:1]),
      lambda: hip.dense(a, w),
      lambda: hip.quantize(bf16.transpose(1, 2)),
      lambda: hip.quantize(bf16, relu_mask=bf16.float()),
      lambda: hip.residual_rms_norm(bf16, None, torch.ones(8, device="cuda")),
      lambda: hip.residual_rms_norm(bf16, bf16[:1], bf16[0, 0]),
      lambda: hip.expert_linear_backward(a, bf16),
      lambda: hip.expert_linear_backward(w, bf16, da=bf16)):
    with pytest.raises(Error):
      call()
  with pytest.raises(ValueError):
    hip.expert_linear(a, w, "softplus")


def test_tensors_without_elements(hip):
  empty = torch.empty(0, 256, dtype=torch.bfloat16, device="cuda")
  q = hip.quantize(empty)
  assert q.shape == (0, 256) and hip.dequantize(q).shape == (0, 256)
  total, y = hip.residual_rms_norm(empty, empty, torch.ones_like(empty[:1].sum(0)))
  assert y.shape == (0, 256) and total.shape == (0, 256)
  w = F.random_operand(np.random.default_rng(0), (1, 8, 256), 1.0)
  assert hip.dense(q, w).shape == (0, 8)


# --- gradients --------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("e,r,k,n", [(1, 1, 8, 16), (2, 70, 200, 136), (1, 300, 256, 520),
                                     (3, 130, 129, 33), (1, 1385, 256, 512)])
def test_expert_linear_backward(hip, e, r, k, n, dtype):
  rng = np.random.default_rng(e + r + k + n)
  a_columns = F.random_operand(rng, (e, k, r), 1.0)
  w_rows = F.random_operand(rng, (e, k, n), 0.05)
  dy = _tensor(rng, (e, r, n), dtype, 0.5)
  mask = torch.from_numpy(np.maximum(rng.standard_normal((e, r, n)), 0)).to(dy)
  count = torch.tensor([r, r // 2, 0][:e], dtype=torch.int32, device="cuda")
  for masked in (False, True):
    kept = _f64(dy)
    if masked:
      kept = np.where(_f64(mask) > 0, kept, 0)
      for i, c in enumerate(count.tolist()):
        kept[i, c:] = 0
    by_row = F.value(*F.quantize(kept.reshape(-1, n)))[:, :n].reshape(e, r, n)
    turned = kept.transpose(0, 2, 1).reshape(-1, r)
    by_column = F.value(*F.quantize(turned))[:, :r].reshape(e, n, r)
    wv, av = F.operand_value(w_rows).transpose(0, 2, 1), F.operand_value(a_columns)
    da0 = torch.full((e, r, k), 3.0, dtype=torch.bfloat16, device="cuda")
    da, dw = hip.expert_linear_backward(
        a_columns, dy, w_rows, relu_mask=mask if masked else None,
        row_count=count if masked else None, da=da0 if masked else None)
    _assert_product(dw, av @ by_column.transpose(0, 2, 1),
                    np.abs(av) @ np.abs(by_column).transpose(0, 2, 1))
    want, magnitudes = by_row @ wv, np.abs(by_row) @ np.abs(wv)
    if masked:
      for i, c in enumerate(count.tolist()):
        want[i, c:], magnitudes[i, c:] = 3.0, 0
    _assert_product(da, want, magnitudes)
    none, dw2 = hip.expert_linear_backward(
        a_columns, dy, relu_mask=mask if masked else None,
        row_count=count if masked else None)
    assert none is None and torch.equal(dw, dw2)


def test_gradient_against_differences(hip):
  """The gradient of sum(y * g) in w and x against differences of the product itself,
  on numbers that e4m3 holds (all blocks have the unit 2^-2 or less, so that nothing is
  rounded before the sums)."""
  rng = np.random.default_rng(2)
  r, k, n = 130, 40, 24

  def small(*shape):       # multiples of 1/8 up to 1: e4m3 numbers
    return torch.from_numpy(rng.integers(-8, 9, shape) / 8.0).to(
        torch.bfloat16).cuda()
  x, w, g = small(1, r, k), small(1, k, n), small(1, r, n)

  def product(x, w):
    y = hip.expert_linear(hip.quantize(x), hip.quantize(w, rows=False, columns=True))
    return _f64(y)
  # y itself is rounded to bf16: its parts are multiples of 1/64 below 40, differences
  # of single elements are at most 2 * 1/8, and sums of those over a row need few bits
  _, a_columns = hip.quantize(x, rows=True, columns=True)
  dx, dw = hip.expert_linear_backward(a_columns, g, hip.quantize(w))
  gd, base = _f64(g), product(x * 0, w * 0)
  assert (base == 0).all()
  for _ in range(20):
    i, j, l = rng.integers(r), rng.integers(k), rng.integers(n)
    one = torch.zeros_like(x)
    one[0, i, j] = 1
    want = (product(one, w) * gd).sum()
    assert abs(_f64(dx)[0, i, j] - want) <= 2.0 ** -8 * abs(want) + 2.0 ** -13 * 40
    one = torch.zeros_like(w)
    one[0, j, l] = 1
    want = (product(x, one) * gd).sum()
    assert abs(_f64(dw)[0, j, l] - want) <= 2.0 ** -8 * abs(want) + 2.0 ** -13 * r


# --- together ---------------------------------------------------------------
def _mlp(hip, x, residual, scale, wi, wo):
  total, y = hip.residual_rms_norm(x, residual, scale)
  h = hip.dense(y, wi, "relu", eight_bit=True)
  return total, hip.dense(h, wo)


def _mlp_inputs(rng, rows, m, f):
  return (_tensor(rng, (rows, m), "bf16", 0.5), _tensor(rng, (rows, m), "bf16", 0.5),
          torch.ones(m, dtype=torch.bfloat16, device="cuda"),
          F.random_operand(rng, (1, f, m), m ** -0.5),
          F.random_operand(rng, (1, m, f), f ** -0.5))


@pytest.mark.parametrize("rows,m,f", [(1, 256, 1024), (40, 384, 1000), (700, 512, 2048)])
def test_dense_block(hip, rows, m, f):
  """Norm, wi, wo as a serving program runs them, against float64 with 8-bit roundings.
  A value on the other side of a rounding border moves by a step, 2^-3 of it; at the
  sums' 2^-13 error about one in 2^9 does, so the results differ by far less than the
  2^-4 that rounding itself costs in the root mean square."""
  x, residual, scale, wi, wo = _mlp_inputs(np.random.default_rng(rows), rows, m, f)
  total, y = _mlp(hip, x, residual, scale, wi, wo)
  a = F.value(*F.quantize(_norm_64(total, scale, None, 1e-6)))[:, :m]
  h = np.maximum(a @ F.operand_value(wi)[0].T, 0)
  h = F.value(*F.quantize(h))[:, :f]
  want = h @ F.operand_value(wo)[0].T
  error = np.sqrt(np.square(_f64(y) - want).mean() / np.square(want).mean())
  assert error < 2.0 ** -7


def test_training_step(hip):
  """A dense block's gradients as a training program makes them: dw of both layers and
  dx, against the same products in float64 without any 8-bit rounding."""
  rng = np.random.default_rng(9)
  r, m, f = 260, 192, 328
  x = _tensor(rng, (1, r, m), "bf16", 0.3)
  wi = torch.from_numpy(rng.standard_normal((1, m, f)) * m ** -0.5).to(x)
  wo = torch.from_numpy(rng.standard_normal((1, f, m)) * f ** -0.5).to(x)
  dy = _tensor(rng, (1, r, m), "bf16", 0.3)
  a, a_columns = hip.quantize(x, rows=True, columns=True)
  wi_rows, wi_columns = hip.quantize(wi, rows=True, columns=True)
  wo_rows, wo_columns = hip.quantize(wo, rows=True, columns=True)
  h = hip.expert_linear(a, wi_columns, "relu")
  hq, h_columns = hip.quantize(h, rows=True, columns=True)
  y = hip.expert_linear(hq, wo_columns)
  dh, dwo = hip.expert_linear_backward(h_columns, dy, wo_rows)
  dx, dwi = hip.expert_linear_backward(a_columns, dh, wi_rows, relu_mask=h)

  def near(got, want):
    assert np.sqrt(np.square(_f64(got) - want).mean() /
                   np.square(want).mean()) < 2.0 ** -3.5
  # (against the products without any rounding to 8 bits: two operands of a root mean
  # square error of at most 2^-4 / sqrt(3) each, and as much from what they came from)
  hx = np.maximum(_f64(x[0]) @ _f64(wi[0]), 0)
  near(y[0], hx @ _f64(wo[0]))
  dhx = _f64(dy[0]) @ _f64(wo[0]).T
  near(dh[0], dhx)
  near(dwo[0], hx.T @ _f64(dy[0]))
  # (the mask is the h that the step has: units near 0 are on the other side of it)
  dhx = dhx * (_f64(h[0]) > 0)
  near(dx[0], dhx @ _f64(wi[0]).T)
  near(dwi[0], _f64(x[0]).T @ dhx)


def test_beyond_2_to_the_31_elements(hip):
  """Operands, results and norms of more than 2^31 elements: their first and last rows
  are what the calls make of those alone."""
  rows, k, n = 140032, 16384, 256
  gen = torch.Generator(device="cuda").manual_seed(5)
  x = torch.empty((rows, k), dtype=torch.bfloat16, device="cuda")
  for at in range(0, rows, 8192):
    x[at:at + 8192] = torch.randn((min(8192, rows - at), k), generator=gen, device="cuda")
  ends = (slice(0, 128), slice(rows - 128, rows))
  q, columns = hip.quantize(x, rows=True, columns=True)
  w, wv = _random(hip, (1, n, k), 0.01, 6)
  y = hip.dense(q, w)
  back = hip.dequantize(q)
  total, norm = hip.residual_rms_norm(x, x, x[7].contiguous())
  assert y.shape == (rows, n) and columns.shape == (k, rows)
  wt = wv[0].t().contiguous()
  for sl in ends:
    part = x[sl].contiguous()
    r, c = hip.quantize(part, rows=True, columns=True)
    assert torch.equal(q.values[sl].view(torch.uint8), r.values.view(torch.uint8))
    assert torch.equal(q.scales[sl], r.scales)
    assert torch.equal(columns.values[:, sl].view(torch.uint8),
                       c.values.view(torch.uint8))
    assert torch.equal(back[sl], hip.dequantize(r))
    a = back[sl].double()
    assert _near(y[sl], a @ wt, a.abs() @ wt.abs())
    t, m = hip.residual_rms_norm(part, part, x[7].contiguous())
    assert torch.equal(total[sl], t)
    assert torch.equal(norm.values[sl].view(torch.uint8), m.values.view(torch.uint8))
  del total, norm, back, columns, x
  wide, _ = _random(hip, (1, 17000, 256), 0.05, 8)       # a result of 2.4e9 elements
  a, av = _random(hip, (1, rows, 256), 1.0, 9)
  y = hip.expert_linear(a, wide)[0]
  wt = hip.dequantize(wide, torch.float32)[0].double().t().contiguous()
  for sl in ends:
    assert _near(y[sl], av[0, sl] @ wt, av[0, sl].abs() @ wt.abs())
  dw_rows = hip.quantize(y[None, -300:].contiguous(), rows=False, columns=True)
  assert dw_rows.shape == (1, 17000, 300)


@pytest.mark.parametrize("eight_bit,n", [(False, 20070400), (True, 40140800)])
def test_wide_results_stay_in_their_rows(hip, eight_bit, n):
  """One row whose bytes times the rows that a tile could hold pass 32 bits: the other
  rows of the buffer that the result is the first row of stay as they were."""
  period, k, rows = 1024, 256, 128
  a, av = _random(hip, (1, 1, k), 1.0, 1)
  w, wv = _random(hip, (1, period, k), k ** -0.5, 2)
  wide = hip.Fp8Blocks(
      w.values.view(torch.uint8).repeat(1, n // period, 1).view(torch.float8_e4m3fn),
      w.scales.repeat(1, n // period, 1), k)
  if eight_bit:
    buffer = torch.full((rows, n), 0x55, dtype=torch.uint8, device="cuda")
    scales = torch.full((rows, hip.scale_bytes(n)), 99, dtype=torch.uint8, device="cuda")
    out = hip.Fp8Blocks(buffer[None, :1].view(torch.float8_e4m3fn), scales[None, :1], n)
    hip.expert_linear(a, wide, eight_bit=True, out=out)
    assert (scales[1:] == 99).all()
    y = hip.dequantize(out, torch.float32)
  else:
    buffer = torch.full((rows, n), 0x5555, dtype=torch.int16, device="cuda")
    y = hip.expert_linear(a, wide, out=buffer[None, :1].view(torch.bfloat16))
  assert (buffer[1:] == buffer[1, 0]).all() and buffer[1, 0] % 256 == 0x55
  y = y.view(-1, period)
  assert torch.equal(y, y[:1].expand_as(y))
  wt = wv[0].t().contiguous()
  want, magnitudes = av[0] @ wt, av[0].abs() @ wt.abs()
  if eight_bit:
    # (half a step of e4m3, or of its least numbers under the block's unit)
    top = want.abs().view(-1, 128).amax(-1, keepdim=True).expand(-1, 128).reshape(1, -1)
    half = want.abs() * 2.0 ** -4 + top * 2.0 ** -17
  else:
    half = want.abs() * 2.0 ** -8
  # (7 products of 8 are cut off by up to 2^-13 of the largest: less than 2^-10 of all)
  assert ((y[:1].double() - want).abs() <= half + magnitudes * 2.0 ** -10).all()


@pytest.mark.parametrize("rows", [1, 300])
def test_captured(hip, rows):
  """The block recorded into a graph, replayed with new inputs and work between the
  replays; two graphs and an eager call do not meet."""
  rng = np.random.default_rng(rows)
  inputs = [_mlp_inputs(rng, rows, 256, 640) for _ in range(2)]
  eager = [_mlp(hip, *i) for i in inputs]
  torch.cuda.synchronize()
  graphs = []
  for i in inputs:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
      outs = _mlp(hip, *i)
    graphs.append((graph, outs))
  for _ in range(3):
    for (graph, outs), want in zip(graphs, eager):
      for t in outs:
        t.fill_(-1)
      graph.replay()
      again = _mlp(hip, *inputs[0])
      torch.cuda.synchronize()
      assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])
      assert torch.equal(again[1], eager[0][1])


def test_captured_gradients(hip):
  rng = np.random.default_rng(4)
  a_columns = F.random_operand(rng, (2, 256, 300), 1.0)
  w_rows = F.random_operand(rng, (2, 256, 520), 0.05)
  dy = _tensor(rng, (2, 300, 520), "bf16", 0.5)
  want = hip.expert_linear_backward(a_columns, dy, w_rows)
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph):
    got = hip.expert_linear_backward(a_columns, dy, w_rows)
  for _ in range(3):
    for t in got:
      t.fill_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_streams(hip):
  """Calls on two streams at once give what they give one after the other."""
  rng = np.random.default_rng(11)
  inputs = [_mlp_inputs(rng, 200 + 100 * i, 512, 1024) for i in range(2)]
  want = [_mlp(hip, *i) for i in inputs]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in range(2)]
  for _ in range(3):
    got = []
    for stream, i in zip(streams, inputs):
      with torch.cuda.stream(stream):
        got.append(_mlp(hip, *i))
    torch.cuda.synchronize()
    for (total, y), (total0, y0) in zip(got, want):
      assert torch.equal(total, total0) and torch.equal(y, y0)
