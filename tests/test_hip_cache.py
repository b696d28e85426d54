"""The paged cache's kernels against float64 on the CPU: what rows are kept as, what comes
back, attention of one token over them, and what has to stay as it was."""

import numpy as np
import pytest
import torch

from mesh_amd import cache_hip
from mesh_amd import moe_hip
from tests import cache_reference as C

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
HALF_STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def _gen(seed):
  return torch.Generator(device="cuda").manual_seed(seed)


def _rows(gen, shape, dtype):
  """Rows whose channels differ in size."""
  x = torch.randn(shape, generator=gen, device="cuda")
  return (x * torch.exp(torch.randn(shape[-1:], generator=gen, device="cuda") * 0.5)
          ).to(dtype)


def _np(t):
  return t.double().cpu().numpy()


def _cache(gen, pages, page, heads, width, dtype, eight, shared=False, fill="rows"):
  """A cache and what its pages hold (keys, values): random rows, or bytes whose values
  are NaN."""
  cache = cache_hip.PagedCache.empty(pages, page, heads, width, E4M3 if eight else dtype,
                                     shared_kv=shared)
  for values, scales in ((cache.k_pages, cache.k_scales), (cache.v_pages, cache.v_scales)):
    if values is None:
      continue
    if fill == "nan":
      values.view(torch.uint8).fill_(0xff)
      if eight:
        scales.fill_(127)
    elif eight:
      x = _rows(gen, (pages * heads * page, width), torch.float32)
      codes, exponents = C.F.quantize(_np(x))
      values.copy_(torch.from_numpy(codes[:, :width].reshape(values.shape)).cuda()
                   .view(E4M3))
      scales.copy_(torch.from_numpy(exponents.reshape(scales.shape)).cuda())
    else:
      values.copy_(_rows(gen, values.shape, dtype))
  return cache, _held(cache)


def _held(cache):
  k = C.values_of(cache.k_pages, cache.k_scales)
  return k, (k if cache.v_pages is None else C.values_of(cache.v_pages, cache.v_scales))


def _table(rng, lengths, page, extra=0):
  """Shuffled pages for sequences of these lengths; -1 or a number that no page has
  behind them.  -> (table, pages)"""
  used = [-(-n // page) for n in lengths]
  columns = max(max(used) + extra, 1)
  pages = sum(used) + 2
  order = rng.permutation(pages)
  table = np.full((len(lengths), columns), -1, np.int32)
  table[:, 1::2] = pages + 7
  at = 0
  for i, n in enumerate(used):
    table[i, :n] = order[at:at + n]
    at += n
  return table, pages


def _gpu(a):
  return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _int32(a):
  return _gpu(np.asarray(a, np.int32))


STORES = [("bf16", False), ("bf16", True), ("f32", False), ("f32", True)]
STORE_IDS = ["bf16", "bf16-8", "f32", "f32-8"]


def _bits(t):
  return t.view(torch.uint8)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [
    # heads, width, page, rows per sequence
    (1, 1, 1, 3), (2, 64, 16, 40), (3, 80, 8, 21), (2, 128, 32, 70), (5, 36, 4, 9),
    (1, 256, 16, 17), (2, 200, 16, 5), (7, 8, 2, 1), (4, 130, 64, 66)],
    ids=lambda c: "x".join(map(str, c)))
def test_write_and_read(case, store):
  """Every written row bit for bit, every other byte of the pages as it was; then the way
  back, zeros where there is nothing."""
  heads, width, page, t = case
  dtype, eight = DTYPES[store[0]], store[1]
  rng = np.random.default_rng(sum(case))
  gen = _gen(sum(case) + eight)
  start = np.array([0, 1, page - 1, 2 * page + 1, -2])
  b = len(start)
  table, pages = _table(rng, [max(s, 0) + t for s in start], page, extra=1)
  table[3, 1] = -1                      # (a sequence whose second page is not there)
  count = np.array([t, t // 2, 0, t + 5, t])
  cache, before = _cache(gen, pages, page, heads, width, dtype, eight)
  rows = [_rows(gen, (b, t, heads * width), dtype) for _ in range(2)]
  rows[0][0, 0, :width] = 0             # (a row of zeros)
  rows[1][0, t // 2, 0] *= 2.0 ** 100
  rows[1][1, 0, :width] *= 2.0 ** -120  # (and one next to the least exponent)
  stored = [C.stored(_np(x).reshape(b, t, heads, width), eight) for x in rows]
  untouched = cache_hip.PagedCache(*(None if x is None else x.clone() for x in (
      cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)))
  for counted in (count, None):
    cache_hip.write(cache, rows[0], rows[1], _int32(table), _int32(start),
                    None if counted is None else _int32(counted))
    for got, was, new in zip(_held(cache), before, stored):
      np.testing.assert_array_equal(got, C.write(was, new, table, start, counted, page))
    if counted is not None:
      written = C.write(np.zeros((pages, heads, page, width)),
                        np.ones((b, t, heads, width)), table, start, counted, page)
      same = torch.from_numpy(written == 0).cuda()
      for name in ("k_pages", "v_pages"):
        a, c = (getattr(x, name).view(torch.uint8 if eight else torch.int32 if dtype ==
                                      torch.float32 else torch.int16)
                for x in (cache, untouched))
        assert torch.equal(a[same], c[same])
      if eight:
        rows_same = same[..., 0]
        assert torch.equal(cache.k_scales[rows_same], untouched.k_scales[rows_same])
    k, v = cache_hip.read(cache, _int32(table), _int32(start), t,
                          None if counted is None else _int32(counted), dtype=dtype)
    for got, held in zip((k, v), _held(cache)):
      assert got.dtype == dtype
      np.testing.assert_array_equal(
          _np(got).reshape(b, t, heads, width),
          C.read(held, table, start, t, counted, page))


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [
    # sequences, rows, heads, width, page
    (3, 903, 1, 36, 16), (3, 901, 4, 40, 4), (2, 1101, 8, 128, 32), (2, 1101, 5, 256, 16),
    (2, 1101, 24, 64, 16), (1, 2099, 16, 80, 8), (2, 1102, 20, 131, 64), (4, 701, 2, 17, 1)],
    ids=lambda c: "x".join(map(str, c)))
def test_many_rows(case, store):
  """Rows in twos and fours, shared by one, two and four wavefronts."""
  b, t, heads, width, page = case
  dtype, eight = DTYPES[store[0]], store[1]
  rng, gen = np.random.default_rng(sum(case)), _gen(sum(case))
  start = np.array([3, -2, 0, page + 1])[:b]
  count = np.array([t, t - 3, t // 2 + 1, 0])[:b]
  table, pages = _table(rng, [max(s, 0) + t for s in start], page, extra=1)
  table[0, 2] = -1
  cache, before = _cache(gen, pages, page, heads, width, dtype, eight)
  rows = [_rows(gen, (b, t, heads * width), dtype) for _ in range(2)]
  cache_hip.write(cache, *rows, _int32(table), _int32(start), count=_int32(count))
  held = [C.write(was, C.stored(_np(x).reshape(b, t, heads, width), eight), table, start,
                  count, page) for was, x in zip(before, rows)]
  for got, want in zip(_held(cache), held):
    np.testing.assert_array_equal(got, want)
  for counted in (count, None):
    got = cache_hip.read(cache, _int32(table), _int32(start), t, dtype=dtype,
                         count=None if counted is None else _int32(counted))
    for x, was in zip(got, held):
      np.testing.assert_array_equal(_np(x).reshape(b, t, heads, width),
                                    C.read(was, table, start, t, counted, page))


@pytest.mark.parametrize("store", STORES[:2], ids=STORE_IDS[:2])
def test_rows_at_any_address_and_shared_keys(store):
  """Dense tensors off 16 bytes; a cache whose keys are its values; one row a sequence."""
  dtype, eight = DTYPES[store[0]], store[1]
  rng, gen = np.random.default_rng(5), _gen(5)
  heads, width, page, b = 3, 64, 16, 4
  start = np.array([0, 15, 16, 40])
  table, pages = _table(rng, start + 1, page)
  cache, (before, _) = _cache(gen, pages, page, heads, width, dtype, eight, shared=True)
  buffer = _rows(gen, (b * heads * width + 1,), dtype)
  k = buffer[1:].reshape(b, heads * width)
  assert k.data_ptr() % 16
  cache_hip.write(cache, k, None, _int32(table), _int32(start))
  want = C.stored(_np(k).reshape(b, 1, heads, width), eight)
  np.testing.assert_array_equal(_held(cache)[0],
                                C.write(before, want, table, start, None, page))
  got, same = cache_hip.read(cache, _int32(table), _int32(start), 1, dtype=dtype)
  assert same is got
  np.testing.assert_array_equal(_np(got).reshape(want.shape), want)


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_rows_that_are_not_finite(name):
  """An infinity or a NaN makes its block NaN, and nothing else; the other storages keep
  it as it is."""
  dtype = DTYPES[name]
  gen = _gen(3)
  rows = _rows(gen, (1, 4, 2 * 160), dtype)
  rows[0, 1, 5] = float("inf")
  rows[0, 2, 160 + 130] = float("nan")
  table, at = _int32([[1, 0]]), _int32([0])
  for kind in (E4M3, dtype):
    cache = cache_hip.PagedCache.empty(2, 2, 2, 160, kind)
    cache_hip.write(cache, rows, rows, table, at)
    got = cache_hip.read(cache, table, at, 4, dtype=dtype)[0].float()
    bad = torch.isnan(got) if kind is E4M3 else ~torch.isfinite(got)
    want = torch.zeros_like(bad)
    if kind is E4M3:
      want[0, 1, :128] = True
      want[0, 2, 160 + 128:] = True
    else:
      want[0, 1, 5] = want[0, 2, 160 + 130] = True
    assert torch.equal(bad, want)


def _relative(gen, rng, heads, dtype, reach, buckets=8):
  values = torch.randn((heads, buckets), generator=gen, device="cuda").to(dtype)
  bucket = rng.integers(0, buckets, 2 * reach - 1).astype(np.int32)
  return values, bucket


def _check(got, q, held, table, position, page, name, relative=None):
  heads, width = q.shape[1] // held[0].shape[3], held[0].shape[3]
  want, bound = C.attention(
      _np(q).reshape(-1, heads, width), held[0], held[1], table, position, page,
      HALF_STEP[name], None if relative is None else _np(relative[0]),
      None if relative is None else relative[1])
  off = np.abs(_np(got).reshape(want.shape) - want)
  assert (off <= bound).all(), (off / bound).max()


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [
    # query heads, key / value heads, width, page, bias
    (4, 4, 64, 16, True), (8, 2, 128, 32, False), (3, 1, 80, 8, True),
    (2, 2, 36, 16, False), (20, 1, 64, 64, True), (6, 3, 256, 16, False),
    (1, 1, 1, 1, False), (5, 5, 100, 4, True), (34, 2, 32, 128, False),
    (2, 1, 192, 2, True), (3, 3, 112, 16, False), (2, 2, 13, 32, True),
    (16, 1, 96, 256, False), (1, 1, 48, 16, True), (3, 1, 17, 16, False),
    (4, 2, 33, 8, True), (2, 1, 131, 16, False), (17, 1, 255, 4, False),
    (2, 2, 16, 1, False), (5, 5, 64, 2, True)],
    ids=lambda c: "x".join(map(str, c)))
def test_attention(case, store):
  """Lengths from none to several hundred, pages that end anywhere and some that are not
  there; whatever else the pages hold is NaN."""
  heads, kv, width, page, bias = case
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(sum(case)), _gen(sum(case))
  lengths = [0, 1, 2, 15, 16, 17, 33, 64, 127, 130, 200, 301, 700]
  table, pages = _table(rng, lengths, page, extra=2)
  if page <= 16:
    table[8, 3], table[9, 0] = -1, pages       # (holes in two sequences)
  cache, _ = _cache(gen, pages, page, kv, width, dtype, eight, fill="nan")
  b, t = len(lengths), max(lengths)
  zeros = _int32([0] * b)
  cache_hip.write(cache, _rows(gen, (b, t, kv * width), dtype),
                  _rows(gen, (b, t, kv * width), dtype), _int32(table), zeros,
                  _int32(lengths))
  q = (torch.randn((b, heads * width), generator=gen, device="cuda")
       * 2 * width ** -0.5).to(dtype)
  position = np.array(lengths) - 1
  relative = _relative(gen, rng, heads, dtype, 50) if bias else None
  got = cache_hip.attention(
      q, cache, _int32(table), _int32(position),
      relative_bias=None if relative is None else (relative[0], _gpu(relative[1])))
  assert got.shape == q.shape and got.dtype == dtype
  assert not got[0].any()
  _check(got, q, _held(cache), table, position, page, name, relative)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [(4, 4, 64, 16), (8, 2, 128, 32), (3, 1, 80, 8),
                                  (2, 2, 36, 16), (6, 1, 256, 64), (1, 1, 20, 1)],
                         ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("shared", [False, True], ids=["kv", "shared"])
def test_step(case, store, shared):
  """A step with its own row: the bits of a write and an attention, and nothing else of
  the pages changes."""
  heads, kv, width, page = case
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(sum(case)), _gen(sum(case))
  lengths = np.array([1, 2, 16, 17, 31, 64, 65, 129, 400, 5, 40])
  table, pages = _table(rng, lengths, page)
  cache, _ = _cache(gen, pages, page, kv, width, dtype, eight, shared=shared)
  position = lengths - 1
  position[9] = -1                          # (a place in the batch without a sequence)
  table[10] = -1                            # (and one without pages)
  b = len(lengths)
  q = (torch.randn((b, heads * width), generator=gen, device="cuda")
       * 2 * width ** -0.5).to(dtype)
  k, v = (_rows(gen, (b, kv * width), dtype) for _ in range(2))
  if shared:
    v = None
  buffers = lambda c: [x for x in (c.k_pages, c.v_pages, c.k_scales, c.v_scales)
                       if x is not None]
  other = cache_hip.PagedCache(*(None if x is None else x.clone() for x in (
      cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)))
  got = cache_hip.attention(q, cache, _int32(table), _int32(position), k_new=k, v_new=v)
  cache_hip.write(other, k, v, _int32(table), _int32(position))
  want = cache_hip.attention(q, other, _int32(table), _int32(position))
  for a, c in zip(buffers(cache), buffers(other)):
    assert torch.equal(_bits(a), _bits(c))
  assert torch.equal(got, want)
  _check(got, q, _held(cache), table, position, page, name)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [(4, 4, 64, 16), (8, 2, 128, 32), (6, 1, 256, 64),
                                  (2, 2, 64, 4), (2, 1, 128, 1), (3, 1, 80, 8),
                                  (2, 2, 8, 16)],
                         ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("off", ["query", "keys", "values", "row", "all"])
def test_attention_at_any_address(case, store, off):
  """Operands that lie on their elements' size and not on 16 bytes: the results against
  float64, and the pages' bytes."""
  heads, kv, width, page = case
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(sum(case)), _gen(sum(case))
  lengths = np.array([1, 17, 64, 130, 700, 33])
  table, pages = _table(rng, lengths, page)
  table[3, 0] = -1
  made, held = _cache(gen, pages, page, kv, width, dtype, eight)
  position = lengths - 1

  def moved(x, name):
    if x is None or off not in (name, "all"):
      return x
    buffer = torch.empty(x.numel() + 1, dtype=x.dtype, device="cuda")
    out = buffer[1:].view(x.shape)
    out.copy_(x)
    assert out.data_ptr() % 16
    return out
  cache = cache_hip.PagedCache(moved(made.k_pages, "keys"), moved(made.v_pages, "values"),
                               moved(made.k_scales, "keys"), moved(made.v_scales, "values"))
  b = len(lengths)
  q = moved((torch.randn((b, heads * width), generator=gen, device="cuda")
             * 2 * width ** -0.5).to(dtype), "query")
  k, v = (moved(_rows(gen, (b, kv * width), dtype), "row") for _ in range(2))
  got = cache_hip.attention(q, cache, _int32(table), _int32(position))
  _check(got, q, held, table, position, page, name)
  got = cache_hip.attention(q, cache, _int32(table), _int32(position), k_new=k, v_new=v)
  held = [C.write(was, C.stored(_np(x).reshape(b, 1, kv, width), eight), table, position,
                  None, page) for was, x in zip(held, (k, v))]
  for a, x in zip(_held(cache), held):
    np.testing.assert_array_equal(a, x)
  _check(got, q, held, table, position, page, name)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("width", [1, 5, 8, 15])
def test_narrow_rows(width, store):
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(width), _gen(width)
  lengths = np.array([1, 64, 255, 256, 257, 1500, 3, 40])
  table, pages = _table(rng, lengths, 8)
  table[7, 1:3] = -1
  cache, held = _cache(gen, pages, 8, 2, width, dtype, eight)
  q = (torch.randn((8, 6 * width), generator=gen, device="cuda") * 2).to(dtype)
  position = lengths - 1
  position[6] = -1
  relative = _relative(gen, rng, 6, dtype, 300)
  for bias in (None, relative):
    got = cache_hip.attention(q, cache, _int32(table), _int32(position),
                              relative_bias=bias and (bias[0], _gpu(bias[1])))
    _check(got, q, held, table, position, 8, name, bias)
  k, v = (_rows(gen, (8, 2 * width), dtype) for _ in range(2))
  got = cache_hip.attention(q, cache, _int32(table), _int32(position), k_new=k, v_new=v)
  held = [C.write(was, C.stored(_np(x).reshape(8, 1, 2, width), eight), table, position,
                  None, 8) for was, x in zip(held, (k, v))]
  _check(got, q, held, table, position, 8, name)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
def test_narrow_rows_in_a_wide_table(store):
  """Rows of fewer than 16 values under a table of 2^30 positions: their kernel does not
  divide them, so that the bound on what is divided is not theirs."""
  name, eight = store
  dtype = DTYPES[name]
  b, kv, heads, page, columns = 4, 64, 128, 1 << 16, 1 << 14
  gen = _gen(30)
  cache = cache_hip.PagedCache.empty(b, page, kv, 1, E4M3 if eight else dtype)
  lengths = np.array([300, 1, 0, 257])
  table = np.full((b, columns), -1, np.int32)
  table[:, 0] = np.arange(b)[::-1]
  rows = [_rows(gen, (b, 300, kv), dtype) for _ in range(2)]
  cache_hip.write(cache, *rows, _int32(table), _int32([0] * b), count=_int32(lengths))
  q = torch.randn((b, heads), generator=gen, device="cuda").to(dtype)
  got = cache_hip.attention(q, cache, _int32(table), _int32(lengths - 1))
  held = [C.stored(_np(x).reshape(b, 300, kv, 1), eight).transpose(0, 2, 1, 3)[::-1]
          for x in rows]
  _check(got, q, held, np.arange(b)[::-1][:, None], lengths - 1, 300, name)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [
    # sequences, longest, query heads, key / value heads, width, page, columns more
    (5, 70, 2, 2, 64, 16, 0), (3, 90, 3, 1, 128, 32, 200), (4, 40, 2, 1, 256, 64, 0),
    (3, 60, 2, 2, 80, 8, 0), (4, 30, 1, 1, 40, 2, 0), (3, 20, 2, 1, 200, 16, 0),
    (3, 20, 2, 1, 8, 16, 0), (800, 25, 2, 2, 64, 32, 0), (800, 25, 1, 1, 128, 8, 500)],
    ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("byte", [0xff, 0x00])
def test_rows_that_nothing_was_written_to(case, store, byte):
  """Whatever bytes pages and scales have where nothing was written, it does not matter."""
  b, longest, heads, kv, width, page, more = case
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(b + width), _gen(b + width)
  lengths = rng.integers(0, longest + 1, b)
  lengths[:3] = longest, 1, 0
  table, pages = _table(rng, lengths, page, extra=more)
  table[0, table.shape[1] // 2] = -1
  cache, _ = _cache(gen, pages, page, kv, width, dtype, eight)
  for x in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales):
    if x is not None:
      x.view(torch.uint8).fill_(byte)
  rows = [_rows(gen, (b, longest, kv * width), dtype) for _ in range(2)]
  cache_hip.write(cache, *rows, _int32(table), _int32([0] * b), count=_int32(lengths))
  held = [C.write(np.zeros((pages, kv, page, width)),
                  C.stored(_np(x).reshape(b, longest, kv, width), eight), table, [0] * b,
                  lengths, page) for x in rows]
  q = (torch.randn((b, heads * width), generator=gen, device="cuda")
       * 2 * width ** -0.5).to(dtype)
  got = cache_hip.attention(q, cache, _int32(table), _int32(lengths - 1))
  _check(got, q, held, table, lengths - 1, page, name)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [
    # lengths, query heads, key / value heads, width, page
    ([20011], 2, 1, 128, 64), ([9000, 3, 4096, 1], 2, 2, 64, 16),
    ([2500] * 3, 1, 1, 40, 32), ([6000, 700], 20, 1, 64, 32), ([5000], 2, 1, 256, 16),
    ([3000, 40], 3, 1, 128, 1), ([4100], 1, 1, 72, 8)],
    ids=["one", "uneven", "odd", "tiles", "wide", "rows", "small"])
def test_long_sequences(case, store):
  lengths, heads, kv, width, page = case
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(len(lengths)), _gen(len(lengths))
  table, pages = _table(rng, lengths, page)
  cache, held = _cache(gen, pages, page, kv, width, dtype, eight)
  q = (torch.randn((len(lengths), heads * width), generator=gen, device="cuda")
       * 2 * width ** -0.5).to(dtype)
  position = np.array(lengths) - 1
  got = cache_hip.attention(q, cache, _int32(table), _int32(position))
  _check(got, q, held, table, position, page, name)
  again = cache_hip.attention(q, cache, _int32(table), _int32(position))
  assert torch.equal(got, again)


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_many_sequences(name):
  """More sequences than a wavefront has lanes, and than several have."""
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(8), _gen(8)
  lengths = rng.integers(0, 60, 700)
  lengths[-1] = 900
  table, pages = _table(rng, lengths, 16)
  cache, held = _cache(gen, pages, 16, 2, 64, dtype, False)
  q = _rows(gen, (700, 4 * 64), torch.float32).mul(0.2).to(dtype)
  position = lengths - 1
  got = cache_hip.attention(q, cache, _int32(table), _int32(position))
  _check(got, q, held, table, position, 16, name)


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("case", [
    # sequences, query heads, key / value heads, width, page, longest, columns more
    (160, 8, 8, 64, 16, 100, 0), (160, 8, 8, 64, 16, 120, 500), (70, 32, 16, 128, 16, 90, 300),
    (400, 19, 1, 80, 8, 60, 700), (400, 3, 3, 33, 2, 60, 0), (800, 1, 1, 256, 1, 30, 9),
    (790, 2, 1, 256, 32, 70, 0), (300, 4, 4, 100, 4, 50, 600), (130, 6, 6, 128, 8, 100, 800)],
    ids=lambda c: "x".join(map(str, c)))
@pytest.mark.parametrize("longer", [False, True], ids=["short", "one-longer"])
def test_many_short_sequences(case, store, longer):
  """More heads of short sequences than there are blocks, with and without a longer
  sequence among them: over what is there, and as a step with a bias."""
  b, heads, kv, width, page, longest, more = case
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(b), _gen(b)
  lengths = rng.integers(0, longest + 1, b)
  lengths[:4] = longest, 0, 1, 17
  if longer:
    lengths[b // 2] = 1500
  table, pages = _table(rng, lengths, page, extra=more)
  table[5, 0] = -1                          # (a sequence without its first page)
  cache, held = _cache(gen, pages, page, kv, width, dtype, eight)
  q = (torch.randn((b, heads * width), generator=gen, device="cuda")
       * 2 * width ** -0.5).to(dtype)
  position = lengths - 1
  got = cache_hip.attention(q, cache, _int32(table), _int32(position))
  _check(got, q, held, table, position, page, name)
  k, v = (_rows(gen, (b, kv * width), dtype) for _ in range(2))
  relative = _relative(gen, rng, heads, dtype, 40)
  got = cache_hip.attention(q, cache, _int32(table), _int32(position), k_new=k, v_new=v,
                            relative_bias=(relative[0], _gpu(relative[1])))
  want = [C.write(was, C.stored(_np(x).reshape(b, 1, kv, width), eight), table, position,
                  None, page) for was, x in zip(held, (k, v))]
  for a, x in zip(_held(cache), want):
    np.testing.assert_array_equal(a, x)
  _check(got, q, want, table, position, page, name, relative)


@pytest.mark.parametrize("eight", [False, True])
def test_more_than_the_grid_has(eight):
  """More rows of a sequence, and more sequences, than a launch has blocks for at once."""
  gen = _gen(21)
  t, page, width = 300001, 1024, 16
  cache, (before, _) = _cache(gen, 295, page, 1, width, torch.bfloat16, eight, shared=True)
  table = np.arange(294, dtype=np.int32)[::-1].copy()[None]
  k = _rows(gen, (1, t, width), torch.bfloat16)
  cache_hip.write(cache, k, None, _int32(table), _int32([5]))
  got = cache_hip.read(cache, _int32(table), _int32([5]), t)[0]
  stored = C.stored(_np(k).reshape(1, t, 1, width), eight)
  there = min(t, 294 * page - 5)
  want = np.zeros((t, width))
  want[:there] = stored[0, :there, 0]
  np.testing.assert_array_equal(_np(got)[0], want)
  np.testing.assert_array_equal(_held(cache)[0][294], before[294])
  b = 17001
  cache, _ = _cache(gen, b, 2, 1, width, torch.bfloat16, eight)
  table = np.random.default_rng(21).permutation(b).astype(np.int32)[:, None]
  rows = [_rows(gen, (b, width), torch.bfloat16) for _ in range(2)]
  at = np.arange(b) % 3 - 1
  cache_hip.write(cache, rows[0], rows[1], _int32(table), _int32(at))
  for got, x in zip(cache_hip.read(cache, _int32(table), _int32(at), 1), rows):
    want = C.stored(_np(x), eight) * (at >= 0)[:, None]
    np.testing.assert_array_equal(_np(got)[:, 0], want)
  held = _held(cache)
  q = _rows(gen, (b, 2 * width), torch.float32).mul(0.3).bfloat16()
  got = cache_hip.attention(q, cache, _int32(table), _int32(at))
  _check(got, q, held, table, at, 2, "bf16")


def test_shared_pages():
  """Sequences that begin with the same pages, and one that has a page twice."""
  rng, gen = np.random.default_rng(22), _gen(22)
  page = 16
  cache, held = _cache(gen, 9, page, 2, 64, torch.bfloat16, False)
  table = np.array([[3, 7, 1, 0], [3, 7, 2, 8], [5, 5, 5, -1]], np.int32)
  position = np.array([60, 49, 47])
  q = _rows(gen, (3, 4 * 64), torch.float32).mul(0.1).bfloat16()
  got = cache_hip.attention(q, cache, _int32(table), _int32(position))
  _check(got, q, held, table, position, page, "bf16")
  k, _ = cache_hip.read(cache, _int32(table), _int32([0, 3, 1]), 30)
  np.testing.assert_array_equal(
      _np(k).reshape(3, 30, 2, 64), C.read(held[0], table, [0, 3, 1], 30, None, page))
  del rng


def test_buckets_that_there_are_not():
  """Bucket numbers out of range read nothing out of bounds: they count as the nearest."""
  gen = _gen(23)
  table = np.arange(5, dtype=np.int32)[None]
  cache, held = _cache(gen, 5, 16, 2, 64, torch.bfloat16, False)
  q = _rows(gen, (1, 128), torch.float32).mul(0.1).bfloat16()
  values = torch.randn((2, 4), generator=gen, device="cuda").bfloat16()
  bucket = np.full(39, 1 << 30, np.int32)
  bucket[::2] = -1 << 30
  got = cache_hip.attention(q, cache, _int32(table), _int32([79]),
                            relative_bias=(values, _gpu(bucket)))
  _check(got, q, held, table, np.array([79]), 16, "bf16", (values, np.clip(bucket, 0, 3)))


def test_positions_behind_the_table():
  """A position from P * S on: what is there is seen, the step's row goes nowhere."""
  rng, gen = np.random.default_rng(9), _gen(9)
  table, pages = _table(rng, [32, 32], 16)
  cache, held = _cache(gen, pages, 16, 2, 64, torch.bfloat16, False)
  q, k = _rows(gen, (2, 128), torch.bfloat16), _rows(gen, (2, 128), torch.bfloat16)
  for position in ([32, 100], [2 ** 31 - 1, -2 ** 31]):
    position = np.array(position)
    got = cache_hip.attention(q, cache, _int32(table), _int32(position), k_new=k, v_new=k)
    for now, was in zip(_held(cache), held):
      np.testing.assert_array_equal(now, was)
    _check(got, q, held, table, position, 16, "bf16")
    rows = cache_hip.read(cache, _int32(table), _int32(position), 3)[0]
    assert not rows[0].any()


@pytest.mark.parametrize("name", ["bf16", "f32"])
def test_biases_of_lowest_values_and_infinities(name):
  """A bias of the type's lowest value or of -infinity takes a position out; where that
  takes all of them out, lowest values leave their differences, -infinities nothing."""
  dtype = DTYPES[name]
  gen = _gen(11)
  heads, width, page, n = 3, 64, 16, 300
  table = np.arange(19, dtype=np.int32)[None]
  cache, held = _cache(gen, 19, page, heads, width, dtype, False)
  q = _rows(gen, (1, heads * width), torch.float32).mul(0.1).to(dtype)
  bucket = np.zeros(2 * n - 1, np.int32)
  bucket[:n] = np.arange(n) % 3
  for low in (float("-inf"), torch.finfo(dtype).min):
    values = torch.zeros((heads, 3), dtype=dtype, device="cuda")
    values[0, 1] = low
    values[1, :2] = low
    got = cache_hip.attention(q, cache, _int32(table), _int32([n - 1]),
                              relative_bias=(values, _gpu(bucket)))
    _check(got, q, held, table, np.array([n - 1]), page, name, (values, bucket))
    values[:] = low
    got = cache_hip.attention(q, cache, _int32(table), _int32([n - 1]),
                              relative_bias=(values, _gpu(bucket)))
    if low == float("-inf"):
      assert not got.any()
    else:
      assert torch.isfinite(got.float()).all()


def test_what_is_not_finite_stays_in_its_head():
  gen = _gen(12)
  table, at = _int32([[0, 1, 2], [3, 4, 5]]), _int32([40, 40])
  cache, _ = _cache(gen, 6, 16, 2, 64, torch.bfloat16, False)
  q = _rows(gen, (2, 256), torch.float32).mul(0.1).bfloat16()
  clean = cache_hip.attention(q, cache, table, at)
  cache.k_pages[1, 0, 3, 5] = float("nan")
  cache.v_pages[4, 1, 2, 7] = float("inf")
  cache.v_pages[5, 0, 15] = float("nan")         # (behind the second sequence's last)
  got = cache_hip.attention(q, cache, table, at).reshape(2, 4, 64)
  clean = clean.reshape(2, 4, 64)
  assert torch.isnan(got[0, :2]).all()
  assert torch.equal(got[0, 2:], clean[0, 2:]) and torch.equal(got[1, :2], clean[1, :2])
  assert torch.isinf(got[1, 2:, 7]).all()
  keep = torch.arange(64, device="cuda") != 7
  assert torch.equal(got[1, 2:][:, keep], clean[1, 2:][:, keep])


@pytest.mark.parametrize("store", STORES, ids=STORE_IDS)
@pytest.mark.parametrize("width,at", [(17, 10), (33, 27), (72, 64), (131, 127), (200, 199)])
def test_queries_that_are_infinite(width, at, store):
  """Every value of a query counts once, also where the pieces of a row overlap: an infinite
  one with keys below zero there makes all logits -infinity, and the output 0."""
  dtype, eight = DTYPES[store[0]], store[1]
  gen = _gen(width + at)
  cache = cache_hip.PagedCache.empty(3, 16, 1, width, E4M3 if eight else dtype)
  k = torch.rand((1, 40, width), generator=gen, device="cuda").sub(0.5).to(dtype)
  k[..., at] = -0.25
  v = _rows(gen, (1, 40, width), dtype)
  table = _int32([[2, 0, 1]])
  cache_hip.write(cache, k, v, table, _int32([0]))
  q = torch.ones((1, 2 * width), dtype=dtype, device="cuda")
  q[0, at] = float("inf")
  out = cache_hip.attention(q, cache, table, _int32([39]))
  assert torch.equal(out[0, :width], torch.zeros_like(out[0, :width]))
  want, _ = cache_hip.attention(torch.ones_like(q), cache, table, _int32([39])).split(width, 1)
  assert torch.equal(out[:, width:], want)


@pytest.mark.parametrize("eight", [False, True])
def test_pages_beyond_32_bits(eight):
  """Pages whose offsets pass 2^32 elements."""
  gen = _gen(13)
  page, heads, width = 64, 4, 256
  pages = (1 << 32) // (page * heads * width) + 40
  cache = cache_hip.PagedCache.empty(pages, page, heads, width,
                                     E4M3 if eight else torch.bfloat16, shared_kv=True)
  ids = np.concatenate([[0], np.arange(pages - 9, pages)]).astype(np.int32)
  table, n = ids[None], 10 * page - 3
  rows = _rows(gen, (1, n, heads * width), torch.bfloat16)
  cache_hip.write(cache, rows, None, _int32(table), _int32([0]))
  got = cache_hip.read(cache, _int32(table), _int32([0]), n)[0]
  want = C.stored(_np(rows).reshape(1, n, heads, width), eight)
  np.testing.assert_array_equal(_np(got).reshape(want.shape), want)
  q = _rows(gen, (1, heads * width), torch.float32).mul(0.1).bfloat16()
  out = cache_hip.attention(q, cache, _int32(table), _int32([n - 1]))
  flat = np.zeros((10 * page, heads, width))
  flat[:n] = want[0]
  held = flat.reshape(10, page, heads, width).transpose(0, 2, 1, 3)
  _check(out, q, (held, held), np.arange(10, dtype=np.int32)[None], np.array([n - 1]),
         page, "bf16")
  del cache, rows, got
  torch.cuda.empty_cache()


@pytest.mark.parametrize("store", STORES[:3], ids=STORE_IDS[:3])
def test_recorded_steps(store):
  """Steps recorded once and replayed as the sequences grow, between eager calls on the
  same cache; two graphs that share the memory of their workspaces."""
  name, eight = store
  dtype = DTYPES[name]
  rng, gen = np.random.default_rng(14), _gen(14)
  heads, width, page = 4, 64, 16
  lengths = np.array([1000, 3, 500])
  table, pages = _table(rng, lengths + 40, page)
  cache, _ = _cache(gen, pages, page, heads, width, dtype, eight)
  other = cache_hip.PagedCache(*(x if x is None else x.clone() for x in (
      cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)))
  tables, position = _int32(table), _int32(lengths)
  q, k, v = (_rows(gen, (3, heads * width), dtype) for _ in range(3))
  q = q * 0.2
  step = lambda c: cache_hip.attention(q, c, tables, position, k_new=k, v_new=v)
  stream = torch.cuda.Stream()
  graphs, outs, reads, pool = [], [], [], None
  torch.cuda.synchronize()
  with torch.cuda.stream(stream):
    step(cache)
    step(other)
    stream.synchronize()
    for _ in range(2):
      graph = torch.cuda.CUDAGraph()
      with torch.cuda.graph(graph, pool=pool, stream=stream):
        outs.append(step(cache))
        reads.append(cache_hip.read(cache, tables, position, 2, dtype=dtype))
      pool = graph.pool()
      graphs.append(graph)
  torch.cuda.synchronize()
  for i in range(6):
    position.add_(1)
    k.copy_(_rows(gen, k.shape, dtype))
    q.copy_(_rows(gen, q.shape, dtype) * 0.2)
    graphs[i % 2].replay()
    want = step(other)
    torch.cuda.synchronize()
    assert torch.equal(outs[i % 2], want), i
    for a, c in zip(reads[i % 2], cache_hip.read(other, tables, position, 2, dtype=dtype)):
      assert torch.equal(a[:, 0], c[:, 0])
    for a, c in ((cache.k_pages, other.k_pages), (cache.v_pages, other.v_pages)):
      assert torch.equal(_bits(a), _bits(c))
    torch.empty(1 << 20, device="cuda").normal_()


@pytest.mark.parametrize("eight", [False, True])
def test_recorded_with_wide_tiles(eight):
  """16 heads of 256 a tile: the launches that ask for more than 64 KB of LDS."""
  rng, gen = np.random.default_rng(24), _gen(24)
  lengths = np.array([700, 90])
  table, pages = _table(rng, lengths, 16)
  cache, held = _cache(gen, pages, 16, 1, 256, torch.bfloat16, eight)
  tables, position = _int32(table), _int32(lengths - 1)
  q = _rows(gen, (2, 16 * 256), torch.float32).mul(0.05).bfloat16()
  stream = torch.cuda.Stream()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph, stream=stream):
    out = cache_hip.attention(q, cache, tables, position)
  for shift in (0, 13, 40):
    position.copy_(_int32(lengths - 1 - shift))
    graph.replay()
    torch.cuda.synchronize()
    _check(out, q, held, table, lengths - 1 - shift, 16, "bf16")
    assert torch.equal(out, cache_hip.attention(q, cache, tables, position))


def test_recorded_while_lengths_grow():
  """A recorded call whose sequences are all short in one replay, and not in the next."""
  rng, gen = np.random.default_rng(25), _gen(25)
  lengths = np.full(100, 200)
  lengths[37] = 1200
  table, pages = _table(rng, lengths, 16, extra=10)
  cache, held = _cache(gen, pages, 16, 8, 128, torch.bfloat16, False)
  tables, position = _int32(table), _int32(lengths * 0)
  q = _rows(gen, (100, 16 * 128), torch.float32).mul(0.1).bfloat16()
  stream = torch.cuda.Stream()
  torch.cuda.synchronize()
  graph = torch.cuda.CUDAGraph()
  with torch.cuda.graph(graph, stream=stream):
    out = cache_hip.attention(q, cache, tables, position)
  for at in (lengths * 0 - 1, np.minimum(lengths - 1, 180), lengths - 1, lengths * 0 + 5):
    position.copy_(_int32(at))
    graph.replay()
    torch.cuda.synchronize()
    _check(out, q, held, table, at, 16, "bf16")
    assert torch.equal(out, cache_hip.attention(q, cache, tables, position))


def test_two_streams():
  """Calls at once on two streams, over the same pages."""
  rng, gen = np.random.default_rng(15), _gen(15)
  lengths = np.array([5000, 900])
  table, pages = _table(rng, lengths, 32)
  cache, held = _cache(gen, pages, 32, 2, 128, torch.bfloat16, False)
  tables, position = _int32(table), _int32(lengths - 1)
  qs = [_rows(gen, (2, 8 * 128), torch.float32).mul(0.1).bfloat16() for _ in range(2)]
  wants = [cache_hip.attention(q, cache, tables, position) for q in qs]
  torch.cuda.synchronize()
  streams = [torch.cuda.Stream() for _ in range(2)]
  outs = [[], []]
  for _ in range(10):
    for i, s in enumerate(streams):
      with torch.cuda.stream(s):
        outs[i].append(cache_hip.attention(qs[i], cache, tables, position))
  torch.cuda.synchronize()
  for want, got in zip(wants, outs):
    assert all(torch.equal(g, want) for g in got)
  _check(wants[0], qs[0], held, table, lengths - 1, 32, "bf16")


def test_refusals():
  gen = _gen(16)
  cache, _ = _cache(gen, 4, 16, 2, 64, torch.bfloat16, False)
  eight, _ = _cache(gen, 4, 16, 2, 64, torch.bfloat16, True)
  shared, _ = _cache(gen, 4, 16, 2, 64, torch.bfloat16, False, shared=True)
  x = torch.zeros((2, 128), dtype=torch.bfloat16, device="cuda")
  table, at = _int32([[0, 1], [2, 3]]), _int32([0, 0])
  bad = moe_hip.MoeHipError
  values = torch.zeros((2, 4), dtype=torch.bfloat16, device="cuda")
  for call in (
      lambda: cache_hip.write(cache, x[:, :64], x[:, :64], table, at),
      lambda: cache_hip.write(cache, x, x[:1], table, at),
      lambda: cache_hip.write(cache, x, None, table, at),
      lambda: cache_hip.write(shared, x, x, table, at),
      lambda: cache_hip.write(cache, x.float(), x.float(), table, at),
      lambda: cache_hip.write(eight, x.half(), x.half(), table, at),
      lambda: cache_hip.write(cache, x, x, table[:1], at),
      lambda: cache_hip.write(cache, x, x, table.long(), at),
      lambda: cache_hip.write(cache, x, x, table, at[:1]),
      lambda: cache_hip.write(cache, x, x, table, at, at.long()),
      lambda: cache_hip.write(cache, x.t().contiguous().t(), x, table, at),
      lambda: cache_hip.read(cache, table, at, 2, dtype=torch.float32),
      lambda: cache_hip.read(cache, table, at[:1], 2),
      lambda: cache_hip.read(cache, table.reshape(-1), at, 2),
      lambda: cache_hip.read(cache, table, at, 1 << 31),
      lambda: cache_hip.attention(x[:, :64].contiguous(), cache, table, at),
      lambda: cache_hip.attention(x.reshape(-1), cache, table, at),
      lambda: cache_hip.attention(x.float(), cache, table, at),
      lambda: cache_hip.attention(x, cache, table, at, k_new=x),
      lambda: cache_hip.attention(x, cache, table, at, v_new=x),
      lambda: cache_hip.attention(x, shared, table, at, k_new=x, v_new=x),
      lambda: cache_hip.attention(x, cache, table, at, k_new=x, v_new=x[:, :64]),
      lambda: cache_hip.attention(x, cache, table, at, relative_bias=(
          values, torch.zeros(4, dtype=torch.int32, device="cuda"))),
      lambda: cache_hip.attention(x, cache, table, at, relative_bias=(
          values[:1], torch.zeros(5, dtype=torch.int32, device="cuda"))),
      lambda: cache_hip.attention(x, cache, table, at, relative_bias=(
          values.float(), torch.zeros(5, dtype=torch.int32, device="cuda")))):
    with pytest.raises(bad):
      call()
  with pytest.raises(ValueError):
    cache_hip.read(cache, table, at, -1)
  # what there is nothing of
  none = torch.zeros((2, 0), dtype=torch.int32, device="cuda")
  cache_hip.write(cache, x, x, none, at)
  assert not cache_hip.attention(x, cache, none, at).any()
  assert not cache_hip.read(cache, none, at, 3)[0].any()
  assert cache_hip.read(cache, table, at, 0)[0].shape == (2, 0, 128)
  assert cache_hip.attention(x[:0], cache, table[:0], at[:0]).shape == (0, 128)
