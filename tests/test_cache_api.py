"""The paged cache's interface on the CPU: exported symbols, what a cache is made of, and
what is refused before a launch."""

import os
import re

import numpy as np
import pytest
import torch

from mesh_amd import cache_hip
from mesh_amd import moe_hip

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E4M3 = torch.float8_e4m3fn


@pytest.fixture(scope="module")
def lib():
  if not os.path.exists(moe_hip.LIB_PATH):
    from mesh_amd.csrc import build
    build.build_library(verbose=False)
  return cache_hip.load_library()


def test_library_exports_every_declared_symbol(lib):
  header = open(os.path.join(ROOT, "include", "mesh_moe_cache.h")).read()
  code = re.sub(r"/\*.*?\*/", " ", header, flags=re.DOTALL)
  declared = set(re.findall(r"\b(mesh_moe_cache_[a-z0-9_]+)\s*\(", code))
  assert declared == set(cache_hip.EXPORTS)
  for name in declared:
    assert getattr(lib, name) is not None
  version = re.search(r"MESH_MOE_CACHE_ABI_VERSION (\d+)", header).group(1)
  assert lib.mesh_moe_cache_abi_version() == cache_hip.ABI_VERSION == int(version)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, E4M3])
@pytest.mark.parametrize("shared", [False, True])
def test_empty_cache(dtype, shared):
  c = cache_hip.PagedCache.empty(5, 16, 3, 200, dtype, "cpu", shared_kv=shared)
  assert (c.pages, c.page_size, c.heads, c.d_kv) == (5, 16, 3, 200)
  assert c.k_pages.shape == (5, 3, 16, 200) and c.dtype == dtype
  assert c.eight_bit == (dtype == E4M3) and c.shared_kv == shared
  assert (c.v_pages is None) == shared
  if c.eight_bit:
    assert c.k_scales.shape == (5, 3, 16, 2) and c.k_scales.dtype == torch.uint8
    assert (c.v_scales is None) == shared
  else:
    assert c.k_scales is None and c.v_scales is None
  assert "page_size=16" in repr(c)


def test_pages_that_are_no_cache():
  def pages(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype)
  k8, s8 = pages(4, 2, 8, 32, dtype=E4M3), pages(4, 2, 8, 1, dtype=torch.uint8)
  for args in ((pages(4, 8, 32), None), (pages(4, 2, 8, 32), pages(4, 2, 8, 16)),
               (pages(4, 2, 8, 32), pages(4, 2, 8, 32, dtype=torch.float32)),
               (pages(0, 2, 8, 32), None), (pages(4, 2, 8, 32), None, s8),
               (k8, k8), (k8, k8, s8), (k8, k8, s8, s8[:1]), (k8, None, s8, s8),
               (k8, k8, s8, s8.to(torch.int8)), (pages(4, 2, 12, 32), None)):
    with pytest.raises(ValueError):
      cache_hip.PagedCache(*args)
  with pytest.raises(moe_hip.MoeHipError, match="dtype"):
    cache_hip.PagedCache(pages(4, 2, 8, 32, dtype=torch.float16))


def test_cpu_tensors_are_refused(lib):
  del lib
  cache = cache_hip.PagedCache.empty(4, 8, 2, 32, device="cpu")
  x = torch.zeros(3, 64, dtype=torch.bfloat16)
  table = torch.zeros(3, 2, dtype=torch.int32)
  at = torch.zeros(3, dtype=torch.int32)
  for call in (lambda: cache_hip.write(cache, x, x, table, at),
               lambda: cache_hip.read(cache, table, at, 4),
               lambda: cache_hip.attention(x, cache, table, at)):
    with pytest.raises(moe_hip.MoeHipError, match="GPU tensor"):
      call()
  with pytest.raises(moe_hip.MoeHipError, match="PagedCache"):
    cache_hip.write(x, x, x, table, at)


# addresses that are never read: every call below is refused before a launch
AT = 1 << 20


def _refused(lib, rc, code, words):
  assert rc == code
  text = lib.mesh_moe_last_error().decode()
  assert words in text, text


def _changed(call, ok):
  def with_(**changes):
    args = list(ok)
    for at, v in changes.items():
      args[int(at[1:])] = v
    return call(*args)
  return with_


def test_write_refusals(lib):
  # k v table position count k_pages v_pages k_scales v_scales B T HK D N S P dtype
  with_ = _changed(lib.mesh_moe_cache_write,
                   [AT] * 4 + [None] + [AT] * 4 + [2, 3, 4, 64, 5, 16, 6, 1, None])
  for change in (dict(_0=None), dict(_2=None), dict(_3=None), dict(_5=None)):
    _refused(lib, with_(**change), -1, "null")
  for change in (dict(_1=None), dict(_6=None)):
    _refused(lib, with_(**change), -1, "go together")
  for change in (dict(_7=None), dict(_8=None), dict(_1=None, _6=None)):
    _refused(lib, with_(**change), -1, "scales")
  for at in range(9, 16):
    _refused(lib, with_(**{"_%d" % at: 0}), -1, "sizes")
  _refused(lib, with_(_16=2), -1, "dtype")
  _refused(lib, with_(_14=24), -2, "power of two")
  _refused(lib, with_(_12=257), -2, "256")
  _refused(lib, with_(_11=65537), -2, "65536")
  _refused(lib, with_(_14=1 << 16, _15=1 << 15), -2, "2^30")
  _refused(lib, with_(_10=(1 << 30) + 1), -2, "2^30")


def test_read_refusals(lib):
  # k_pages v_pages k_scales v_scales table position count k v B T HK D N S P dtype
  with_ = _changed(lib.mesh_moe_cache_read,
                   [AT] * 6 + [None] + [AT] * 2 + [2, 3, 4, 64, 5, 16, 6, 0, None])
  for change in (dict(_0=None), dict(_4=None), dict(_5=None), dict(_7=None)):
    _refused(lib, with_(**change), -1, "null")
  for change in (dict(_1=None), dict(_8=None)):
    _refused(lib, with_(**change), -1, "go together")
  for change in (dict(_2=None), dict(_3=None)):
    _refused(lib, with_(**change), -1, "scales")
  for at in range(9, 16):
    _refused(lib, with_(**{"_%d" % at: -1}), -1, "sizes")
  _refused(lib, with_(_16=2), -1, "dtype")
  _refused(lib, with_(_14=3), -2, "power of two")
  _refused(lib, with_(_10=(1 << 30) + 1), -2, "2^30")


def test_attention_refusals(lib):
  # q k_new v_new k_pages v_pages k_scales v_scales table position rel_values rel_bucket
  # num_buckets reach out B H HK D N S P dtype workspace bytes
  with_ = _changed(lib.mesh_moe_cache_attention,
                   [AT] * 9 + [None, None, 0, 0, AT, 2, 8, 4, 64, 5, 16, 6, 1, AT,
                               1 << 40, None])
  for change in (dict(_0=None), dict(_3=None), dict(_7=None), dict(_8=None),
                 dict(_13=None)):
    _refused(lib, with_(**change), -1, "null")
  for change in (dict(_1=None), dict(_2=None), dict(_4=None, _6=None)):
    _refused(lib, with_(**change), -1, "go together")
  for change in (dict(_5=None), dict(_6=None)):
    _refused(lib, with_(**change), -1, "scales")
  for change in (dict(_9=AT), dict(_10=AT), dict(_9=AT, _10=AT, _11=4),
                 dict(_9=AT, _10=AT, _12=4)):
    _refused(lib, with_(**change), -1, "go together")
  for at in (14, 16, 17, 18, 19, 20):
    _refused(lib, with_(**{"_%d" % at: 0}), -1, "sizes")
  for heads in (0, 6):
    _refused(lib, with_(_15=heads), -1, "query heads")
  _refused(lib, with_(_21=5), -1, "dtype")
  _refused(lib, with_(_17=260), -2, "256")
  _refused(lib, with_(_14=1 << 30), -2, "more than a launch")
  need = lib.mesh_moe_cache_attention_workspace_bytes(2, 8, 4, 64, 16, 1 << 20, 1, 1)
  if need:
    _refused(lib, with_(_20=1 << 20, _23=need - 1), -1, "workspace")
    _refused(lib, with_(_20=1 << 20, _22=None), -1, "workspace")


def test_paged_states_of_layers():
  """What a layer takes for its state, and where it looks for it."""
  import mesh_amd as mtf
  from mesh_amd.transformer import attention
  from mesh_amd.transformer import transformer
  cache = cache_hip.PagedCache.empty(6, 8, 2, 16, device="cpu")
  state = attention.PagedState(cache, torch.zeros(3, 2, dtype=torch.int32))
  state.check(32, 2, [3], False)
  for args in ((64, 2, [3], False), (32, 4, [3], False), (32, 2, [3], True),
               (32, 2, [2], False), (32, 2, [3, 1], False)):
    with pytest.raises(ValueError):
      state.check(*args)
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  batch, channels = mtf.Dimension("batch", 3), mtf.Dimension("heads", 32)
  t = lambda *dims, **kw: mtf.import_tf_tensor(
      mesh, torch.zeros([d.size for d in dims], **kw), mtf.Shape(list(dims)))
  q, other = t(batch, channels), t(batch, mtf.Dimension("heads", 16))
  position = t(batch, dtype=torch.int32)
  op = attention.PagedDecodeOperation(q, q, q, position, state, 2)
  assert op.outputs[0].shape == q.shape
  for args in ((q, other, q, position, state, 2), (q, q, q, other, state, 2),
               (q, q, q, position, state, 4), (q, q, None, position, state, 2)):
    with pytest.raises(ValueError):
      attention.PagedDecodeOperation(*args)
  model = transformer.Unitransformer(None, d_model=16)
  context = transformer.Context(
      model, mesh, [batch], mtf.Dimension("length", 8), mtf.VariableDType(torch.float32),
      mode="incremental", position=position, states=[q, q, state])
  assert context.paged_state() is None
  context.record_new_states(context.get_states(2))
  assert context.paged_state() is state
  context.record_new_states([state])
  assert context.paged_state() is None
  # pages that an earlier layer has already
  context = transformer.Context(
      model, mesh, [batch], mtf.Dimension("length", 8), mtf.VariableDType(torch.float32),
      mode="incremental", position=position,
      states=[state, attention.PagedState(cache, state.table)])
  context.record_new_states([context.paged_state()])
  with pytest.raises(ValueError, match="the same pages"):
    context.paged_state()


@pytest.mark.parametrize("bidirectional", [False, True])
def test_distances_that_share_the_last_bucket(bidirectional):
  """A bucket table that ends where the last bucket begins stands for all distances behind
  it; where there is no last bucket, none is cut."""
  from mesh_amd.transformer import attention
  once = 2 if bidirectional else 1
  for buckets in list(range(2, 70)) + list(range(250, 256)):
    buckets *= once
    far = attention.last_bucket_from(bidirectional, buckets)
    assert far <= attention.MAX_DISTANCE
    got = attention.relative_position_bucket(-np.arange(far, 5000), bidirectional, buckets)
    assert (got == got[0]).all()
  for buckets in (256, 257, 300, 1000):
    assert attention.last_bucket_from(bidirectional, buckets * once) is None
  # the distance at which a table of 129 positions was wrong
  got = attention.relative_position_bucket(np.array([-128, -139]), bidirectional, 300 * once)
  assert got.tolist() == [128, 139]


@pytest.mark.parametrize("bidirectional", [False, True])
def test_bucket_tables_hold_buckets(bidirectional):
  """Kernels index the bias with what a table holds, so all of it is in range, also where
  the formula (which ends at MAX_DISTANCE) gives far positions negative numbers."""
  from mesh_amd.transformer import attention
  for buckets in (8, 32, 254, 256, 257, 258, 300, 512, 600, 1000):
    for length in (1, 129, 150, 512, 3001):
      with np.errstate(all="ignore"):        # (it divides by log(1) for some of them)
        table = attention.relative_bucket_table(length, bidirectional, buckets, "cpu")
      assert table.dtype == torch.int32 and table.shape == (2 * length - 1,)
      assert 0 <= int(table.min()) and int(table.max()) < buckets, (buckets, length)
  # (what the formula has in range stays as it is)
  got = attention.relative_bucket_table(512, bidirectional, 300, "cpu").numpy()
  formula = attention.relative_position_bucket(np.arange(-511, 512), bidirectional, 300)
  inside = (formula >= 0) & (formula < 300)
  np.testing.assert_array_equal(got[inside], formula[inside])


@pytest.mark.parametrize("eight", [False, True])
def test_layers_with_the_same_buffers(eight):
  """Two layers' caches are two objects, but one memory: refused; parts of one buffer that
  do not meet are taken."""
  import mesh_amd as mtf
  from mesh_amd.transformer import attention
  from mesh_amd.transformer import transformer
  mesh = mtf.Mesh(mtf.Graph(), "mesh")
  batch = mtf.Dimension("batch", 3)
  position = mtf.import_tf_tensor(mesh, torch.zeros(3, dtype=torch.int32),
                                  mtf.Shape([batch]))
  table = torch.zeros(3, 2, dtype=torch.int32)
  kind = E4M3 if eight else torch.bfloat16

  def caches(first, second):
    """Of pages `first` and `second` (keys, values) of one buffer."""
    pages = torch.empty((6, 4, 2, 8, 16), dtype=kind)
    scales = [torch.empty((6, 4, 2, 8, 1), dtype=torch.uint8) if eight else None] * 2
    return [cache_hip.PagedCache(pages[k], None if v is None else pages[v], *(
        None if x is None or at is None else x[at] for x, at in zip(scales, (k, v))))
            for k, v in (first, second)]

  def second_state(one, two):
    context = transformer.Context(
        transformer.Unitransformer(None, d_model=16), mesh, [batch],
        mtf.Dimension("length", 8), mtf.VariableDType(torch.float32), mode="incremental",
        position=position, states=[attention.PagedState(c, table) for c in (one, two)])
    context.record_new_states([context.paged_state()])
    return context.paged_state()

  for pair in (((0, 1), (0, 1)), ((0, 1), (2, 1)), ((0, 1), (1, 0)), ((0, None), (1, 0)),
               ((3, None), (3, None))):
    with pytest.raises(ValueError, match="the same pages"):
      second_state(*caches(*pair))
  for pair in (((0, 1), (2, 3)), ((5, 0), (1, 4)), ((0, None), (1, None))):
    one, two = caches(*pair)
    assert second_state(one, two).cache is two
  # buffers that meet in a part only
  flat = torch.empty(6 * 2 * 8 * 16, dtype=torch.float32)
  size = 4 * 2 * 8 * 16
  one, two = (cache_hip.PagedCache(flat[at:at + size].view(4, 2, 8, 16))
              for at in (0, flat.numel() - size))
  with pytest.raises(ValueError, match="the same pages"):
    second_state(one, two)


def test_workspaces_that_are_too_small(lib):
  """A table of 2^24 positions is divided among blocks, which takes a workspace; one that
  is short, or of narrow rows, is not."""
  # (arguments as above)
  with_ = _changed(lib.mesh_moe_cache_attention,
                   [AT] * 9 + [None, None, 0, 0, AT, 2, 8, 4, 64, 5, 16, 1 << 20, 1, AT,
                               1 << 40, None])
  for dtype in (0, 1):
    for eight in (0, 1):
      for d in (16, 64, 128, 200, 256):
        need = lib.mesh_moe_cache_attention_workspace_bytes(2, 8, 4, d, 16, 1 << 20, dtype,
                                                            eight)
        assert need > 0
        pages = dict() if eight else dict(_5=None, _6=None)
        # (rows of other widths may do with fewer blocks)
        short = need - 1 if d in (64, 128, 256) else need // 4
        _refused(lib, with_(_17=d, _21=dtype, _23=short, **pages), -1, "workspace")
        _refused(lib, with_(_17=d, _21=dtype, _22=None, **pages), -1, "workspace")
        assert lib.mesh_moe_cache_attention_workspace_bytes(2, 8, 4, d, 16, 4, dtype,
                                                            eight) == 0
      assert lib.mesh_moe_cache_attention_workspace_bytes(2, 8, 4, 15, 16, 1 << 20, dtype,
                                                          eight) == 0


@pytest.mark.parametrize("d,dtype,eight,rows", [
    (64, 1, True, 256), (128, 1, True, 256), (256, 1, True, 128), (64, 1, False, 128),
    (256, 1, False, 128), (64, 0, True, 128), (256, 0, True, 64), (64, 0, False, 128),
    (128, 0, False, 64), (16, 0, False, 128)])
def test_limits_of_attention(lib, d, dtype, eight, rows):
  """The header's bound on heads times positions, from both sides: within it a call goes
  on, up to its missing workspace."""
  scales = dict() if eight else dict(_5=None, _6=None)
  with_ = _changed(lib.mesh_moe_cache_attention,
                   [AT] * 9 + [None, None, 0, 0, AT, 1, 34, 2, d, 5, 1 << 10, 1 << 20,
                               dtype, None, 0, None])
  units = 2 * 2                                 # (17 heads in tiles of 16, twice)
  most = ((1 << 31) - 1) // ((1 << 30) // rows + 1) // units
  _refused(lib, with_(_14=most, **scales), -1, "workspace")
  _refused(lib, with_(_14=most + 1, **scales), -2, "more than a launch")
  assert lib.mesh_moe_cache_attention_workspace_bytes(
      most, 34, 2, d, 1 << 10, 1 << 20, dtype, int(eight)) > 0
  assert lib.mesh_moe_cache_attention_workspace_bytes(
      most + 1, 34, 2, d, 1 << 10, 1 << 20, dtype, int(eight)) == 0
  # more heads than workgroups, however short the table, also with narrow rows
  _refused(lib, with_(_14=1 << 22, _19=1, _20=1, **scales), -2, "more than a launch")
  _refused(lib, with_(_14=(1 << 24) // 34 + 1, _17=8, _19=1, _20=1, **scales), -2,
           "more than a launch")


def test_sizes_that_are_kept_are_bounded(lib):
  """A server's batches and tables change without end; what is kept of them does not."""
  del lib
  most = cache_hip._workspace_bytes.cache_info().maxsize
  assert most is not None
  for columns in range(1, most + 50):
    cache_hip._workspace_bytes(2, 8, 4, 64, 16, columns, 1, False)
  assert cache_hip._workspace_bytes.cache_info().currsize <= most
