"""ctypes binding of the paged cache of libmesh_moe_hip.so (declared in
include/mesh_moe_cache.h): keys and values of sequences in pages, in the activations' type
or in 8 bits, and attention of one new token over them.

The calls follow those of moe_hip, whose attention_decode keeps its states as whole
tensors: GPU tensors that are contiguous, checked on the host; launched on the current
stream; nothing kept between calls but how large a workspace of some sizes is, so that each
can be recorded into a HIP graph.  All tensors of a call have to lie on the current device.

A decoding program keeps a PagedCache for each layer and one table for all of them:

  cache = PagedCache.empty(pages, page_size, heads, d_kv, torch.float8_e4m3fn, "cuda")
  write(cache, k, v, table, start, count)          # a prompt's rows, [batch, length, ...]
  out = attention(q, cache, table, position, k_new=k, v_new=v)   # then step by step

Which pages a sequence has is the program's business: table [batch, columns] int32 names
the page of every page_size positions, -1 one that it does not have (yet).
"""

import ctypes
import functools

import torch

from mesh_amd import fp8_hip
from mesh_amd import moe_hip
from mesh_amd.moe_hip import MoeHipError

ABI_VERSION = 2
BLOCK = fp8_hip.BLOCK
_E4M3 = torch.float8_e4m3fn

_vp = ctypes.c_void_p
_int = ctypes.c_int
_size = ctypes.c_size_t
_SIGNATURES = {
    "mesh_moe_cache_abi_version": (_int, []),
    "mesh_moe_cache_write": (_int, [_vp] * 9 + [_int] * 8 + [_vp]),
    "mesh_moe_cache_read": (_int, [_vp] * 9 + [_int] * 8 + [_vp]),
    "mesh_moe_cache_attention_workspace_bytes": (_size, [_int] * 8),
    "mesh_moe_cache_attention": (_int, [_vp] * 11 + [_int] * 2 + [_vp] + [_int] * 8 + [
        _vp, _size, _vp]),
}
EXPORTS = sorted(_SIGNATURES)

_lib = None


def load_library():
  """The library with the entry points of this module declared."""
  global _lib
  if _lib is None:
    lib = moe_hip.load_library()
    for name, (restype, argtypes) in _SIGNATURES.items():
      fn = getattr(lib, name)  # AttributeError if a symbol is missing
      fn.restype = restype
      fn.argtypes = argtypes
    version = lib.mesh_moe_cache_abi_version()
    if version != ABI_VERSION:
      raise MoeHipError("cache ABI version %d, expected %d" % (version, ABI_VERSION))
    _lib = lib
  return _lib


_empty = torch.empty
_empty_like = torch.empty_like
_current_device = moe_hip.current_device
_dev = fp8_hip._dev        # pylint: disable=protected-access
_stage = moe_hip._stage    # pylint: disable=protected-access
_check = moe_hip._check    # pylint: disable=protected-access
_stream = moe_hip._stream  # pylint: disable=protected-access
_ints = fp8_hip._ints      # pylint: disable=protected-access


def scale_blocks(d):
  """Scale bytes of a row of d 8-bit values."""
  return (d + BLOCK - 1) // BLOCK


class PagedCache(object):
  """Pages of keys and values: k_pages, v_pages [pages, heads, page_size, d_kv] in
  float32, bfloat16 or float8_e4m3fn, the latter with k_scales, v_scales [pages, heads,
  page_size, scale_blocks(d_kv)] uint8; value i of a row stands for value *
  2^(scales[i // 128] - 127).  v_pages None: the keys are the values (shared_kv)."""

  __slots__ = ("_k", "_v", "_k_scales", "_v_scales", "_shape", "_device")

  def __init__(self, k_pages, v_pages=None, k_scales=None, v_scales=None):
    shape, dtype = k_pages.shape, k_pages.dtype
    eight = dtype is _E4M3
    if len(shape) != 4 or 0 in shape or (v_pages is None and v_scales is not None):
      raise ValueError("pages %s: expected [pages, heads, page_size, d_kv]"
                       % (tuple(shape),))
    if shape[2] & (shape[2] - 1):
      raise ValueError("pages of %d rows, not a power of two" % shape[2])
    if not eight:
      moe_hip.dtype_code(dtype)
    if (v_pages is not None and (
        v_pages.dtype is not dtype or v_pages.shape != shape or
        (v_scales is not None) != eight)) or (k_scales is not None) != eight:
      raise ValueError("pages of keys %s and of values %s differ, or are without their "
                       "scales" % (tuple(shape), None if v_pages is None else
                                   tuple(v_pages.shape)))
    if eight:
      blocks = shape[:-1] + (scale_blocks(shape[3]),)
      for scales in (k_scales, v_scales):
        if scales is not None and (scales.dtype is not torch.uint8 or
                                   scales.shape != blocks):
          raise ValueError("scales %s of %s do not go with pages %s"
                           % (tuple(scales.shape), scales.dtype, tuple(shape)))
    self._k, self._v = k_pages, v_pages
    self._k_scales, self._v_scales = k_scales, v_scales
    self._shape = shape
    # the device of all buffers, where they are what the library takes
    self._device = None
    if k_pages.is_cuda:
      device = k_pages.get_device()
      if k_pages.is_contiguous() and all(
          x is None or (x.is_cuda and x.get_device() == device and x.is_contiguous())
          for x in ((v_pages, k_scales, v_scales) if eight else (v_pages,))):
        self._device = device

  @classmethod
  def empty(cls, pages, page_size, heads, d_kv, dtype=torch.bfloat16, device="cuda",
            shared_kv=False):
    """A cache whose rows hold nothing yet."""
    sizes = (pages, heads, page_size, d_kv)
    blocks = sizes[:-1] + (scale_blocks(d_kv),)
    made = []
    for wanted in (True, not shared_kv):
      made.append(_empty(sizes, dtype=dtype, device=device) if wanted else None)
    for wanted in (True, not shared_kv):
      made.append(_empty(blocks, dtype=torch.uint8, device=device)
                  if wanted and dtype is _E4M3 else None)
    return cls(*made)

  k_pages = property(lambda self: self._k)
  v_pages = property(lambda self: self._v)
  k_scales = property(lambda self: self._k_scales)
  v_scales = property(lambda self: self._v_scales)
  pages = property(lambda self: self._shape[0])
  heads = property(lambda self: self._shape[1])
  page_size = property(lambda self: self._shape[2])
  d_kv = property(lambda self: self._shape[3])
  dtype = property(lambda self: self._k.dtype)
  eight_bit = property(lambda self: self._k_scales is not None)
  shared_kv = property(lambda self: self._v is None)

  def overlaps(self, other):
    """Whether some of this cache's buffers and of the other's are the same memory."""
    def spans(cache):
      return [(t.device, t.data_ptr(), t.data_ptr() + t.numel() * t.element_size())
              for t in (cache.k_pages, cache.v_pages, cache.k_scales, cache.v_scales)
              if t is not None]
    return any(a[0] == b[0] and a[1] < b[2] and b[1] < a[2]
               for a in spans(self) for b in spans(other))

  def __repr__(self):
    return "PagedCache(pages=%d, heads=%d, page_size=%d, d_kv=%d, dtype=%s)" % (
        tuple(self._shape) + (self.dtype,))


def _pointers(cache):
  """Of the pages and scales, in the order of the library's arguments."""
  if not isinstance(cache, PagedCache):
    raise MoeHipError("cache must be a PagedCache")
  # pylint: disable=protected-access
  k, v, ks, vs = cache._k, cache._v, cache._k_scales, cache._v_scales
  if cache._device is None or cache._device != _current_device():
    for t, name in ((k, "k_pages"), (v, "v_pages"), (ks, "k_scales"), (vs, "v_scales")):
      if t is not None:
        _dev(t, name)            # (says what is wrong with it)
  return (k.data_ptr(), None if v is None else v.data_ptr(),
          None if ks is None else ks.data_ptr(), None if vs is None else vs.data_ptr())


def _type(cache, dtype):
  """The library's code of the dense tensors' type, which is the cache's own if that
  is not of 8 bits."""
  if cache._k_scales is None and dtype is not cache._k.dtype:  # pylint: disable=protected-access
    raise MoeHipError("%s and a cache of %s" % (dtype, cache.dtype))
  return moe_hip.dtype_code(dtype)


def _table(table, batch):
  if table.dim() != 2:
    raise MoeHipError("table %s, expected [batch, columns]" % (tuple(table.shape),))
  columns = table.shape[1]
  return _dev(table, "table", torch.int32, (batch, columns)), columns


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes):
  return load_library().mesh_moe_cache_attention_workspace_bytes(*sizes)


def write(cache, k, v, table, position, count=None):
  """Rows k, v [B, T, heads * d_kv] (or one row per sequence, [B, heads * d_kv]) become
  the positions position[b] + t of sequence b (position [B] int32); with count [B] int32
  only the first count[b] of them.  v is None for a cache with shared_kv.  Rows without a
  page are left out."""
  lib = load_library()
  pointers = _pointers(cache)
  n, heads, s, d = cache._shape  # pylint: disable=protected-access
  shape = k.shape
  if len(shape) not in (2, 3) or shape[-1] != heads * d:
    raise MoeHipError("k %s, expected [batch, rows, %d]" % (tuple(shape), heads * d))
  b, t = shape[0], (shape[1] if len(shape) == 3 else 1)
  code = _type(cache, k.dtype)
  if (v is None) != cache.shared_kv:
    raise MoeHipError("v is given with caches that have pages of values, and only there")
  _ints(b, t, n, table.shape[-1])
  kp = _dev(k, "k")
  vp = None if v is None else _dev(v, "v", k.dtype, shape)
  tp, columns = _table(table, b)
  pp = _dev(position, "position", torch.int32, (b,))
  cp = None if count is None else _dev(count, "count", torch.int32, (b,))
  if k.numel() and columns:
    with _stage("cache_write"):
      _check(lib.mesh_moe_cache_write(
          kp, vp, tp, pp, cp, *pointers, b, t, heads, d, n, s, columns, code,
          _stream()), "cache_write")


def read(cache, table, position, length, count=None, dtype=None):
  """What the cache holds, dense: (k, v) [B, length, heads * d_kv], row t of sequence b
  being position position[b] + t; zeros from count[b] on ([B] int32, None: none are) and
  where there is no page.  v is k for a cache with shared_kv.  dtype: of the result, for
  8-bit caches (bfloat16 if not given); exact."""
  lib = load_library()
  pointers = _pointers(cache)
  n, heads, s, d = cache._shape  # pylint: disable=protected-access
  b = position.shape[0] if position.dim() else 0
  if dtype is None:
    dtype = torch.bfloat16 if cache.eight_bit else cache.dtype
  code = _type(cache, dtype)
  _ints(b, length, n, table.shape[-1])
  if length < 0:
    raise ValueError("length %d" % length)
  tp, columns = _table(table, b)
  pp = _dev(position, "position", torch.int32, (b,))
  cp = None if count is None else _dev(count, "count", torch.int32, (b,))
  make = _empty if columns else torch.zeros
  k = make((b, length, heads * d), dtype=dtype, device=position.device)
  v = None if cache.shared_kv else _empty_like(k) if columns else k.clone()
  if k.numel() and columns:
    with _stage("cache_read"):
      _check(lib.mesh_moe_cache_read(
          *pointers, tp, pp, cp, k.data_ptr(), None if v is None else v.data_ptr(), b,
          length, heads, d, n, s, columns, code, _stream()), "cache_read")
  return k, (k if v is None else v)


def _relative_bias(relative_bias, dtype, heads):
  if relative_bias is None:
    return None, None, 0, 0
  values, bucket = relative_bias
  if values.dim() != 2 or bucket.dim() != 1 or bucket.shape[0] % 2 == 0:
    raise MoeHipError("relative_bias %s, %s: expected [heads, buckets] and [2 reach - 1]"
                      % (tuple(values.shape), tuple(bucket.shape)))
  buckets, reach = values.shape[1], (bucket.shape[0] + 1) // 2
  _ints(buckets, reach)
  return (_dev(values, "relative values", dtype, (heads, buckets)),
          _dev(bucket, "relative bucket", torch.int32), buckets, reach)


def attention(q, cache, table, position, k_new=None, v_new=None, relative_bias=None):
  """One decoding step: q [B, H * d_kv] over the positions 0 .. position[b] ([B] int32)
  that sequence b has in the cache -> out [B, H * d_kv]; zeros for a sequence without any
  (position -1).  H is a multiple of the cache's heads, H / heads query heads that follow
  each other share one.  Logits are q . k: scaling is part of q.

  k_new, v_new [B, heads * d_kv] (v_new None with shared_kv): the step's own row, which
  becomes position[b] first.  relative_bias = (values [H, NB] of q's dtype, bucket
  [2 reach - 1] int32) or None: values[h][bucket[j - position[b] + reach - 1]] is added
  to the logit of position j; farther back than reach - 1 the bucket of that distance
  counts."""
  lib = load_library()
  pointers = _pointers(cache)
  n, heads, s, d = cache._shape  # pylint: disable=protected-access
  shape = q.shape
  if len(shape) != 2 or shape[1] % (heads * d) or not shape[1]:
    raise MoeHipError("q %s, expected [batch, a multiple of %d]"
                      % (tuple(shape), heads * d))
  b, h = shape[0], shape[1] // d
  dtype = q.dtype
  code = _type(cache, dtype)
  if (k_new is None and v_new is not None) or (
      k_new is not None and (v_new is None) != cache.shared_kv):
    raise MoeHipError("k_new and v_new go together, as the cache's keys and values do")
  _ints(b, h, n, table.shape[-1])
  qp = _dev(q, "q")
  kp = None if k_new is None else _dev(k_new, "k_new", dtype, (b, heads * d))
  vp = None if v_new is None else _dev(v_new, "v_new", dtype, (b, heads * d))
  tp, columns = _table(table, b)
  pp = _dev(position, "position", torch.int32, (b,))
  relative = _relative_bias(relative_bias, dtype, h)
  if not (b and columns):
    return torch.zeros_like(q)
  out = _empty_like(q)
  ws_bytes = _workspace_bytes(b, h, heads, d, s, columns, code, cache.eight_bit)
  ws = _empty((ws_bytes,), dtype=torch.uint8, device=q.device) if ws_bytes else None
  with _stage("cache_attention"):
    _check(lib.mesh_moe_cache_attention(
        qp, kp, vp, *pointers, tp, pp, *relative, out.data_ptr(), b, h, heads, d, n, s,
        columns, code, None if ws is None else ws.data_ptr(), ws_bytes, _stream()),
           "cache_attention")
  return out
