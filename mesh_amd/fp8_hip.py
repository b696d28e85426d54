"""ctypes binding of the 8-bit operands of libmesh_moe_hip.so (declared in
include/mesh_moe_fp8.h): dense layers and experts on e4m3 numbers with a scale for each
block of 128, the passes that make such operands, and the RMS norm that ends in one.

An operand is an Fp8Blocks.  The calls follow those of moe_hip, whose bf16 forms they
are: GPU tensors that are contiguous, checked on the host; launched on the current
stream; nothing kept between calls, so that each can be recorded into a HIP graph.  All
tensors of a call have to lie on the current device.

A dense layer in training (w [K, N] bf16, x [rows, K], dy [rows, N]):

  w_rows, w_columns = quantize(w.unsqueeze(0), rows=True, columns=True)  # per update
  a, a_columns = quantize(x.unsqueeze(0), rows=True, columns=True)
  y = expert_linear(a, w_columns)
  dx, dw = expert_linear_backward(a_columns, dy.unsqueeze(0), w_rows)
"""

import ctypes

import torch

from mesh_amd import moe_hip
from mesh_amd.moe_hip import MoeHipError

ABI_VERSION = 3
BLOCK = 128
_E4M3 = torch.float8_e4m3fn

_vp = ctypes.c_void_p
_int = ctypes.c_int
_size = ctypes.c_size_t
_SIGNATURES = {
    "mesh_moe_fp8_abi_version": (_int, []),
    "mesh_moe_fp8_quantize": (_int, [_vp] * 7 + [_int] * 4 + [_vp]),
    "mesh_moe_fp8_dequantize": (_int, [
        _vp, _vp, _vp, ctypes.c_int64, _int, _int, _vp]),
    "mesh_moe_fp8_residual_rms_norm": (_int, [_vp] * 8 + [
        ctypes.c_int64, _int, ctypes.c_double, _int, _vp]),
    "mesh_moe_fp8_expert_linear_exact": (_int, [_int] * 6),
    "mesh_moe_fp8_expert_linear_workspace_bytes": (_size, [_int] * 5),
    "mesh_moe_fp8_expert_linear": (_int, [_vp] * 7 + [_int] * 5 + [
        _vp, _size, _vp]),
    "mesh_moe_fp8_expert_linear_backward_workspace_bytes": (_size, [_int] * 5),
    "mesh_moe_fp8_expert_linear_backward": (_int, [_vp] * 9 + [_int] * 5 + [
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
    version = lib.mesh_moe_fp8_abi_version()
    if version != ABI_VERSION:
      raise MoeHipError("8-bit ABI version %d, expected %d" % (version, ABI_VERSION))
    _lib = lib
  return _lib


def row_bytes(n):
  """Bytes of a row of n values: whole blocks."""
  return (n + BLOCK - 1) // BLOCK * BLOCK


def scale_bytes(n):
  """Scale bytes of a row of n values: a byte per block, whole groups of four."""
  return ((n + BLOCK - 1) // BLOCK + 3) // 4 * 4


class Fp8Blocks(object):
  """An 8-bit operand: values [..., rows, row_bytes(n)] of torch.float8_e4m3fn, scales
  [..., rows, scale_bytes(n)] of torch.uint8; value i of a row stands for values[i] *
  2^(scales[i // 128] - 127).  The values from n on are zeros."""

  __slots__ = ("_values", "_scales", "_shape")

  def __init__(self, values, scales, n):
    n = int(n)
    shape = values.shape
    lead = tuple(shape[:-1])
    if (values.dtype is not _E4M3 or scales.dtype is not torch.uint8 or n < 1 or
        not shape or shape[-1] != row_bytes(n) or
        scales.shape != lead + (scale_bytes(n),)):
      raise ValueError(
          "values %s of %s and scales %s of %s are not rows of %d 8-bit values"
          % (tuple(shape), values.dtype, tuple(scales.shape), scales.dtype, n))
    self._set(values, scales, lead + (n,))

  def _set(self, values, scales, shape):
    self._values = values
    self._scales = scales
    self._shape = shape
    return self

  @property
  def values(self):
    return self._values

  @property
  def scales(self):
    return self._scales

  @property
  def n(self):
    return self._shape[-1]

  @property
  def shape(self):
    """Of the tensor that the operand stands for."""
    return self._shape

  @classmethod
  def empty(cls, shape, device):
    """An operand for a tensor of `shape`, not filled in."""
    shape = tuple(shape)
    rows, n = shape[:-1], shape[-1]
    if n < 1:
      raise ValueError("rows without values: shape %s" % (shape,))
    # (what __init__ checks holds by construction)
    return cls.__new__(cls)._set(  # pylint: disable=protected-access
        _empty(rows + (row_bytes(n),), dtype=torch.float8_e4m3fn, device=device),
        _empty(rows + (scale_bytes(n),), dtype=torch.uint8, device=device), shape)

  def reshape(self, *rows):
    """The same rows under other leading dimensions."""
    values = self._values.reshape(rows + self._values.shape[-1:])
    scales = self._scales.reshape(rows + self._scales.shape[-1:])
    return Fp8Blocks.__new__(Fp8Blocks)._set(
        values, scales, tuple(values.shape[:-1]) + self._shape[-1:])

  def __repr__(self):
    return "Fp8Blocks%s" % (self.shape,)


_empty = torch.empty
_Tensor = torch.Tensor
_current_device = moe_hip.current_device


def _dev(t, name, dtype=None, shape=None):
  # (one expression for what passes: the checks cost as much as a small kernel)
  if (isinstance(t, _Tensor) and t.is_cuda and t.get_device() == _current_device() and
      t.is_contiguous() and (dtype is None or t.dtype is dtype) and
      (shape is None or t.shape == shape)):
    return t.data_ptr()
  at = moe_hip._dev(t, name, dtype, shape)  # pylint: disable=protected-access
  if t.get_device() != _current_device():
    raise MoeHipError("%s lies on %s, the current device is %d"
                      % (name, t.device, _current_device()))
  return at


def _operand(q, name, shape=None):
  """Pointers to an operand's values and scales."""
  if not isinstance(q, Fp8Blocks):
    raise MoeHipError("%s must be an Fp8Blocks" % name)
  if shape is not None and q.shape != shape:
    raise MoeHipError("%s: shape %s, expected %s" % (name, q.shape, shape))
  values, scales = q._values, q._scales  # pylint: disable=protected-access
  if (values.is_cuda and scales.is_cuda and
      values.get_device() == scales.get_device() == _current_device() and
      values.is_contiguous() and scales.is_contiguous()):
    return values.data_ptr(), scales.data_ptr()
  return _dev(values, name + ".values"), _dev(scales, name + ".scales")


def _pointers(q):
  """Of an operand that was made here."""
  if q is None:
    return None, None
  return q._values.data_ptr(), q._scales.data_ptr()  # pylint: disable=protected-access


# (a larger argument of a C call would lose its upper bits)
_INT_MAX = 0x7fffffff


def _ints(*sizes):
  """Refuses sizes that the library's calls cannot be given."""
  if max(sizes) > _INT_MAX:
    raise MoeHipError("a size of %s is beyond 2^31 - 1" % (sizes,))


def _counts(row_count, e):
  return (None if row_count is None
          else _dev(row_count, "row_count", torch.int32, (e,)))


def _workspace(nbytes, like):
  return _empty((nbytes,), dtype=torch.uint8, device=like.device)


def _activation(name):
  if name not in moe_hip.ACTIVATIONS:
    raise ValueError("unsupported activation %r" % (name,))
  return moe_hip.ACTIVATIONS[name]


_stage = moe_hip._stage    # pylint: disable=protected-access
_check = moe_hip._check    # pylint: disable=protected-access
_stream = moe_hip._stream  # pylint: disable=protected-access


def quantize(x, rows=True, columns=False, relu_mask=None, row_count=None, out=None):
  """x [E, R, K] (or [R, K]) as 8-bit operands, in one pass over it: its rows
  [E, R, K], for products over K, its columns [E, K, R], for products over R, or both.
  relu_mask (shape and dtype of x): elements whose mask is not positive count as 0.
  row_count [E] int32: rows of an expert from its count on count as zeros.  out: the
  operand, or the pair, to write to instead of new ones.
  -> the one operand asked for, or (rows, columns)

  The columns of a weight [E, K, N] are what expert_linear multiplies by (as
  moe_hip.pack_weights lays out a bf16 one), its rows what expert_linear_backward
  needs."""
  lib = load_library()
  if not (rows or columns):
    raise ValueError("neither rows nor columns are wanted")
  if x.dim() not in (2, 3):
    raise ValueError("x %s, expected [E, R, K] or [R, K]" % (tuple(x.shape),))
  sizes = tuple(x.shape)
  e, r, k = (1,) * (3 - x.dim()) + sizes
  _ints(e, r, k)
  code = moe_hip.dtype_code(x.dtype)
  turned = sizes[:-2] + (k, r)
  by_row = by_column = None
  if out is None:
    if rows:
      by_row = Fp8Blocks.empty(sizes, x.device)
    if columns:
      by_column = Fp8Blocks.empty(turned, x.device)
    outs = _pointers(by_row) + _pointers(by_column)
  else:
    by_row, by_column = (out if rows and columns else (out, None) if rows
                         else (None, out))
    outs = ((_operand(by_row, "rows", sizes) if rows else (None, None)) +
            (_operand(by_column, "columns", turned) if columns else (None, None)))
  xp = _dev(x, "x")
  mp = None if relu_mask is None else _dev(relu_mask, "relu_mask", x.dtype, sizes)
  cp = _counts(row_count, e)
  if x.numel():
    with _stage("fp8_quantize"):
      _check(lib.mesh_moe_fp8_quantize(
          xp, mp, cp, *outs, e, r, k, code, _stream()), "fp8_quantize")
  return (by_row, by_column) if rows and columns else by_row if rows else by_column


def dequantize(q, dtype=torch.bfloat16):
  """The tensor that an operand stands for, exact in bfloat16 and float32."""
  lib = load_library()
  code = moe_hip.dtype_code(dtype)
  _ints(q.n)
  y = _empty(q.shape, dtype=dtype, device=q.values.device)
  values, scales = _operand(q, "q")
  if y.numel():
    with _stage("fp8_dequantize"):
      _check(lib.mesh_moe_fp8_dequantize(values, scales, y.data_ptr(),
                                         y.numel() // q.n, q.n, code, _stream()),
             "fp8_dequantize")
  return y


def residual_rms_norm(x, residual, scale, epsilon=1e-6, row_mask=None,
                      want_norm=False):
  """rms_norm(x + residual) * row_mask as an 8-bit operand: x, residual (or None) [...,
  M], scale [M], row_mask [...] (or None) -> (x + residual or x itself, Fp8Blocks [...,
  M]).  want_norm: also the result in x's dtype, as a third one (what a training step
  quantizes the columns of; for programs without a graph: a graph with gradients makes the
  norm in bfloat16 and quantizes that, rows and columns, in one pass)."""
  lib = load_library()
  m = x.shape[-1]
  shape = tuple(x.shape)
  code = moe_hip.dtype_code(x.dtype)
  _ints(m)
  xp, sp = _dev(x, "x"), _dev(scale, "scale", x.dtype, (m,))
  rp = None if residual is None else _dev(residual, "residual", x.dtype, shape)
  mp = None if row_mask is None else _dev(row_mask, "row_mask", x.dtype, shape[:-1])
  total = x if residual is None else torch.empty_like(x)
  norm = torch.empty_like(x) if want_norm else None
  y = Fp8Blocks.empty(shape, x.device)
  if x.numel():
    with _stage("rms_norm"):
      _check(lib.mesh_moe_fp8_residual_rms_norm(
          xp, rp, sp, mp, None if residual is None else total.data_ptr(),
          None if norm is None else norm.data_ptr(), *_pointers(y),
          x.numel() // m, m, float(epsilon), code, _stream()), "fp8_residual_rms_norm")
  return (total, y, norm) if want_norm else (total, y)


def _linear(a, w, sizes, shape, activation, eight_bit, row_count, out):
  """expert_linear with sizes (e, r, k, n); `shape`: of the result."""
  lib = load_library()
  e, r, k, n = sizes
  _ints(e, r, k, n)
  ap, asp = _operand(a, "a")
  wp, wsp = _operand(w, "w", (e, n, k))
  act = _activation(activation)
  cp = _counts(row_count, e)
  if eight_bit:
    if out is None:
      out = Fp8Blocks.empty(shape, a.values.device)
      yp, ysp = _pointers(out)
    else:
      yp, ysp = _operand(out, "out", shape)
  else:
    if out is None:
      out = _empty(shape, dtype=torch.bfloat16, device=a.values.device)
      yp = out.data_ptr()
    else:
      yp = _dev(out, "out", torch.bfloat16, shape)
    ysp = None
  if e * r * n == 0:
    return out
  ws_bytes = lib.mesh_moe_fp8_expert_linear_workspace_bytes(e, r, k, n, int(eight_bit))
  ws = _workspace(ws_bytes, a.values) if ws_bytes else None
  with _stage("fp8_linear"):
    _check(lib.mesh_moe_fp8_expert_linear(
        ap, asp, wp, wsp, cp, yp, ysp, e, r, k, n, act,
        None if ws is None else ws.data_ptr(), ws_bytes, _stream()),
           "fp8_expert_linear")
  return out


def expert_linear(a, w, activation="linear", eight_bit=False, row_count=None, out=None):
  """a [E, R, K] and w [E, N, K], 8-bit operands over K -> act(a[e] . w[e]^T) [E, R, N],
  in bfloat16, or (eight_bit) as an 8-bit operand over N.  row_count [E] int32: only the
  first rows of an expert, as many as its count, are multiplied, the others of `out` stay
  as they were (without an `out` they are unspecified)."""
  if not isinstance(a, Fp8Blocks) or not isinstance(w, Fp8Blocks):
    raise MoeHipError("a and w must be Fp8Blocks")
  if len(a.shape) != 3 or len(w.shape) != 3:
    raise MoeHipError("a %s, w %s: expected [E, R, K] and [E, N, K]"
                      % (a.shape, w.shape))
  e, r, k = a.shape
  n = w.shape[1]
  return _linear(a, w, (e, r, k, n), (e, r, n), activation, eight_bit, row_count, out)


def multiplies_exactly(e, r, k, n, eight_bit=False, counted=False):
  """Whether expert_linear (counted: with row_count) of these sizes multiplies exactly and
  adds up in float32.  Otherwise sums lose up to 2^-10 of their products' magnitudes (about
  2^-14 of themselves with normally distributed operands): the matrix instructions for 8
  bits cut the products of 8 neighbouring values off below 2^-13 of the largest.  The faster
  way is taken, so one row's bits may depend on what is beside it."""
  _ints(e, r, k, n)
  return load_library().mesh_moe_fp8_expert_linear_exact(
      e, r, k, n, int(eight_bit), int(counted)) == 1


def dense(x, w, activation=None, eight_bit=False):
  """x [..., K] times a kernel [1, N, K], 8-bit operands over K -> act(x . w^T) [..., N],
  in bfloat16, or (eight_bit) as an 8-bit operand (mtf.layers.dense without bias)."""
  if not isinstance(x, Fp8Blocks) or not isinstance(w, Fp8Blocks):
    raise MoeHipError("x and w must be Fp8Blocks")
  if len(w.shape) != 3:
    raise MoeHipError("w %s: expected [1, N, K]" % (w.shape,))
  lead, k, n = x.shape[:-1], x.shape[-1], w.shape[1]
  rows = 1
  for size in lead:
    rows *= size
  return _linear(x, w, (1, rows, k, n), lead + (n,), activation, eight_bit, None, None)


def expert_linear_backward(a_columns, dy, w_rows=None, relu_mask=None, row_count=None,
                           da=None):
  """The gradients of expert_linear: a_columns [E, K, R] (the columns of a), dy [E, R, N]
  in bfloat16 or float32, w_rows [E, K, N] (the rows of w [E, K, N]; None: da is not
  wanted) -> (da [E, R, K] or None, dw [E, K, N]), both bfloat16.  dy becomes an 8-bit
  operand along N for da and along R for dw.  relu_mask [E, R, N]: the output of a
  product with a ReLU, behind which dy counts as 0 where it is not positive.  row_count
  as given to expert_linear: rows of dy behind it count as zeros, those of `da` stay as
  they were (rows of a behind it are zeros in a_columns, or finite)."""
  lib = load_library()
  if dy.dim() != 3:
    raise MoeHipError("dy %s, expected [E, R, N]" % (tuple(dy.shape),))
  e, r, n = dy.shape
  if not isinstance(a_columns, Fp8Blocks) or len(a_columns.shape) != 3:
    raise MoeHipError("a_columns must be an Fp8Blocks [E, K, R]")
  k = a_columns.shape[1]
  _ints(e, r, k, n)
  code = moe_hip.dtype_code(dy.dtype)
  ap, asp = _operand(a_columns, "a_columns", (e, k, r))
  yp = _dev(dy, "dy")
  mp = (None if relu_mask is None
        else _dev(relu_mask, "relu_mask", dy.dtype, (e, r, n)))
  cp = _counts(row_count, e)
  wp = wsp = None
  if w_rows is not None:
    wp, wsp = _operand(w_rows, "w_rows", (e, k, n))
    if da is None:
      da = _empty((e, r, k), dtype=torch.bfloat16, device=dy.device)
  elif da is not None:
    raise MoeHipError("da needs w_rows")
  dap = None if da is None else _dev(da, "da", torch.bfloat16, (e, r, k))
  if dy.numel() == 0 or k == 0:
    dw = torch.zeros((e, k, n), dtype=torch.bfloat16, device=dy.device)
    return (None if da is None else da.zero_() if r and n == 0 else da), dw
  dw = _empty((e, k, n), dtype=torch.bfloat16, device=dy.device)
  ws_bytes = lib.mesh_moe_fp8_expert_linear_backward_workspace_bytes(
      e, r, k, n, int(da is not None))
  ws = _workspace(ws_bytes, dy)
  with _stage("fp8_linear_backward"):
    _check(lib.mesh_moe_fp8_expert_linear_backward(
        ap, asp, yp, mp, cp, wp, wsp, dap, dw.data_ptr(), e, r, k, n, code,
        ws.data_ptr(), ws_bytes, _stream()), "fp8_expert_linear_backward")
  return da, dw
