"""The 8-bit operands' interface on the CPU: exported symbols, layout of an operand, what
is refused before a launch, and the reference itself."""

import ctypes
import os
import re

import numpy as np
import pytest
import torch

from mesh_amd import fp8_hip
from mesh_amd import moe_hip
from tests import fp8_reference as F

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
  if not os.path.exists(moe_hip.LIB_PATH):
    from mesh_amd.csrc import build
    build.build_library(verbose=False)
  return fp8_hip.load_library()


def test_library_exports_every_declared_symbol(lib):
  header = open(os.path.join(ROOT, "include", "mesh_moe_fp8.h")).read()
  code = re.sub(r"/\*.*?\*/", " ", header, flags=re.DOTALL)
  declared = set(re.findall(r"\b(mesh_moe_fp8_[a-z0-9_]+)\s*\(", code))
  assert declared == set(fp8_hip.EXPORTS)
  for name in declared:
    assert getattr(lib, name) is not None
  version = re.search(r"MESH_MOE_FP8_ABI_VERSION (\d+)", header).group(1)
  assert lib.mesh_moe_fp8_abi_version() == fp8_hip.ABI_VERSION == int(version)


def test_reference_numbers_are_e4m3():
  """The reference's table and rounding against torch's cast."""
  codes = torch.arange(256, dtype=torch.int32).to(torch.uint8)
  np.testing.assert_array_equal(F.e4m3_table(),
                                codes.view(torch.float8_e4m3fn).float().numpy())
  x = torch.cat([torch.linspace(-448, 448, 40001), torch.randn(10000) * 2.0 ** -7])
  want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy() & 127
  np.testing.assert_array_equal(F._codes(np.abs(x.double().numpy())), want)


def test_reference_scales():
  """448 fits the unit, what is above takes the next power of two."""
  x = np.zeros((6, 130))
  x[0, 3], x[1, 3], x[2, 129] = 448, -449, 896
  x[3, 0], x[4, 0] = np.inf, 1e-40
  codes, scales = F.quantize(x)
  assert scales.tolist() == [[127, 10], [128, 10], [10, 128], [127, 10], [10, 10],
                             [10, 10]]
  got = F.value(codes, scales)
  assert got[0, 3] == 448 and got[2, 129] == 896 and got[1, 3] == -448
  assert np.isnan(got[3, :128]).all() and (got[3, 128:] == 0).all()
  assert (got[4] == 0).all()


def test_operand_layout():
  assert [fp8_hip.row_bytes(n) for n in (1, 128, 129, 512)] == [128, 128, 256, 512]
  assert [fp8_hip.scale_bytes(n) for n in (1, 512, 513)] == [4, 4, 8]
  q = fp8_hip.Fp8Blocks.empty((2, 3, 200), "cpu")
  assert q.shape == (2, 3, 200) and q.values.shape == (2, 3, 256)
  assert q.reshape(6).shape == (6, 200)
  for values, scales, n in ((q.values, q.scales, 300), (q.values, q.scales, 0),
                            (q.values, q.scales[..., :2], 200),
                            (q.values.view(torch.uint8), q.scales, 200),
                            (q.values, q.scales.to(torch.int8), 200),
                            (q.values, q.scales[:1], 200)):
    with pytest.raises(ValueError):
      fp8_hip.Fp8Blocks(values, scales, n)


def test_cpu_tensors_are_refused(lib):
  del lib
  x = torch.zeros(4, 256)
  q = fp8_hip.Fp8Blocks.empty((1, 4, 256), "cpu")
  for call in (lambda: fp8_hip.quantize(x), lambda: fp8_hip.dequantize(q),
               lambda: fp8_hip.residual_rms_norm(x, None, torch.ones(256)),
               lambda: fp8_hip.expert_linear(q, q),
               lambda: fp8_hip.dense(q, q),
               lambda: fp8_hip.expert_linear_backward(q, torch.zeros(1, 256, 8))):
    with pytest.raises(moe_hip.MoeHipError, match="GPU tensor"):
      call()
  for call in (lambda: fp8_hip.quantize(x.half()),
               lambda: fp8_hip.dequantize(q, torch.float16)):
    with pytest.raises(moe_hip.MoeHipError, match="dtype"):
      call()
  with pytest.raises(ValueError):
    fp8_hip.quantize(x, rows=False)
  with pytest.raises(ValueError):
    fp8_hip.quantize(x.reshape(-1))
  for call in (lambda: fp8_hip.dense(x, q), lambda: fp8_hip.expert_linear(x, q),
               lambda: fp8_hip.expert_linear_backward(x, torch.zeros(1, 4, 8))):
    with pytest.raises(moe_hip.MoeHipError, match="Fp8Blocks"):
      call()


# addresses that are never read: every call below is refused before a launch
AT = 1 << 20


def _refused(lib, rc, code, words):
  assert rc == code
  text = lib.mesh_moe_last_error().decode()
  assert words in text, text


def test_quantize_refusals(lib):
  call = lib.mesh_moe_fp8_quantize
  ok = [AT, None, None, AT, AT, AT, AT, 2, 3, 4, 1, None]

  def with_(**changes):
    args = list(ok)
    for at, v in changes.items():
      args[int(at[1:])] = v
    return call(*args)
  for change in (dict(_0=None), dict(_4=None), dict(_5=None),
                 dict(_3=None, _4=None, _5=None, _6=None)):
    _refused(lib, with_(**change), -1, "null")
  for change in (dict(_7=0), dict(_8=0), dict(_9=-1), dict(_8=0x7fffffff)):
    _refused(lib, with_(**change), -1, "sizes")
  _refused(lib, with_(_10=7), -1, "dtype")
  for change in (dict(_3=AT + 8), dict(_5=AT + 4), dict(_0=AT + 1)):
    _refused(lib, with_(**change), -2, "16 bytes")
  _refused(lib, with_(_7=1 << 20, _8=1 << 20, _9=1 << 20), -2, "tiles")


def test_dequantize_and_norm_refusals(lib):
  call = lib.mesh_moe_fp8_dequantize
  _refused(lib, call(None, AT, AT, 1, 1, 1, None), -1, "null")
  _refused(lib, call(AT, AT, AT, 0, 1, 1, None), -1, "sizes")
  _refused(lib, call(AT, AT, AT, 1, 0, 1, None), -1, "sizes")
  _refused(lib, call(AT, AT, AT, 1, 1, 2, None), -1, "dtype")
  _refused(lib, call(AT + 8, AT, AT, 1, 1, 1, None), -2, "16 bytes")
  call = lib.mesh_moe_fp8_residual_rms_norm
  ok = [AT, AT, AT, None, AT, None, AT, AT, 4, 8, 1e-6, 1, None]

  def with_(**changes):
    args = list(ok)
    for at, v in changes.items():
      args[int(at[1:])] = v
    return call(*args)
  for change in (dict(_0=None), dict(_1=None), dict(_2=None), dict(_4=None),
                 dict(_6=None), dict(_7=None)):
    _refused(lib, with_(**change), -1, "null")
  for change in (dict(_8=0), dict(_9=0), dict(_8=1 << 31)):
    _refused(lib, with_(**change), -1, "sizes")
  _refused(lib, with_(_11=3), -1, "dtype")
  _refused(lib, with_(_6=AT + 8), -2, "16 bytes")
  _refused(lib, with_(_7=AT + 2), -2, "16 bytes")


def test_linear_refusals(lib):
  call = lib.mesh_moe_fp8_expert_linear
  ok = [AT, AT, AT, AT, None, AT, None, 1, 4, 128, 64, 1, AT, 1 << 40, None]

  def with_(**changes):
    args = list(ok)
    for at, v in changes.items():
      args[int(at[1:])] = v
    return call(*args)
  for at in (0, 1, 2, 3, 5):
    _refused(lib, with_(**{"_%d" % at: None}), -1, "null")
  for change in (dict(_7=0), dict(_8=0), dict(_9=0), dict(_10=0), dict(_9=0x7fffff80)):
    _refused(lib, with_(**change), -1, "sizes")
  _refused(lib, with_(_11=6), -1, "activation")
  for change in (dict(_0=AT + 8), dict(_2=AT + 8), dict(_1=AT + 2), dict(_3=AT + 1),
                 dict(_5=AT + 1), dict(_5=AT + 8, _6=AT), dict(_6=AT + 2),
                 dict(_12=AT + 8)):
    _refused(lib, with_(**change), -2, "16 bytes")
  need = lib.mesh_moe_fp8_expert_linear_workspace_bytes(1, 4, 128, 64, 1)
  if need:
    _refused(lib, with_(_6=AT, _13=need - 1), -1, "workspace")
    _refused(lib, with_(_6=AT, _12=None, _13=need), -1, "workspace")
  assert lib.mesh_moe_fp8_expert_linear_workspace_bytes(0, 4, 128, 64, 1) == 0


def test_linear_backward_refusals(lib):
  call = lib.mesh_moe_fp8_expert_linear_backward
  ok = [AT, AT, AT, None, None, AT, AT, AT, AT, 1, 4, 128, 64, 1, AT, 1 << 40, None]

  def with_(**changes):
    args = list(ok)
    for at, v in changes.items():
      args[int(at[1:])] = v
    return call(*args)
  for at in (0, 1, 2, 5, 6, 8, 14):
    _refused(lib, with_(**{"_%d" % at: None}), -1, "null")
  for at in (9, 10, 11, 12):
    _refused(lib, with_(**{"_%d" % at: 0}), -1, "sizes")
  _refused(lib, with_(_13=5), -1, "dtype")
  for change in (dict(_0=AT + 8), dict(_1=AT + 2), dict(_5=AT + 8), dict(_14=AT + 8),
                 dict(_7=AT + 1), dict(_8=AT + 1), dict(_2=AT + 1)):
    _refused(lib, with_(**change), -2, "16 bytes")
  need = lib.mesh_moe_fp8_expert_linear_backward_workspace_bytes(1, 4, 128, 64, 1)
  assert need > 0
  _refused(lib, with_(_15=need - 1), -1, "workspace")
  assert lib.mesh_moe_fp8_expert_linear_backward_workspace_bytes(1, 0, 128, 64, 1) == 0
  assert ctypes.sizeof(ctypes.c_size_t) == 8


def test_layers_on_8_bit_operands():
  """The same variables and shapes as without, and float32 activations are refused."""
  from mesh_amd import layers as mtf_layers
  from mesh_amd import ops as mtf

  def build(eight_bit, dtype):
    graph = mtf.Graph()
    mesh = mtf.Mesh(graph, "mesh")
    dims = [mtf.Dimension("batch", 2), mtf.Dimension("d_model", 64)]
    x = mtf.import_tf_tensor(mesh, torch.zeros(2, 64, dtype=dtype), mtf.Shape(dims))
    y = mtf_layers.dense(
        x, mtf.Dimension("d_ff", 96), use_bias=False, activation="relu", name="wi",
        variable_dtype=mtf.VariableDType(torch.float32, torch.float32, dtype),
        eight_bit=eight_bit)
    grads = mtf.gradients([y], [x] + [v.outputs[0] for v in graph.trainable_variables])
    return ([(v.name, str(v.shape)) for v in graph.all_variables], str(y.shape), y.dtype,
            [(str(g.shape), g.dtype) for g in grads])
  assert build(True, torch.bfloat16) == build(False, torch.bfloat16)
  with pytest.raises(ValueError, match="bfloat16"):
    build(True, torch.float32)


def test_sizes_that_are_multiplied_exactly(lib):
  """Few rows at most; none of the sizes that a call refuses."""
  del lib
  assert fp8_hip.multiplies_exactly(1, 1, 4096, 16384)
  assert fp8_hip.multiplies_exactly(1, 16, 100, 1000, eight_bit=True, counted=True)
  assert not fp8_hip.multiplies_exactly(64, 6, 4096, 1024)
  for eight_bit in (False, True):
    for counted in (False, True):
      for e in (1, 8, 64):
        for k in (1, 128, 129, 1024, 16384):
          for n in (1, 200, 4096, 65536):
            for r in (129, 500, 8192):
              assert not fp8_hip.multiplies_exactly(e, r, k, n, eight_bit, counted)
  for sizes in ((0, 1, 1, 1), (1, 0, 1, 1), (1, 1, 0, 1), (1, 1, 1, 0)):
    assert not fp8_hip.multiplies_exactly(*sizes)


def test_sizes_beyond_an_int_are_refused(lib):
  """2^32 + 8 would be 8 in a C int: the first 8 values of a row alone."""
  del lib
  many = 2 ** 32 + 128
  one = torch.zeros(1, dtype=torch.bfloat16)
  byte = torch.zeros(1, dtype=torch.uint8)

  def operand(*shape):
    n = shape[-1]
    return fp8_hip.Fp8Blocks(
        byte.view(torch.float8_e4m3fn).expand(shape[:-1] + (fp8_hip.row_bytes(n),)),
        byte.expand(shape[:-1] + (fp8_hip.scale_bytes(n),)), n)
  for call in (
      lambda: fp8_hip.quantize(one.expand(1, many)),
      lambda: fp8_hip.quantize(one.expand(many, 4), rows=False, columns=True),
      lambda: fp8_hip.quantize(one.expand(many, 4, 4)),
      lambda: fp8_hip.dequantize(operand(1, many)),
      lambda: fp8_hip.residual_rms_norm(one.expand(1, many), None, one.expand(many)),
      lambda: fp8_hip.expert_linear(operand(1, 4, many), operand(1, 4, many)),
      lambda: fp8_hip.expert_linear(operand(1, 4, 128), operand(1, many, 128)),
      lambda: fp8_hip.dense(operand(2 ** 16, 2 ** 16, 128), operand(1, 4, 128)),
      lambda: fp8_hip.expert_linear_backward(operand(1, many, 4), one.expand(1, 4, 4)),
      lambda: fp8_hip.expert_linear_backward(operand(1, 4, 4), one.expand(1, 4, many)),
      lambda: fp8_hip.multiplies_exactly(1, 1, 1, many)):
    with pytest.raises(moe_hip.MoeHipError, match="2\\^31"):
      call()


def test_more_than_a_launch_has_is_refused(lib):
  """2^32 threads; a number of tiles that passes 64 bits."""
  for e, r, k in ((1 << 20, 1, 1), (1 << 19, 0x7fffff00, 0x7fffff00)):
    _refused(lib, lib.mesh_moe_fp8_quantize(AT, None, None, AT, AT, AT, AT, e, r, k, 1,
                                            None), -2, "tiles")
  for n, scales in ((0x7fffff00, AT), (0x7fffff00, None), (1 << 30, None)):
    _refused(lib, lib.mesh_moe_fp8_expert_linear(
        AT, AT, AT, AT, None, AT, scales, 1, 4, 128, n, 1, AT, 1 << 40, None),
             -2, "too many tiles")
