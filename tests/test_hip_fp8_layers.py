"""Dense layers on 8-bit operands in graphs: the same numbers, bit for bit, as the calls of
fp8_hip that they stand for (tests/test_hip_fp8.py tests those), in eager runs, gradients
and captured steps, before and after an assignment."""

import pytest
import torch

import mesh_amd as mtf
from mesh_amd import layers as mtf_layers
from mesh_amd.transformer import moe
from mesh_amd.transformer import transformer
from mesh_amd.transformer import transformer_layers

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def hip():
  from mesh_amd import fp8_hip
  fp8_hip.load_library()
  return fp8_hip


def _normal(seed, sizes, std=1.0):
  gen = torch.Generator().manual_seed(seed)
  return torch.randn(sizes, generator=gen) * std


def _graph(b, l, m, f, seed=0, dtype=BF16, master=torch.float32):
  """x -> wi (relu) -> h -> wo -> y, with the variables' values."""
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  dims = [mtf.Dimension("batch", b), mtf.Dimension("length", l),
          mtf.Dimension("d_model", m)]
  x = mtf.import_tf_tensor(mesh, _normal(seed, (b, l, m)).to(dtype), mtf.Shape(dims))
  kind = dict(use_bias=False, eight_bit=True,
              variable_dtype=mtf.VariableDType(master, master, dtype))
  h = mtf_layers.dense(x, mtf.Dimension("d_ff", f), activation="relu", name="wi", **kind)
  y = mtf_layers.dense(h, dims[-1], name="wo", **kind)
  values = {"wi/kernel": _normal(seed + 1, (m, f), m ** -0.5),
            "wo/kernel": _normal(seed + 2, (f, m), f ** -0.5)}
  return graph, mesh, x, h, y, values


def _lower(graph, mesh, values):
  return mtf.Lowering(graph, {mesh: mtf.HipMeshImpl()}, initial_values=values)


def _columns(hip, w):
  return hip.quantize(w.cuda().unsqueeze(0), rows=False, columns=True)


def _forward(hip, x, values):
  a = hip.quantize(x.cuda().reshape(-1, x.shape[-1]))
  h = hip.dense(a, _columns(hip, values["wi/kernel"]), "relu", eight_bit=True)
  y = hip.dense(h, _columns(hip, values["wo/kernel"]))
  return hip.dequantize(h).reshape(x.shape[:-1] + (-1,)), y.reshape(x.shape)


SIZES = [(1, 1, 128, 512), (2, 5, 200, 333), (3, 100, 256, 1024)]


@pytest.mark.parametrize("sizes", SIZES)
@pytest.mark.parametrize("master", [torch.float32, BF16])
def test_forward_and_assignment(hip, sizes, master):
  graph, mesh, x, h, y, values = _graph(*sizes, master=master)
  values = {k: v.to(master) for k, v in values.items()}
  lowering = _lower(graph, mesh, values)
  given = lowering.export_to_tf_tensor(x)
  for step in range(3):
    want_h, want_y = _forward(hip, given, values)
    assert torch.equal(lowering.export_to_tf_tensor(y), want_y)
    assert torch.equal(lowering.export_to_tf_tensor(h), want_h)
    values = {k: v * 1.5 - 0.01 for k, v in values.items()}
    for var, laid_out in lowering.variables.items():
      laid_out.assign(values[var.name])
    given = _normal(10 + step, sizes[:3]).to(BF16)
    lowering.run({x: given})


@pytest.mark.parametrize("sizes", SIZES)
def test_gradients(hip, sizes):
  graph, mesh, x, h, y, values = _graph(*sizes)
  dy = mtf.import_tf_tensor(mesh, _normal(7, sizes[:3]).to(BF16), y.shape)
  variables = [v.outputs[0] for v in graph.trainable_variables]
  grads = mtf.gradients([y], [x] + variables, [dy])
  lowering = _lower(graph, mesh, values)
  b, l, m, f = sizes
  for step in range(2):
    xs, dys = (lowering.export_to_tf_tensor(t) for t in (x, dy))
    wi, wo = (values[k].cuda().unsqueeze(0) for k in ("wi/kernel", "wo/kernel"))
    wi_rows, wi_columns = hip.quantize(wi, rows=True, columns=True)
    wo_rows, wo_columns = hip.quantize(wo, rows=True, columns=True)
    a, a_columns = hip.quantize(xs.reshape(1, -1, m), rows=True, columns=True)
    hs = hip.expert_linear(a, wi_columns, "relu")
    hq, h_columns = hip.quantize(hs, rows=True, columns=True)
    ys = hip.expert_linear(hq, wo_columns)
    dh, dwo = hip.expert_linear_backward(h_columns, dys.reshape(1, -1, m), wo_rows)
    dx, dwi = hip.expert_linear_backward(a_columns, dh, wi_rows, relu_mask=hs)
    for tensor, want in [(h, hs), (y, ys), (grads[0], dx), (grads[1], dwi),
                         (grads[2], dwo)]:
      got = lowering.export_to_tf_tensor(tensor)
      assert torch.equal(got.reshape(-1), want.reshape(-1).to(got.dtype))
    values = {k: v * 0.5 + 0.02 for k, v in values.items()}
    for var, laid_out in lowering.variables.items():
      laid_out.assign(values[var.name])
    lowering.run({x: _normal(20 + step, sizes[:3]).to(BF16)})


def test_hidden_tensor_that_is_read_twice(hip):
  """Another reader of the hidden tensor: it is a bfloat16 tensor then."""
  graph, mesh, x, h, y, values = _graph(2, 40, 256, 512)
  twice = mtf_layers.dense(h, mtf.Dimension("d_out", 64), use_bias=False, name="w2",
                           variable_dtype=mtf.VariableDType(torch.float32, torch.float32,
                                                            BF16))
  values["w2/kernel"] = _normal(5, (512, 64), 0.05)
  lowering = _lower(graph, mesh, values)
  a = hip.quantize(lowering.export_to_tf_tensor(x).reshape(-1, 256))
  hs = hip.dense(a, _columns(hip, values["wi/kernel"]), "relu")
  assert torch.equal(lowering.export_to_tf_tensor(h).reshape(80, 512), hs)
  ys = hip.dense(hip.quantize(hs), _columns(hip, values["wo/kernel"]))
  assert torch.equal(lowering.export_to_tf_tensor(y).reshape(80, 256), ys)
  assert lowering.export_to_tf_tensor(twice).shape == (2, 40, 64)


@pytest.mark.parametrize("with_gradients", [False, True])
def test_captured_step(hip, with_gradients):
  sizes = (2, 33, 256, 640)
  graph, mesh, x, h, y, values = _graph(*sizes)
  outputs = [y]
  if with_gradients:
    dy = mtf.import_tf_tensor(mesh, _normal(7, sizes[:3]).to(BF16), y.shape)
    variables = [v.outputs[0] for v in graph.trainable_variables]
    outputs += mtf.gradients([y], [x] + variables, [dy])
  lowering = _lower(graph, mesh, values)
  step = lowering.capture()
  other = _lower(graph, mesh, values)
  for i in range(3):
    given = _normal(30 + i, sizes[:3]).to(BF16)
    step.replay({x: given})
    got = [lowering.export_to_tf_tensor(t).clone() for t in outputs]
    other.run({x: given})
    for t, value in zip(outputs, got):
      assert torch.equal(value, other.export_to_tf_tensor(t))
    values = {k: v * 0.9 + 0.01 for k, v in values.items()}
    for low in (lowering, other):
      for var, laid_out in low.variables.items():
        laid_out.assign(values[var.name])


@pytest.mark.parametrize("padded", [False, True])
def test_layer_stack(hip, padded):
  """DenseReluDense in a stack with and without 8-bit operands.  Two operands of a root
  mean square error of at most 2^-4 / sqrt(3) each, in two layers one behind the other,
  half of whose result the residual is.  Norms leave as operands: nothing is quantized
  on the way."""
  from mesh_amd import moe_hip
  b, l, m, f = 2, 70, 256, 1024
  results = []
  for eight_bit in (False, True):
    graph = mtf.Graph()
    mesh = mtf.Mesh(graph, "mesh")
    dims = [mtf.Dimension("batch", b), mtf.Dimension("length", l),
            mtf.Dimension("d_model", m)]
    x = mtf.import_tf_tensor(mesh, _normal(1, (b, l, m)).to(BF16), mtf.Shape(dims))
    stack = transformer.make_layer_stack(
        [(transformer_layers.DenseReluDense, dict(hidden_size=f, eight_bit=eight_bit))],
        num_layers=2)
    model = transformer.Unitransformer(stack, d_model=m, name="encoder")
    ids = None
    if padded:
      ids = torch.ones((b, l), dtype=torch.int32)
      ids[:, 50:] = 0
      ids = mtf.import_tf_tensor(mesh, ids, mtf.Shape(dims[:2]))
    y, _ = model.call_layers(
        x, mtf.VariableDType(torch.float32, torch.float32, BF16), mode="eval",
        sequence_id=ids)
    values = {}
    for i, v in enumerate(graph.all_variables):
      sizes = v.shape.to_integer_list
      values[v.name] = (1 + 0.1 * _normal(40 + i, sizes) if len(sizes) == 1
                        else _normal(50 + i, sizes, sizes[0] ** -0.5))
    lowering = _lower(graph, mesh, values)
    first = lowering.export_to_tf_tensor(y).clone()
    with moe_hip.StageTimer() as timer:
      lowering.run()
    assert ("fp8_linear" in timer.totals()) == eight_bit
    assert "fp8_quantize" not in timer.totals()
    assert torch.equal(lowering.export_to_tf_tensor(y), first)
    if eight_bit:
      # the first layer by hand
      norm = [op for op in graph.operations
              if isinstance(op, transformer.RmsNormOperation)][0]
      mask = None
      if padded:
        mask = torch.zeros((b, l), dtype=BF16, device="cuda")
        mask[:, :50] = 1
      given = lowering.export_to_tf_tensor(norm.inputs[0])
      scale = lowering.export_to_tf_tensor(norm.inputs[1])
      _, want = hip.residual_rms_norm(given, None, scale, row_mask=mask)
      reader = norm.mask or norm
      assert torch.equal(lowering.export_to_tf_tensor(reader.outputs[0]),
                         hip.dequantize(want))
      if padded:
        assert torch.equal(lowering.export_to_tf_tensor(norm.outputs[0]),
                           moe_hip.rms_norm(given, scale, 1e-6))
    results.append(first.double())
  exact, got = results
  error = ((got - exact).square().mean() / exact.square().mean()).sqrt()
  assert 0 < error < 2.0 ** -3.5


def _moe(b, l, m, f, e, gating="top_2", activation="relu", eight_bit=True, grads=False):
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  dims = [mtf.Dimension("batch", b), mtf.Dimension("length", l),
          mtf.Dimension("d_model", m)]
  x = mtf.import_tf_tensor(mesh, _normal(1, (b, l, m)).to(BF16), mtf.Shape(dims))
  hparams = moe.HParams()
  moe.set_default_moe_hparams(hparams)
  for name, value in (("moe_gating", gating), ("moe_num_experts", e),
                      ("moe_hidden_size", f), ("moe_group_size", 64),
                      ("moe_min_expert_capacity", 4), ("moe_dropout_rate", 0.0),
                      ("moe_use_experts_attention", False), ("moe_z_loss", None),
                      ("moe_second_policy_train", "all"),
                      ("moe_second_policy_eval", "all"),
                      ("moe_switch_policy_train", "argmax"),
                      ("moe_switch_policy_eval", "argmax"), ("moe_switch_dropout", 0.0),
                      ("moe_switch_temperature", 1.0), ("moe_switch_jitter", 0.0),
                      ("moe_ntlb_top_k", 2), ("moe_eight_bit", eight_bit)):
    setattr(hparams, name, value)
  nonpadding = None
  if gating == "expert_selection":
    nonpadding = mtf.import_tf_tensor(mesh, torch.ones((b, l), dtype=BF16),
                                      mtf.Shape(dims[:2]))
  y, loss = moe.transformer_moe_layer_v1(
      x, dims[-1], hparams, grads, mtf.VariableDType(torch.float32, torch.float32, BF16),
      nonpadding=nonpadding, activation=activation)
  outputs = [y]
  if grads:
    dy = mtf.import_tf_tensor(mesh, _normal(2, (b, l, m)).to(BF16), y.shape)
    outputs += mtf.gradients(
        [y, loss], [x] + [v.outputs[0] for v in graph.trainable_variables], [dy, None])
  values = {}
  for i, v in enumerate(graph.all_variables):
    sizes = v.shape.to_integer_list
    values[v.name] = _normal(60 + i, sizes, sizes[-2] ** -0.5)
  return _lower(graph, mesh, values), x, outputs, values


def _error(got, exact):
  got, exact = got.double(), exact.double()
  return float(((got - exact).square().mean() / exact.square().mean()).sqrt())


@pytest.mark.parametrize("gating", ["top_2", "switch", "ntlb", "expert_selection"])
@pytest.mark.parametrize("activation", ["relu", "gelu"])
def test_experts(hip, gating, activation):
  """The layer against the one in bfloat16: the same routing, and two products whose
  operands are off by at most 2^-4 / sqrt(3) each in the root mean square."""
  del hip
  sizes = (2, 128, 256, 640, 8)
  lowering, x, (y,), _ = _moe(*sizes, gating=gating, activation=activation)
  plain, _, (exact,), _ = _moe(*sizes, gating=gating, activation=activation,
                               eight_bit=False)
  got, want = lowering.export_to_tf_tensor(y), plain.export_to_tf_tensor(exact)
  assert 0 < _error(got, want) < 2.0 ** -3.5
  # (tokens without a slot; single elements may be 0 in one of them)
  assert torch.equal((got == 0).all(-1), (want == 0).all(-1))
  step = lowering.capture()
  given = _normal(9, sizes[:3]).to(BF16)
  lowering.run({x: given})
  eager = lowering.export_to_tf_tensor(y).clone()
  for i in range(4):
    other = _normal(10 + i, sizes[:3]).to(BF16)
    step.replay({x: other})
    replayed = lowering.export_to_tf_tensor(y).clone()
    lowering.run({x: other})
    assert torch.equal(replayed, lowering.export_to_tf_tensor(y))
  step.replay({x: given})
  assert torch.equal(lowering.export_to_tf_tensor(y), eager)


@pytest.mark.parametrize("gating", ["top_2", "switch", "ntlb"])
def test_gradients_of_experts(hip, gating):
  """dx, dwi and dwo against those of the bfloat16 layer; the router's gradient reads the
  experts' outputs, which are as far apart as the products make them.  (Where the two
  hidden tensors differ in sign the masks do: 2^-2.5 instead of 2^-3.5.)"""
  del hip
  sizes = (2, 128, 256, 640, 8)
  lowering, x, got, values = _moe(*sizes, gating=gating, grads=True)
  plain, _, exact, _ = _moe(*sizes, gating=gating, grads=True, eight_bit=False)
  assert len(got) == len(exact) == 5
  for a, b in zip(got, exact):
    assert a.shape.to_integer_list == b.shape.to_integer_list and a.dtype == b.dtype
    assert 0 < _error(lowering.export_to_tf_tensor(a),
                      plain.export_to_tf_tensor(b)) < 2.0 ** -2.5
  for low in (lowering, plain):
    for var, laid_out in low.variables.items():
      laid_out.assign(values[var.name] * 0.8)
    low.run()
  for a, b in zip(got, exact):
    assert 0 < _error(lowering.export_to_tf_tensor(a),
                      plain.export_to_tf_tensor(b)) < 2.0 ** -2.5


def test_experts_refusals(hip):
  del hip
  with pytest.raises(NotImplementedError, match="8-bit"):
    _moe(1, 64, 64, 64, 4, activation=["relu", "linear"])
  with pytest.raises(NotImplementedError, match="8-bit"):
    _moe(1, 64, 64, 64, 4, activation="gelu", grads=True)


def test_moe_layer_in_a_stack(hip):
  del hip
  results = []
  for layer in (moe.MoE1D, moe.EightBitMoE1D):
    graph = mtf.Graph()
    mesh = mtf.Mesh(graph, "mesh")
    dims = [mtf.Dimension("batch", 2), mtf.Dimension("length", 96),
            mtf.Dimension("d_model", 128)]
    x = mtf.import_tf_tensor(mesh, _normal(1, (2, 96, 128)).to(BF16), mtf.Shape(dims))
    stack = transformer.make_layer_stack(
        [(layer, dict(num_experts=4, hidden_size=384, group_size=64,
                      second_policy_eval="all"))], num_layers=1)
    model = transformer.Unitransformer(stack, d_model=128, name="encoder")
    y, losses = model.call_layers(
        x, mtf.VariableDType(torch.float32, torch.float32, BF16), mode="eval")
    values = {}
    for i, v in enumerate(graph.all_variables):
      sizes = v.shape.to_integer_list
      values[v.name] = (torch.ones(sizes) if len(sizes) == 1
                        else _normal(70 + i, sizes, sizes[-2] ** -0.5))
    lowering = _lower(graph, mesh, values)
    results.append((lowering.export_to_tf_tensor(y),
                    [float(lowering.export_to_tf_tensor(t)) for t in losses]))
  assert results[0][1] == results[1][1]
  assert 0 < _error(results[1][0], results[0][0]) < 2.0 ** -3.5


def test_forward_with_and_without_gradients(hip):
  """With a gradient to follow, a norm and a hidden tensor are rounded to bfloat16 before
  they are to 8 bits, the norm in each of its three steps.  A rounding moves a value by
  2^-9 of it at most, so with a probability of at most 2 * 2^-9 / 2^-4 over a border to
  the next 8-bit one, 2^-3 of it away at most: 2^-2 * 2^-3 in the root mean square behind
  the hidden tensor, sqrt(3) times that behind the norm."""
  del hip
  results = []
  for grads in (False, True):
    graph = mtf.Graph()
    mesh = mtf.Mesh(graph, "mesh")
    dims = [mtf.Dimension("batch", 2), mtf.Dimension("length", 70),
            mtf.Dimension("d_model", 256)]
    x = mtf.import_tf_tensor(mesh, _normal(1, (2, 70, 256)).to(BF16), mtf.Shape(dims))
    with mtf.variable_scope("norm"):
      scale = mtf.get_variable(
          mesh, "scale", mtf.Shape(dims[-1:]),
          dtype=mtf.VariableDType(torch.float32, torch.float32, BF16))
    norm = transformer.RmsNormOperation(x, scale, 1e-6).outputs[0]
    kind = dict(use_bias=False, eight_bit=True,
                variable_dtype=mtf.VariableDType(torch.float32, torch.float32, BF16))
    h = mtf_layers.dense(norm, mtf.Dimension("d_ff", 1024), name="wi", **kind)
    y = mtf_layers.dense(h, dims[-1], name="wo", **kind)
    if grads:
      mtf.gradients([y], [v.outputs[0] for v in graph.trainable_variables],
                    [mtf.import_tf_tensor(mesh, _normal(2, (2, 70, 256)).to(BF16),
                                          y.shape)])
    values = {"norm/scale": 1 + 0.1 * _normal(3, (256,)),
              "wi/kernel": _normal(4, (256, 1024), 1.0 / 16),
              "wo/kernel": _normal(5, (1024, 256), 1.0 / 32)}
    lowering = _lower(graph, mesh, values)
    lowering.run()
    results.append(lowering.export_to_tf_tensor(y))
  assert 0 < _error(results[1], results[0]) < (1 + 3 ** 0.5) * 2.0 ** -5


@pytest.mark.parametrize("padded", [False, True])
def test_training_a_layer_stack(hip, padded):
  """DenseReluDense layers with norms, residual sums, a padding mask and gradients: every
  8-bit layer and its gradients are what the calls make of the tensors that reach them,
  in an eager step and in recorded ones."""
  b, l, m, f = 2, 70, 256, 1024
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  dims = [mtf.Dimension("batch", b), mtf.Dimension("length", l),
          mtf.Dimension("d_model", m)]
  x = mtf.import_tf_tensor(mesh, _normal(1, (b, l, m)).to(BF16), mtf.Shape(dims))
  stack = transformer.make_layer_stack(
      [(transformer_layers.DenseReluDense, dict(hidden_size=f, eight_bit=True))],
      num_layers=2)
  model = transformer.Unitransformer(stack, d_model=m, name="encoder")
  ids = None
  if padded:
    ids = torch.ones((b, l), dtype=torch.int32)
    ids[:, 50:] = 0
    ids = mtf.import_tf_tensor(mesh, ids, mtf.Shape(dims[:2]))
  y, _ = model.call_layers(
      x, mtf.VariableDType(torch.float32, torch.float32, BF16), mode="train",
      sequence_id=ids)
  dy = mtf.import_tf_tensor(mesh, _normal(2, (b, l, m)).to(BF16), y.shape)
  grads = mtf.gradients([y], [x] + [v.outputs[0] for v in graph.trainable_variables],
                        [dy])
  values = {}
  for i, v in enumerate(graph.all_variables):
    sizes = v.shape.to_integer_list
    values[v.name] = (1 + 0.1 * _normal(40 + i, sizes) if len(sizes) == 1
                      else _normal(50 + i, sizes, sizes[0] ** -0.5))
  lowering = _lower(graph, mesh, values)
  layers = [op for op in graph.operations if isinstance(op, mtf_layers.DenseOperation)]
  backward = [op for op in graph.operations
              if isinstance(op, mtf_layers.DenseGradOperation)]
  assert len(layers) == len(backward) == 4 and all(op.eight_bit for op in layers)

  def check():
    got = lowering.export_to_tf_tensor
    for op in layers:
      xs = got(op.inputs[0])
      a, a_columns = hip.quantize(xs.reshape(1, -1, xs.shape[-1]), columns=True)
      w = hip.quantize(lowering.variables[op.inputs[1].operation].master.unsqueeze(0),
                       columns=True)
      want = hip.expert_linear(a, w[1], op._activation)
      ys = got(op.outputs[0])
      assert torch.equal(ys, want.reshape(ys.shape))
      back = [g for g in backward if g.inputs[1] is op.inputs[0]]
      assert len(back) == 1
      dx, dw = hip.expert_linear_backward(
          a_columns, got(back[0].inputs[0]).reshape(want.shape), w[0],
          relu_mask=want if op._activation == "relu" else None)
      for tensor, value in zip(back[0].outputs, (dx, dw)):
        value = value.to(tensor.dtype)
        assert torch.equal(got(tensor).reshape(-1), value.reshape(-1))
    return [got(t).clone() for t in [y] + grads]
  lowering.run()
  first = check()
  assert all(torch.isfinite(t).all() for t in first)
  step = lowering.capture()
  for i in range(3):
    given = _normal(3 + i, (b, l, m)).to(BF16)
    step.replay({x: given})
    replayed = check()
    lowering.run({x: given, dy: lowering.export_to_tf_tensor(dy)})
    for t, value in zip([y] + grads, replayed):
      assert torch.equal(lowering.export_to_tf_tensor(t), value)
