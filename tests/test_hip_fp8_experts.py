"""Experts of a layer on 8-bit operands, bit for bit against the calls of fp8_hip that they
stand for (tests/test_hip_fp8.py tests those).  The rows of an expert are gathered and put
together here, from the router's record; gating, and the way from the slots' gradients to
the tokens' and the router's, are the calls that the bfloat16 layer makes."""

import pytest
import torch

import mesh_amd as mtf
from mesh_amd.transformer import moe

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


class _Layer(object):
  """transformer_moe_layer_v1 with 8-bit experts and, with `grads`, the gradients of
  <y, dy> + loss.  unused: an expert that no token chooses (the first feature of every
  token is 4, and its router weight -50)."""

  def __init__(self, gating, activation, b, l, m, f, e, group, factor, grads, unused=None):
    graph = mtf.Graph()
    mesh = mtf.Mesh(graph, "mesh")
    dims = [mtf.Dimension("batch", b), mtf.Dimension("length", l),
            mtf.Dimension("d_model", m)]
    self.sizes = (b, l, m)
    self.x = mtf.import_tf_tensor(mesh, self.tokens(1), mtf.Shape(dims))
    hparams = moe.HParams()
    moe.set_default_moe_hparams(hparams)
    for name, value in (
        ("moe_gating", gating), ("moe_num_experts", e), ("moe_hidden_size", f),
        ("moe_group_size", group), ("moe_min_expert_capacity", 4),
        ("moe_capacity_factor_train", factor), ("moe_capacity_factor_eval", factor),
        ("moe_dropout_rate", 0.0), ("moe_use_experts_attention", False),
        ("moe_z_loss", None), ("moe_second_policy_train", "all"),
        ("moe_second_policy_eval", "all"), ("moe_switch_policy_train", "argmax"),
        ("moe_switch_policy_eval", "argmax"), ("moe_switch_dropout", 0.0),
        ("moe_switch_temperature", 1.0), ("moe_switch_jitter", 0.0),
        ("moe_ntlb_top_k", 2), ("moe_eight_bit", True)):
      setattr(hparams, name, value)
    nonpadding = None
    if gating == "expert_selection":
      nonpadding = mtf.import_tf_tensor(mesh, torch.ones((b, l), dtype=BF16),
                                        mtf.Shape(dims[:2]))
    y, loss = moe.transformer_moe_layer_v1(
        self.x, dims[-1], hparams, grads,
        mtf.VariableDType(torch.float32, torch.float32, BF16), nonpadding=nonpadding,
        activation=activation)
    self.outputs = [y]
    if grads:
      self.dy = mtf.import_tf_tensor(mesh, _normal(2, (b, l, m)).to(BF16), y.shape)
      self.outputs += mtf.gradients(
          [y, loss], [self.x] + [v.outputs[0] for v in graph.trainable_variables],
          [self.dy, None])
    values = {}
    for i, v in enumerate(graph.all_variables):
      sizes = v.shape.to_integer_list
      values[v.name] = _normal(60 + i, sizes, sizes[-2] ** -0.5)
      if unused is not None and sizes == [m, e]:
        values[v.name][0, unused] = -50.0
    self.lowering = mtf.Lowering(graph, {mesh: mtf.HipMeshImpl()}, initial_values=values)
    self.op = [op for op in graph.operations if isinstance(op, moe.MoEV1Operation)][0]
    self.grad_op = ([op for op in graph.operations
                     if isinstance(op, moe.MoEV1GradOperation)] or [None])[0]

  def tokens(self, seed):
    x = _normal(seed, self.sizes)
    x[..., 0] = 4.0
    return x.to(BF16)

  def get(self, tensor):
    return self.lowering.export_to_tf_tensor(tensor)

  def by_hand(self, hip):
    """The outputs, and the rows of each expert that are multiplied (None: all)."""
    from mesh_amd import moe_hip
    op, gating = self.op, self.op._gating
    _, g, s, m = op.inputs[0].shape.to_integer_list
    e, c = op._num_experts, op._capacity
    xg = self.get(self.x).reshape(g, s, m)
    variables = [self.lowering.variables[t.operation] for t in op.inputs[1:4]]
    wg, wi, wo = (v.master.reshape(-1, *v.master.shape[-2:]) for v in variables)
    importance = (torch.ones((g, s), dtype=BF16, device="cuda")
                  if op._has_importance else None)
    wg_packed = moe_hip.pack_weights(wg, BF16)
    wg = wg.to(BF16)
    r, logits = gating.route(xg.reshape(1, g * s, m), wg, wg_packed, s, e, c, importance,
                             want_logits=True)
    by_slot = isinstance(r, moe_hip.SlotRouting)
    count = offsets = None
    expert_in = torch.zeros((e, g * c, m), dtype=BF16, device="cuda")
    if by_slot:
      expert_in = moe_hip.slot_dispatch(xg, r).reshape(e, g * c, m)
    else:
      used = r.fill.t().long()
      first = (torch.arange(g, device="cuda") * c).expand(e, g)
      if op._counts_rows(g, s):
        count = used.sum(1).int()
        first = used.cumsum(1) - used
        offsets = first.int().contiguous()
      token, choice = (r.kept != 0).reshape(g * s, 2).nonzero(as_tuple=True)
      expert, pos, gate = (t.reshape(g * s, 2)[token, choice]
                           for t in (r.idx.long(), r.pos.long(), r.gate))
      row = first[expert, token // s] + pos
      expert_in[expert, row] = torch.where((gate.to(BF16) != 0)[:, None],
                                           xg.reshape(g * s, m)[token], 0)
    counted = {"row_count": count}
    wi_rows, wi_columns = hip.quantize(wi.contiguous(), rows=True, columns=True)
    wo_rows, wo_columns = hip.quantize(wo.contiguous(), rows=True, columns=True)
    a, a_columns = hip.quantize(expert_in, rows=True, columns=True)
    n = self.outputs[0].shape.to_integer_list[-1]
    relu = op._activation == "relu"
    if self.grad_op is None:
      h = hip.expert_linear(a, wi_columns, op._activation, eight_bit=True, **counted)
    else:
      f = wi.shape[-1]
      h_values = torch.zeros((e, g * c, f), dtype=BF16, device="cuda")
      hip.expert_linear(a, wi_columns, op._activation, out=h_values, **counted)
      h, h_columns = hip.quantize(h_values, rows=True, columns=True)
    ys = torch.zeros((e, g * c, n), dtype=BF16, device="cuda")
    hip.expert_linear(h, wo_columns, out=ys, **counted)
    if by_slot:
      out = moe_hip.slot_combine(ys.reshape(e, g, c, n), r, s)
    else:
      # w0 * y0 + w1 * y1, each operation rounded to float32, the sum to bfloat16
      parts = torch.zeros((2, g * s, n), device="cuda")
      weight = gate.to(BF16).float()[:, None]
      parts[choice, token] = torch.where(weight != 0, ys[expert, row].float() * weight, 0)
      out = (parts[0] + parts[1]).to(BF16)
    outputs = [out.reshape(self.get(self.outputs[0]).shape)]
    if self.grad_op is None:
      return outputs, count
    dout = self.get(self.dy).reshape(g, s, n)
    y4 = ys.reshape(e, g, c, n)
    compact = {} if offsets is None else {"row_offsets": offsets}
    if by_slot:
      dys, dgate = moe_hip.slot_combine_backward(dout, y4, r)
    else:
      dys, dgate = moe_hip.combine_backward(dout, y4, r, **compact)
    dys = dys.reshape(e, g * c, n)
    if count is not None:
      # (behind the count lies what was there before)
      dead = torch.arange(g * c, device="cuda") >= count[:, None]
      dys = torch.where(dead[..., None], 0, dys)
    dh = torch.zeros_like(h_values)
    _, dwo = hip.expert_linear_backward(h_columns, dys, wo_rows, da=dh, **counted)
    dxe = torch.zeros_like(expert_in)
    _, dwi = hip.expert_linear_backward(a_columns, dh, wi_rows, da=dxe,
                                        relu_mask=h_values if relu else None, **counted)
    d_loss = self.get(self.grad_op.inputs[5]).reshape(1).float()
    if by_slot:
      dlogits = moe_hip.expert_choice_backward(logits, r, dgate, d_loss, 1.0,
                                               importance=importance)
      back = moe_hip.slot_dispatch_backward
    else:
      dlogits = moe_hip.gating_backward(
          logits, r, dgate, d_loss, 1.0, router=gating.router,
          top_k=getattr(gating, "top_k", 0), importance=importance,
          use_second_place_loss=gating.use_second_place_loss,
          softmax_dtype=BF16 if gating.router == "ntlb" else torch.float32)
      back = moe_hip.dispatch_backward
    dx = back(dxe.reshape(e, g, c, m), r, s, dlogits, wg_packed.reshape(e, m),
              w_gate=wg.reshape(m, e).contiguous(), **compact)
    dwg = moe_hip.router_backward_weights(xg.reshape(g * s, m),
                                          dlogits.reshape(g * s, e))
    return outputs + [dx, dwg, dwi, dwo], count

  def check(self, hip):
    want, count = self.by_hand(hip)
    assert len(want) == len(self.outputs)
    for tensor, value in zip(self.outputs, want):
      got = self.get(tensor)
      assert torch.isfinite(got).all()
      assert torch.equal(got.reshape(-1), value.reshape(-1).to(got.dtype)), tensor
    return count


# top-2 with more slots than choices (its rows are counted) and with fewer; odd groups
# and widths, an expert without tokens, rows per expert that are and are not whole tiles
CASES = [("top_2", (4, 64, 256, 384, 64, 64, 64.0)),
         ("top_2", (3, 50, 200, 333, 120, 50, 120.0)),
         ("top_2", (5, 33, 131, 257, 100, 33, 100.0)),
         ("top_2", (2, 2048, 256, 640, 8, 1024, 4.0)),
         ("top_2", (2, 128, 256, 640, 8, 64, 2.0)),
         ("top_2", (3, 50, 200, 333, 6, 50, 1.25)),
         ("switch", (2, 128, 256, 640, 8, 64, 1.25)),
         ("switch", (3, 50, 131, 333, 6, 50, 2.0)),
         ("ntlb", (2, 128, 200, 257, 8, 64, 1.25)),
         ("expert_selection", (2, 128, 256, 640, 8, 64, 1.25)),
         ("expert_selection", (3, 50, 131, 333, 6, 50, 2.0))]


@pytest.mark.parametrize("grads", [False, True])
@pytest.mark.parametrize("activation", ["relu", "linear"])
@pytest.mark.parametrize("gating,sizes", CASES)
def test_experts_bit_for_bit(hip, gating, sizes, activation, grads):
  unused = None if gating == "expert_selection" else 1
  layer = _Layer(gating, activation, *sizes, grads=grads, unused=unused)
  count = layer.check(hip)
  slots_per_choice = layer.op._capacity * sizes[4] / (2.0 * sizes[5])
  assert (count is not None) == (gating in ("switch", "ntlb") or
                                 (gating == "top_2" and slots_per_choice > 1.25))
  if count is not None:
    assert count[1] == 0 and count.sum() > 0
  # another step, with other weights, in memory that is NaN where nothing is written
  poison = [torch.full((1 << 24,), float("nan"), device="cuda") for _ in range(8)]
  del poison
  for var, laid_out in layer.lowering.variables.items():
    laid_out.assign(laid_out.master * 0.75)
  layer.lowering.run({layer.x: layer.tokens(5)})
  layer.check(hip)


@pytest.mark.parametrize("gating,sizes", CASES[1:4] + CASES[6:7] + CASES[9:10])
def test_recorded_training_step(hip, gating, sizes):
  """Replays with other tokens and weights, eager work between them."""
  layer = _Layer(gating, "relu", *sizes, grads=True)
  step = layer.lowering.capture()
  for i in range(3):
    step.replay({layer.x: layer.tokens(10 + i)})
    layer.check(hip)
    replayed = [layer.get(t).clone() for t in layer.outputs]
    layer.lowering.run({layer.x: layer.tokens(10 + i)})
    for tensor, value in zip(layer.outputs, replayed):
      assert torch.equal(layer.get(tensor), value)
    for var, laid_out in layer.lowering.variables.items():
      laid_out.assign(laid_out.master * 0.9)


@pytest.mark.parametrize("gating,sizes", CASES[:1] + CASES[3:5] + CASES[6:7])
def test_forward_with_and_without_gradients(hip, gating, sizes):
  """With a gradient to follow the hidden tensor is rounded to bfloat16 before it is to 8
  bits.  That moves a value by 2^-9 of it at most, so with a probability of at most 2 *
  2^-9 / 2^-4 over a border to the next one, a step of at most 2^-3 of it away: 2^-2 *
  2^-3 in the root mean square."""
  del hip
  outs = []
  for grads in (False, True):
    layer = _Layer(gating, "linear", *sizes, grads=grads)
    outs.append(layer.get(layer.outputs[0]).double())
  error = ((outs[1] - outs[0]).square().mean() / outs[0].square().mean()).sqrt()
  assert 0 < error < 2.0 ** -5
