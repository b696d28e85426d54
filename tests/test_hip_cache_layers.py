"""Decoding with states in pages through the layers: "first_part" and "incremental" mode
against the full forward pass, steps recorded into a HIP graph, and the operations against
the calls."""

import numpy as np
import pytest
import torch

import mesh_amd as mtf
from mesh_amd import cache_hip
from mesh_amd.transformer import attention
from mesh_amd.transformer import moe
from mesh_amd.transformer import transformer
from mesh_amd.transformer import transformer_layers

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HEADS, WIDTH, PAGE = 4, 16, 8
MODEL = 64


def _model(mesh, shared_kv, relative):
  att = dict(num_heads=HEADS, key_value_size=WIDTH, shared_kv=shared_kv,
             relative_attention_type=relative, relative_attention_num_buckets=8)
  stack = transformer.make_layer_stack(
      [(transformer_layers.SelfAttention, att),
       (moe.MoE1D, dict(num_experts=4, hidden_size=96, group_size=32,
                        second_policy_eval="all", capacity_factor_eval=4.0)),
       (transformer_layers.SelfAttention, att),
       (transformer_layers.DenseReluDense, dict(hidden_size=128))],
      num_layers=1, block_scope=False)
  del mesh
  return transformer.Unitransformer(stack, d_model=MODEL, name="decoder",
                                    autoregressive=True)


def _states(b, length, kind, shared_kv, layers=2):
  """A PagedState per attention layer; one table, pages in no order."""
  columns = -(-length // PAGE)
  order = torch.randperm(b * columns + 3, generator=torch.Generator().manual_seed(1))
  table = order[:b * columns].reshape(b, columns).int().cuda()
  return [attention.PagedState(
      cache_hip.PagedCache.empty(b * columns + 3, PAGE, HEADS, WIDTH, kind, "cuda",
                                 shared_kv=shared_kv), table) for _ in range(layers)]


def _initial_values(graph, rng):
  def value(v):
    shape = v.shape.to_integer_list
    if v.name.endswith("scale"):
      return (1 + 0.1 * rng.standard_normal(shape)).astype(np.float32)
    if v.name.endswith("relative_attention_bias"):
      return rng.standard_normal(shape).astype(np.float32)
    return (rng.standard_normal(shape) / np.sqrt(shape[-2])).astype(np.float32)
  return {v.name: value(v) for v in graph.all_variables}


@pytest.mark.parametrize("shared_kv,relative", [(False, None), (True, None),
                                                (False, "bias"), (True, "bias_shared")])
@pytest.mark.parametrize("act_dtype", [torch.float32, torch.bfloat16])
def test_decoding_in_pages_matches_the_full_forward(act_dtype, shared_kv, relative):
  """What a step gives at a position is what the full pass over the row gives there (the
  tolerances are those of decoding with whole states)."""
  b, length, first = 3, 27, 19
  rng = np.random.default_rng(3)
  x = torch.from_numpy(rng.standard_normal((b, length, MODEL)).astype(np.float32)).to(
      act_dtype)
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  batch, len_dim, model_dim = (mtf.Dimension("batch", b), mtf.Dimension("length", length),
                               mtf.Dimension("d_model", MODEL))
  vdt = mtf.VariableDType(torch.float32, torch.float32, act_dtype)
  model = _model(mesh, shared_kv, relative)
  whole = mtf.import_tf_tensor(mesh, x, mtf.Shape([batch, len_dim, model_dim]))
  y_full, _ = model.call_layers(whole, vdt, mode="eval")
  known = x.clone()
  known[:, first:] = 0
  states = _states(b, length, act_dtype, shared_kv)
  new_states = []
  y_first, _ = model.call_layers(
      mtf.import_tf_tensor(mesh, known, mtf.Shape([batch, len_dim, model_dim])), vdt,
      mode="first_part", states=states, new_states=new_states, reuse=True)
  assert new_states == states
  steps = []
  for p in range(first, length):
    token = mtf.import_tf_tensor(mesh, x[:, p].contiguous(),
                                 mtf.Shape([batch, model_dim]))
    position = mtf.import_tf_tensor(mesh, torch.full((b,), p, dtype=torch.int32),
                                    mtf.Shape([batch]))
    steps.append(model.call_layers(token, vdt, mode="incremental", position=position,
                                   states=states, length_dim=len_dim)[0])
  lowering = mtf.Lowering(graph, {mesh: mtf.HipMeshImpl()},
                          initial_values=_initial_values(graph, rng))
  tol = (dict(rtol=2e-4, atol=2e-4) if act_dtype == torch.float32
         else dict(rtol=5e-2, atol=5e-2))
  want = lowering.export_to_tf_tensor(y_full).float()
  torch.testing.assert_close(
      lowering.export_to_tf_tensor(y_first).float()[:, :first], want[:, :first], **tol)
  for p, step in zip(range(first, length), steps):
    torch.testing.assert_close(lowering.export_to_tf_tensor(step).float(), want[:, p],
                               **tol)


@pytest.mark.parametrize("kind", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("relative", [False, True])
def test_operations_are_the_calls(kind, relative):
  """The operations' results and pages, bit for bit, over two runs of a step (the second
  from a recorded graph, between eager work)."""
  b, length = 3, 40
  heads, width = HEADS, WIDTH
  gen = torch.Generator(device="cuda").manual_seed(4)
  mk = lambda *s: torch.randn(s, generator=gen, device="cuda").bfloat16()
  state, other = (_states(b, length, kind, False, 1)[0] for _ in range(2))
  for s in (state, other):                   # (rows that nothing writes)
    for buffer in (s.cache.k_pages, s.cache.v_pages, s.cache.k_scales, s.cache.v_scales):
      if buffer is not None:
        buffer.view(torch.uint8).fill_(60)
  rows = [mk(b, length, heads * width) for _ in range(2)]
  values = mk(heads, 8)
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  batch, len_dim, chan = (mtf.Dimension("batch", b), mtf.Dimension("length", length),
                          mtf.Dimension("heads", heads * width))
  t = lambda a, *dims: mtf.import_tf_tensor(mesh, a, mtf.Shape(dims))
  attention.PagedWriteOperation(t(rows[0], batch, len_dim, chan),
                                t(rows[1], batch, len_dim, chan), state, heads)
  mtf.Lowering(graph, {mesh: mtf.HipMeshImpl()})
  cache_hip.write(other.cache, rows[0], rows[1], other.table,
                  torch.zeros(b, dtype=torch.int32, device="cuda"))
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  q, k, v = (mk(b, heads * width) for _ in range(3))
  position = torch.tensor([30, 0, 17], dtype=torch.int32, device="cuda")
  feeds = [t(q, batch, chan), t(k, batch, chan), t(v, batch, chan), t(position, batch)]
  rel = t(values, mtf.Dimension("h", heads), mtf.Dimension("buckets", 8))
  out = attention.PagedDecodeOperation(
      feeds[0], feeds[1], feeds[2], feeds[3], state, heads,
      relative_values=rel if relative else None).outputs[0]
  lowering = mtf.Lowering(graph, {mesh: mtf.HipMeshImpl()})
  bias = (values, attention.relative_bucket_table(40, False, 8, values.device))

  def check(q, k, v, position):
    want = cache_hip.attention(q, other.cache, other.table, position, k_new=k, v_new=v,
                               relative_bias=bias if relative else None)
    assert torch.equal(lowering.export_to_tf_tensor(out), want)
    for name in ("k_pages", "v_pages", "k_scales", "v_scales"):
      a, c = getattr(state.cache, name), getattr(other.cache, name)
      assert a is None or torch.equal(a.view(torch.uint8), c.view(torch.uint8))
  check(q, k, v, position)
  recorded = lowering.capture()
  for i in range(4):
    q, k, v = (mk(b, heads * width) for _ in range(3))
    position = position + torch.tensor([1, 7, 2], dtype=torch.int32, device="cuda")
    if i == 2:                               # a sequence whose last page is taken away
      for s in (state, other):
        s.table[0, -1] = -1
    recorded.replay(dict(zip(feeds, (q, k, v, position))))
    check(q, k, v, position)
    torch.empty(1 << 20, device="cuda").normal_()


@pytest.mark.parametrize("buckets,bidirectional,memory", [
    (300, False, 150), (600, True, 150), (320, False, 150), (254, False, 150),
    # (and distances for which the formula has no bucket)
    (300, False, 400), (258, False, 400), (512, True, 300)])
@pytest.mark.parametrize("act_dtype", [torch.float32, torch.bfloat16])
def test_biases_of_many_buckets(act_dtype, buckets, bidirectional, memory):
  """More buckets than the distances that usually differ: a position far back has the bias
  that it has on whole states."""
  b = 3
  rng, gen = np.random.default_rng(6), torch.Generator(device="cuda").manual_seed(6)
  mk = lambda *s: torch.randn(s, generator=gen, device="cuda").to(act_dtype)
  state = _states(b, memory, act_dtype, False, 1)[0]
  assert state.table.shape[-1] * PAGE >= memory
  old = [mk(b, memory, HEADS * WIDTH) for _ in range(2)]
  cache_hip.write(state.cache, old[0], old[1], state.table,
                  torch.zeros(b, dtype=torch.int32, device="cuda"))
  q, k, v = (mk(b, HEADS * WIDTH) for _ in range(3))
  q *= WIDTH ** -0.5
  values = torch.from_numpy(rng.standard_normal((HEADS, buckets)).astype(np.float32)).cuda()
  position = torch.tensor([memory - 1, 128, memory - 11], dtype=torch.int32, device="cuda")
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  batch, length, chan = (mtf.Dimension("batch", b), mtf.Dimension("memory_length", memory),
                         mtf.Dimension("heads", HEADS * WIDTH))
  t = lambda a, *dims: mtf.import_tf_tensor(mesh, a, mtf.Shape(dims))
  feeds = [t(q, batch, chan), t(k, batch, chan), t(v, batch, chan)]
  states = [t(x, batch, length, chan) for x in old]
  at = t(position, batch)
  bias = dict(relative_values=t(values.to(act_dtype), mtf.Dimension("h", HEADS),
                                mtf.Dimension("buckets", buckets)),
              relative_bidirectional=bidirectional)
  on_pages = attention.PagedDecodeOperation(*feeds, at, state, HEADS, **bias).outputs[0]
  whole = attention.AttentionDecodeOperation(*feeds, *states, at, HEADS, **bias).outputs[0]
  lowering = mtf.Lowering(graph, {mesh: mtf.HipMeshImpl()})
  got, want = (lowering.export_to_tf_tensor(x).float() for x in (on_pages, whole))
  # (bfloat16: weights and the result are rounded, each by half a step of 2^-8, and the sum of
  # weights times |v| is below 2, so each is off by 2 * 2^-8 * 2 + 2^-8 |out| at most, which
  # is 0.016 and 0.4 %, twice.  float32: logits below 16 and up to 400 terms, each side off
  # by 2 * 2^-24 * (17 * 16 + 10 * 16 + 8 + 400) * 2 = 2e-4 at most.)
  torch.testing.assert_close(
      got, want, **(dict(rtol=0, atol=4e-4) if act_dtype == torch.float32
                    else dict(rtol=5e-2, atol=5e-2)))
  # and the bits of the call with the whole table
  table = attention.relative_bucket_table(memory + 1, bidirectional, buckets, values.device)
  assert torch.equal(got, cache_hip.attention(
      q, state.cache, state.table, position,
      relative_bias=(values.to(act_dtype), table)).float())


@pytest.mark.parametrize("act_dtype", [torch.float32, torch.bfloat16])
def test_decoding_with_pages_shared_by_sequences(act_dtype):
  """Three sequences of which two begin with the same 16 tokens: the first part's table names
  their two pages for one of them, the steps' table for both."""
  b, length, first, shared = 3, 27, 19, 2 * PAGE
  rng = np.random.default_rng(8)
  x = torch.from_numpy(rng.standard_normal((b, length, MODEL)).astype(np.float32)).to(
      act_dtype)
  x[2, :shared] = x[0, :shared]
  graph = mtf.Graph()
  mesh = mtf.Mesh(graph, "mesh")
  batch, len_dim, model_dim = (mtf.Dimension("batch", b), mtf.Dimension("length", length),
                               mtf.Dimension("d_model", MODEL))
  vdt = mtf.VariableDType(torch.float32, torch.float32, act_dtype)
  model = _model(mesh, False, "bias")
  t = lambda a: mtf.import_tf_tensor(mesh, a, mtf.Shape([batch, len_dim, model_dim]))
  y_full, _ = model.call_layers(t(x), vdt, mode="eval")
  known = x.clone()
  known[:, first:] = 0
  begin = _states(b, length, act_dtype, False)
  spare = begin[0].table[2, :2].clone()
  steps_table = begin[0].table.clone()
  steps_table[2, :2] = steps_table[0, :2]
  begin[0].table[2, :2] = -1                 # (one tensor for both layers)
  going_on = [attention.PagedState(s.cache, steps_table) for s in begin]
  model.call_layers(t(known), vdt, mode="first_part", states=begin, reuse=True)
  steps = []
  for p in range(first, length):
    token = mtf.import_tf_tensor(mesh, x[:, p].contiguous(),
                                 mtf.Shape([batch, model_dim]))
    position = mtf.import_tf_tensor(mesh, torch.full((b,), p, dtype=torch.int32),
                                    mtf.Shape([batch]))
    steps.append(model.call_layers(token, vdt, mode="incremental", position=position,
                                   states=going_on, length_dim=len_dim)[0])
  for s in begin:                            # (nobody's pages any more)
    s.cache.k_pages[spare.long()] = s.cache.v_pages[spare.long()] = float("nan")
  lowering = mtf.Lowering(graph, {mesh: mtf.HipMeshImpl()},
                          initial_values=_initial_values(graph, rng))
  # (the tolerances of decoding above)
  tol = (dict(rtol=2e-4, atol=2e-4) if act_dtype == torch.float32
         else dict(rtol=5e-2, atol=5e-2))
  want = lowering.export_to_tf_tensor(y_full).float()
  for p, step in zip(range(first, length), steps):
    torch.testing.assert_close(lowering.export_to_tf_tensor(step).float(), want[:, p],
                               **tol)
  for s in begin:
    assert torch.isnan(s.cache.k_pages[spare.long()].float()).all()
