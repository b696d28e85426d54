"""The layer-stack part of mesh_tensorflow/transformer/transformer.py that a
Mixture-of-Experts transformer block needs: TransformerLayer, Context,
LayerStack with its sublayers (RMS norm, layer call, dropout, residual,
padding mask), make_layer_stack, and the layer-stack call of Unitransformer.

Decoding: the "first_part" and "incremental" modes of the Context and of
SelfAttention (recurrent key / value states); the sampling loop around them
stays with the caller.

Not here: embeddings, vocabularies, logits and losses of Unitransformer /
Bitransformer, ensembles, subsequence ids.
"""

from mesh_amd import layers as mtf_layers
from mesh_amd import ops as mtf

TRAIN = "train"   # tf.estimator.ModeKeys.TRAIN
EVAL = "eval"     # tf.estimator.ModeKeys.EVAL
FIRST_PART = "first_part"     # decoding: the known first part, records states
INCREMENTAL = "incremental"   # decoding: one position per call, states in/out


class _Position(object):
  """Stands for mtf.range(mesh, length_dim, int32), the value Unitransformer
  gives read_priority and write_priority of an autoregressive model
  (transformer.py:1032-1040): position a sees position b iff a >= b."""

  def __repr__(self):
    return "POSITION"


POSITION = _Position()


class TransformerLayer(object):
  """Base class of the layers (transformer.py:56-105): the constructor records
  hyperparameters, call(context, x) builds the layer and its variables."""

  def call(self, context, x):
    raise NotImplementedError("Not implemented")

  def set_name(self, name):
    self._name = name

  @property
  def name(self):
    return getattr(self, "_name", None)


# Context fields that only decoding, beam search, encoder-decoder attention or
# parameter sharing use; accepted for signature compatibility, must stay None.
_UNUSED_CONTEXT_FIELDS = (
    "beam_dim", "subsequence_id", "initial_position",
    "encoder_output", "encoder_sequence_id", "constant_states",
    "shared_params", "encoder_layer_outputs", "inputs", "encoder_inputs")


class Context(object):
  """What layers need at call time (transformer.py:107-311), for the "train"
  and "eval" modes.  read_priority / write_priority are None (every position
  sees every position) or POSITION (autoregressive); sequence_id is None, 1
  (no padding) or an int32 Tensor [batch..., length] (packed sequences; 0 marks
  padding).  The reference's remaining constructor arguments
  (_UNUSED_CONTEXT_FIELDS) are accepted as keywords and must be None."""

  def __init__(self, model, mesh, batch_dims, length_dim, variable_dtype,
               mode=TRAIN, position=None, position_is_default=False,
               sequence_id=None, losses=None, layer_outputs=None,
               write_priority=None, read_priority=None, num_microbatches=1,
               states=None, new_states=None, **unused):
    if mode not in (TRAIN, EVAL, FIRST_PART, INCREMENTAL):
      raise ValueError("unknown mode %r" % (mode,))
    if mode == INCREMENTAL and not isinstance(position, mtf.Tensor):
      raise ValueError("incremental mode needs the position tensor "
                       "[batch dims] (int32)")
    for key, value in unused.items():
      if key not in _UNUSED_CONTEXT_FIELDS:
        raise TypeError("Context got an unexpected argument %r" % key)
      if value is not None:
        raise NotImplementedError("Context.%s is not implemented" % key)
    if (write_priority is None) != (read_priority is None):
      raise ValueError("read_priority and write_priority go together")
    if write_priority not in (None, POSITION) or read_priority not in (
        None, POSITION):
      raise NotImplementedError("read/write priorities other than the position")
    for key in _UNUSED_CONTEXT_FIELDS:
      setattr(self, key, None)
    self.shared_params = {}
    self.model, self.mesh = model, mesh
    self.batch_dims, self.length_dim = batch_dims, length_dim
    self.variable_dtype = variable_dtype
    self.mode = mode
    self.position, self.position_is_default = position, position_is_default
    self.sequence_id = sequence_id
    self.losses = losses
    self.layer_outputs = [] if layer_outputs is None else layer_outputs
    self.write_priority, self.read_priority = write_priority, read_priority
    self.num_microbatches = num_microbatches
    # recurrent states of decoding (transformer.py:251-272): layers read
    # theirs with get_states in "incremental" mode and append the new values
    # with record_new_states in "first_part" and "incremental" modes
    self.states = [] if states is None else list(states)
    self.new_states = [] if new_states is None else new_states
    self.layer_index = 0
    self.cache = {}            # values shared between layers

  train = property(lambda self: self.mode == TRAIN)

  def get_states(self, n):
    """The next n recurrent states (transformer.py:251-261)."""
    got = self.states[len(self.new_states):len(self.new_states) + n]
    if len(got) != n:
      raise ValueError("incremental mode: %d states were passed, a layer asks "
                       "for states %d..%d" % (len(self.states),
                                              len(self.new_states),
                                              len(self.new_states) + n - 1))
    return got

  def paged_state(self):
    """The next recurrent state, where it is kept in pages (attention.PagedState), else
    None."""
    from mesh_amd.transformer import attention
    states = self.states[:len(self.new_states) + 1]
    if len(states) <= len(self.new_states) or not isinstance(
        states[-1], attention.PagedState):
      return None
    state = states.pop()
    if any(isinstance(s, attention.PagedState) and s.cache.overlaps(state.cache)
           for s in states):
      raise ValueError("two layers were given the same pages")
    return state

  def record_new_states(self, new_states):
    """transformer.py:263-271."""
    self.new_states.extend(new_states)
  activation_dtype = property(
      lambda self: self.variable_dtype.activation_dtype)

  @property
  def nonpadding(self):
    """Zeros in padding positions and ones elsewhere (transformer.py:297-306):
    None without a sequence_id, the integer 1 when sequence_id == 1, else
    cast(sequence_id != 0, activation dtype) (built once per context)."""
    if self.sequence_id is None:
      return None
    if isinstance(self.sequence_id, int) and self.sequence_id == 1:
      return 1
    if "nonpadding" not in self.cache:
      self.cache["nonpadding"] = mtf.cast(
          mtf.not_equal(self.sequence_id, 0), self.activation_dtype)
    return self.cache["nonpadding"]


def _is_ahead(tensor, operation):
  """Is `tensor` computed before `operation` runs?"""
  operations = operation.graph.operations
  return operations.index(tensor.operation) < operations.index(operation)


def _slice_of(lowering, tensor):
  return lowering.tensors[tensor].to_laid_out_tensor().tensor_list[0]


class ResidualAddOperation(mtf.Operation):
  """x + y of one shape and dtype (sublayer_residual).  Where an RMS norm reads the
  sum, the norm (and the padding mask behind it) is made by the same kernel, once
  its scale is there (variables are lowered in graph order: from the second run
  on)."""

  def __init__(self, x, y, name=None):
    super(ResidualAddOperation, self).__init__([x, y], name=name or "add")
    self.norm = None         # the RmsNormOperation of the sum
    self._outputs = [mtf.Tensor(self, x.shape, x.dtype)]

  def gradient(self, grad_ys):
    return [grad_ys[0], grad_ys[0]]

  def lower(self, lowering):
    if self.norm is None or not self.norm.lower_with(lowering, self):
      lowering.set_tensor_lowering(
          self.outputs[0], lowering.mesh_impl(self).slicewise(
              lambda a, b: a + b, *[lowering.tensors[t] for t in self.inputs]))


class RmsNormOperation(mtf.Operation):
  """x * rsqrt(mean(square(x)) + epsilon) * scale over the last dim: the five
  ops of sublayer_rms_norm (transformer.py:493-516) in one kernel."""

  def __init__(self, x, scale, epsilon, name=None):
    super(RmsNormOperation, self).__init__([x, scale], name=name or "rms_norm")
    if scale.shape.dims != x.shape.dims[-1:]:
      raise ValueError("scale %s does not match the last dim of %s"
                       % (scale.shape, x.shape))
    self._epsilon = float(epsilon)
    self._outputs = [mtf.Tensor(self, x.shape, x.dtype)]
    self._handed_over = (0, False)
    self.mask = None         # the MaskPaddingOperation of the result
    residual = x.operation
    if (isinstance(residual, ResidualAddOperation) and residual.norm is None and
        (isinstance(scale.operation, mtf.Variable) or _is_ahead(scale, residual))):
      residual.norm = self

  def _hands_over(self):
    """Whether nothing but an 8-bit dense layer reads the (masked) norm, which then
    leaves as its operand."""
    count, mask, y = len(self.graph.operations), self.mask, self.outputs[0]
    if self._handed_over[0] != count:
      over = mtf_layers.only_eight_bit_dense_reads(y if mask is None
                                                   else mask.outputs[0])
      if mask is not None:
        over = over and [mask] == [op for op in self.graph.operations if y in op.inputs]
      self._handed_over = (count, over)
    return self._handed_over[1]

  def _lower_to_eight_bits(self, lowering, residual):
    """lower_with() into the operand of an 8-bit dense layer."""
    from mesh_amd import fp8_hip
    x, scale = self.inputs
    mask, eps = self.mask, self._epsilon
    if scale not in lowering.tensors or not self._hands_over():
      return False
    ins = residual.inputs if residual is not None else [x]
    rows = [_slice_of(lowering, t).contiguous() for t in ins]
    w = _slice_of(lowering, scale).contiguous()
    if w.dtype != rows[0].dtype or rows[0].numel() == 0:
      return False
    row_mask = None if mask is None else _slice_of(lowering, mask.inputs[1]).contiguous()
    mesh_impl = lowering.mesh_impl(self)
    total, operand = [t.tensor_list[0] for t in mesh_impl.slicewise(
        lambda: fp8_hip.residual_rms_norm(
            rows[0], rows[1] if residual is not None else None, w, eps, row_mask))]
    # (whoever else asks for the tensors sees the values that are multiplied, or the
    # norm without its mask)
    y = self.outputs[0] if mask is None else mask.outputs[0]
    lowering.run_values[y] = operand
    sizes = y.shape.to_integer_list
    lowering.set_tensor_lowering(y, mesh_impl.LazyLaidOutTensor(
        lambda: mesh_impl.slicewise(lambda: fp8_hip.dequantize(operand)), sizes))
    if mask is not None:
      laid_out = mesh_impl.LaidOutTensor
      lowering.set_tensor_lowering(self.outputs[0], mesh_impl.LazyLaidOutTensor(
          lambda: self._alone(mesh_impl, laid_out([total]), laid_out([w])), sizes))
      lowering.done_ahead.add(mask)
    if residual is not None:
      lowering.set_tensor_lowering(x, mesh_impl.LaidOutTensor([total]))
      lowering.done_ahead.add(self)
    return True

  def lower_with(self, lowering, residual):
    """Makes this norm, the residual sum in front of it (`residual`, or None: the
    norm's input is there) and the padding mask behind it in one kernel.  False
    where that cannot be done."""
    from mesh_amd import moe_hip
    x, scale = self.inputs
    mask = self.mask
    if self._lower_to_eight_bits(lowering, residual):
      return True
    if scale not in lowering.tensors or (residual is None and mask is None):
      return False
    ins = residual.inputs if residual is not None else [x]
    rows = [_slice_of(lowering, t) for t in ins]
    w = _slice_of(lowering, scale).contiguous()
    if w.dtype != rows[0].dtype or not moe_hip.residual_rms_norm_supported(
        *rows, w):
      return False
    row_mask = None if mask is None else _slice_of(lowering, mask.inputs[1])
    mesh_impl = lowering.mesh_impl(self)
    eps = self._epsilon

    def fn(first_rows):
      return moe_hip.residual_rms_norm(
          first_rows, rows[1] if residual is not None else None, w, eps,
          None if row_mask is None else row_mask.contiguous(),
          want_norm=row_mask is not None)
    results = mesh_impl.slicewise(fn, lowering.tensors[ins[0]])
    if residual is not None:
      lowering.set_tensor_lowering(x, results[0])
      lowering.done_ahead.add(self)
    if mask is not None:
      lowering.set_tensor_lowering(mask.outputs[0], results[1])
      lowering.done_ahead.add(mask)
    lowering.set_tensor_lowering(self.outputs[0], results[-1])
    return True

  def _alone(self, mesh_impl, x, scale):
    from mesh_amd import moe_hip
    eps = self._epsilon

    def fn(x, scale):
      return moe_hip.rms_norm(x.contiguous(), scale.contiguous(), eps)
    return mesh_impl.slicewise(fn, x, scale)

  def lower(self, lowering):
    if self in lowering.done_ahead or self.lower_with(lowering, None):
      return
    lowering.set_tensor_lowering(
        self.outputs[0],
        self._alone(lowering.mesh_impl(self),
                    *[lowering.tensors[t] for t in self.inputs]))

  def gradient(self, grad_ys):
    return list(RmsNormGradOperation(self, grad_ys[0]).outputs)


class MaskPaddingOperation(mtf.Operation):
  """x * nonpadding (sublayer_mask_padding): x [..., M], nonpadding [...] of x's
  dtype."""

  def __init__(self, x, nonpadding, name=None):
    super(MaskPaddingOperation, self).__init__([x, nonpadding],
                                               name=name or "mul")
    self._outputs = [mtf.Tensor(self, x.shape, x.dtype)]
    self.of_gradient = False   # made by gradient() below
    norm = x.operation
    if isinstance(norm, RmsNormOperation) and norm.mask is None:
      residual = norm.inputs[0].operation
      first = residual if getattr(residual, "norm", None) is norm else norm
      if _is_ahead(nonpadding, first):
        norm.mask = self

  def gradient(self, grad_ys):
    masked = MaskPaddingOperation(grad_ys[0], self.inputs[1])
    masked.of_gradient = True
    return [masked.outputs[0], mtf.smaller_factor_gradient(self, grad_ys[0])]

  def lower(self, lowering):
    if self in lowering.done_ahead:
      return
    mesh_impl = lowering.mesh_impl(self)
    lowering.set_tensor_lowering(
        self.outputs[0], mesh_impl.slicewise(
            lambda a, m: a * m.unsqueeze(-1),
            *[lowering.tensors[t] for t in self.inputs]))


class RmsNormGradOperation(mtf.Operation):
  """(dx, dscale) of an RmsNormOperation.  It also takes over the gradient of a
  padding mask behind the norm, and adds the gradient that reaches x on another way
  to dx (add_to_output): with the inputs dy, x, scale, mask (or None) and addend (or
  None), dx = addend + d norm(dy * mask)."""

  def __init__(self, forward, dy, name=None):
    x, scale = forward.inputs
    self._mask = self._addend = None
    masked = dy.operation
    if (isinstance(masked, MaskPaddingOperation) and masked.of_gradient and
        not mtf.gradient_is_returned(forward.outputs[0])):
      # this is the only reader of the masked gradient: it leaves the graph
      dy, self._mask = masked.inputs
      masked.graph.operations.remove(masked)
    super(RmsNormGradOperation, self).__init__(
        [dy, x, scale] + ([] if self._mask is None else [self._mask]),
        name=name or "rms_norm_grad")
    self._epsilon = forward._epsilon   # pylint: disable=protected-access
    self._outputs = [mtf.Tensor(self, x.shape, x.dtype, index=0),
                     mtf.Tensor(self, scale.shape, scale.dtype, index=1)]

  def add_to_output(self, output, addend):
    """Makes `output` the sum of what it was and addend, before anything reads it;
    False where this operation cannot."""
    if (output is not self._outputs[0] or self._addend is not None or
        addend.shape != output.shape or addend.dtype != output.dtype or
        not _is_ahead(addend, self)):
      return False
    self._addend = addend
    self._inputs.append(addend)
    return True

  def lower(self, lowering):
    from mesh_amd import moe_hip
    eps = self._epsilon

    def fn(dy, x, scale, mask, addend):
      x, dy = x.contiguous(), dy.contiguous()
      w = scale.to(x.dtype).contiguous()
      added = [] if addend is None else [addend.contiguous()]
      if ((mask is not None or added) and
          moe_hip.residual_rms_norm_supported(x, w, dy, *added)):
        dx, dscale = moe_hip.rms_norm_backward(
            x, w, dy, eps, row_mask=None if mask is None else mask.contiguous(),
            addend=added[0] if added else None)
        return dx, dscale.to(scale.dtype)
      if mask is not None:
        dy = dy * mask.unsqueeze(-1)
      dx, dscale = moe_hip.rms_norm_backward(x, w, dy, eps)
      return dx if addend is None else addend + dx, dscale.to(scale.dtype)
    dx, dscale = lowering.mesh_impl(self).slicewise(
        fn, *[None if t is None else lowering.tensors[t] for t in
              self.inputs[:3] + [self._mask, self._addend]])
    lowering.set_tensor_lowering(self.outputs[0], dx)
    lowering.set_tensor_lowering(self.outputs[1], dscale)


def sublayer_call_layer(x, layer_stack, context):
  """transformer.py:462-466."""
  x = sublayer_mask_padding(x, layer_stack, context)
  layer = context.current_layer
  with mtf.variable_scope(layer.__class__.__name__):
    return layer.call(context, x)


def sublayer_mask_padding(x, layer_stack, context):
  """Zeroes the padding positions (transformer.py:469-489); without a
  sequence_id tensor there is nothing to mask."""
  del layer_stack
  if not isinstance(context.sequence_id, mtf.Tensor):
    return x
  mask = context.nonpadding
  if x.dtype == mask.dtype and x.shape.dims[:-1] == mask.shape.dims:
    return MaskPaddingOperation(x, mask).outputs[0]
  return x * mask


def sublayer_rms_norm(x, layer_stack, context, epsilon=1e-6, name="rms_norm"):
  """RMS normalisation with a learned scale `<name>/scale` [d_model]
  (transformer.py:493-516)."""
  del layer_stack
  model_dim = context.model.model_dim
  if context.model.ensemble_dims:
    raise NotImplementedError("ensembles are not implemented")
  with mtf.variable_scope(name):
    scale = mtf.get_variable(context.mesh, "scale", mtf.Shape([model_dim]),
                             initializer=mtf_layers.ones_initializer(),
                             dtype=context.variable_dtype)
  return RmsNormOperation(x, scale, epsilon, name=name).outputs[0]


def sublayer_legacy_rms_norm(x, layer_stack, context):
  """transformer.py:519-522."""
  return sublayer_rms_norm(x, layer_stack, context, name="layer_norm")


def sublayer_legacy_final_rms_norm(x, layer_stack, context):
  """transformer.py:525-528."""
  return sublayer_rms_norm(x, layer_stack, context, name="final_layer_norm")


def sublayer_residual(x, layer_stack, context):
  """transformer.py:584-587."""
  del layer_stack
  y = context.current_layer_input
  if x.shape == y.shape and x.dtype == y.dtype:
    return ResidualAddOperation(x, y).outputs[0]
  return x + y


def sublayer_dropout(x, layer_stack, context, dropout_rate=0.0):
  """transformer.py:590-599: while training, one noise value per (batch
  entry, channel), shared by the positions of a sequence."""
  del layer_stack
  if context.train and dropout_rate > 0:
    return mtf.dropout(
        x, context.train, rate=dropout_rate,
        noise_shape=mtf.Shape(context.batch_dims + [context.model.model_dim]))
  return x


def sublayer_legacy_dropout(x, layer_stack, context):
  """transformer.py:627-636."""
  return sublayer_dropout(x, layer_stack, context,
                          dropout_rate=layer_stack.dropout_rate)


class LayerStack(TransformerLayer):
  """A stack of layers with residual connections and norms
  (transformer.py:314-457).  The default sublayers are those of the
  reference's defaults.gin."""

  def __init__(self, layers, sublayers_initial=None, sublayers_per_layer=None,
               sublayers_final=None, dropout_rate=None, norm_epsilon=None,
               recompute_grads=False):
    if recompute_grads:
      raise NotImplementedError("recompute_grads is not implemented")
    self._layers = layers
    self._sublayers_initial = sublayers_initial
    self._sublayers_per_layer = sublayers_per_layer
    self._sublayers_final = sublayers_final
    if (dropout_rate is not None) != (norm_epsilon is not None):
      raise ValueError(
          "LayerStack.dropout_rate and LayerStack.norm_epsilon should either "
          "be both not None (legacy mode) or both None (normal mode)")
    if dropout_rate is not None:
      # legacy mode, for old checkpoints' variable names (transformer.py:383-406)
      self.dropout_rate = dropout_rate
      self.norm_epsilon = norm_epsilon
      self._sublayers_initial = [sublayer_legacy_dropout]
      self._sublayers_per_layer = [sublayer_legacy_rms_norm,
                                   sublayer_call_layer,
                                   sublayer_legacy_dropout, sublayer_residual]
      self._sublayers_final = [sublayer_legacy_final_rms_norm,
                               sublayer_legacy_dropout]
    else:
      if self._sublayers_initial is None:
        self._sublayers_initial = [sublayer_dropout]
      if self._sublayers_per_layer is None:
        self._sublayers_per_layer = [sublayer_rms_norm, sublayer_call_layer,
                                     sublayer_dropout, sublayer_residual]
      if self._sublayers_final is None:
        self._sublayers_final = [sublayer_rms_norm, sublayer_dropout]

  def call(self, context, x):
    """transformer.py:408-428."""
    if isinstance(context.sequence_id, mtf.Tensor):
      context.nonpadding       # built here, ahead of everything that is masked
    x = self._call_sublayers(self._sublayers_initial, x, context)
    context.layer_outputs.append(x)
    for lnum, layer in enumerate(self._layers):
      with mtf.variable_scope(layer.name or ""):
        x = self._layer_fn(x, layer, context)
      if lnum != len(self._layers) - 1:
        context.layer_outputs.append(x)
      context.layer_index += 1
    x = self._call_sublayers(self._sublayers_final, x, context)
    x = sublayer_mask_padding(x, self, context)
    context.layer_outputs.append(x)
    return x

  def _call_sublayers(self, sublayers, x, context):
    for s in sublayers:
      x = s(x, self, context)
    return x

  def _layer_fn(self, x, layer, context):
    context.current_layer = layer
    context.current_layer_input = x
    y = self._call_sublayers(self._sublayers_per_layer, x, context)
    if y.shape != x.shape:
      raise ValueError("Layer %s returned misshaped output x=%s y=%s"
                       % (layer.__class__.__name__, x, y))
    return y

  @property
  def num_layers(self):
    return len(self.layers)

  @property
  def layers(self):
    return self._layers


def _layer_spec(spec):
  """A class, or a list / tuple holding a class and optionally a name (str)
  and constructor arguments (dict), in any order."""
  if not isinstance(spec, (list, tuple)):
    return spec, None, {}
  cls, name, kwargs = None, None, {}
  for item in spec:
    if isinstance(item, str):
      name = item
    elif isinstance(item, dict):
      kwargs = item
    else:
      cls = item
  return cls, name, kwargs


def make_layer_stack(layers, num_layers=6, block_scope=True,
                     layer_stack_cls=LayerStack):
  """transformer.py:1876-1948: `layers` describes one block, repeated
  num_layers times.  Layer names are block_%03d/<name or layer_%03d> with
  block_scope, else <name> or layer_%03d counted over the whole stack."""
  built = []
  for block in range(num_layers):
    for n, spec in enumerate(layers):
      cls, name, kwargs = _layer_spec(spec)
      if block_scope:
        name = "block_%03d/%s" % (block, name or "layer_%03d" % n)
      elif not name:
        name = "layer_%03d" % len(built)
      layer = cls(**kwargs)
      layer.set_name(name)
      built.append(layer)
  return layer_stack_cls(built)


class Unitransformer(object):
  """The layer-stack call of the reference's Unitransformer
  (transformer.py:696-1075) on activations that are already embedded: model
  dims, the Context, and LayerStack.call under the model's name scope."""

  def __init__(self, layer_stack, d_model=1024, name="transformer",
               autoregressive=False, layout=None, mesh_shape=None,
               ensemble=None):
    if ensemble:
      raise NotImplementedError("ensembles are not implemented")
    self.layer_stack = layer_stack
    self.model_dim = mtf.Dimension("d_model", d_model)
    self.name = name
    self.autoregressive = autoregressive
    self.layout = layout
    self.mesh_shape = mesh_shape
    self.ensemble_dim = None

  @property
  def ensemble_dims(self):
    return []

  @property
  def fully_autoregressive(self):
    return self.autoregressive

  def call_layers(self, x, variable_dtype, mode=EVAL, num_microbatches=1,
                  sequence_id=None, position=None, states=None,
                  new_states=None, length_dim=None, reuse=None):
    """x [batch dims..., length, d_model] -> (y, losses).  The Context is the
    one _call_internal builds (transformer.py:1032-1062): read and write
    priorities are the position for an autoregressive model.

    Decoding, as sample_autoregressive drives it (transformer.py:1140-1248):
    mode "first_part" runs the known first part and appends every attention
    layer's keys and values to the list `new_states`; mode "incremental" takes
    x [batch dims..., d_model] (one position per batch entry), `position`
    [batch dims...] int32, the states of the previous call as `states`, the
    sequences' `length_dim`, and appends the updated states to `new_states`.
    Where the states passed in either mode are attention.PagedState objects, one per
    attention layer, keys and values are written into their pages instead, and the same
    objects are the new states (`new_states` may be left out).
    The loop around it (sampling, stopping) stays with the caller.  `reuse`:
    take the variables an earlier call on this graph created (the default in
    "incremental" mode, as the reference's loop body does)."""
    if x.shape.dims[-1] != self.model_dim:
      raise ValueError("x %s does not end in %s" % (x.shape, self.model_dim))
    priority = POSITION if self.autoregressive else None
    losses = []
    if mode == INCREMENTAL:
      if length_dim is None:
        raise ValueError("incremental mode needs length_dim")
      batch_dims = x.shape.dims[:-1]
    else:
      batch_dims, length_dim = x.shape.dims[:-2], x.shape.dims[-2]
    context = Context(
        model=self, mesh=x.mesh, batch_dims=batch_dims,
        length_dim=length_dim, variable_dtype=variable_dtype, mode=mode,
        position=position, position_is_default=position is None,
        sequence_id=sequence_id, losses=losses,
        write_priority=priority, read_priority=priority,
        num_microbatches=num_microbatches, states=states,
        new_states=new_states)
    if reuse is None:
      reuse = mode == INCREMENTAL
    with mtf.variable_scope(self.name, reuse=reuse):
      y = self.layer_stack.call(context, x)
    return y, losses
