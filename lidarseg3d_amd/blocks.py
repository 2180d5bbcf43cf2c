"""Operators of a transformer block in training and serving: what stands between its matrix products and its attention.

    from lidarseg3d_amd import blocks
    rng = blocks.DropoutState(seed=0, device="cuda")
    h = blocks.embedding(table, tokens, scale=32.0)                                             # lookup, gradient by sorted tokens
    y, h = blocks.residual_norm(block(y), h, norm=blocks.Norm.of(ln), p=0.1, state=rng, return_sum=True)  # the norm of h + dropout(block), and that sum
    y = blocks.dropout(linear(y), 0.1, rng, relu=True)                                          # dropout(relu(.))
    loss.backward(); rng.advance()

All three take float32, bfloat16 and float16 tensors with any leading dimensions, run on the current stream of the tensors' device, allocate their
outputs with torch and give the same bits for the same inputs.  Sums, statistics and parameter gradients are formed in 32 bits and rounded once.  They are
differentiable once, in reverse mode; tracers, fake tensors, torch.func's transforms and forward-mode tangents are refused.

`use_in_training(model, rng)` puts the training forward of this package's models on them (counter-based dropout, residual and norm in one pass,
camera sampling with a deterministic gradient)."""
import torch
from torch import nn

from . import _lib, ops

_KINDS = {"layer": 1, "rms": 2}
_TYPES = (torch.float32, torch.bfloat16, torch.float16)
_NO_NORM = (None, None, 0, 0.0)


class Norm(object):
    """Norm("layer" | "rms", weight [c] or None, bias [c] or None, eps): what `norm` and `norm_in` of residual_norm take; Norm.of(module) for an
    nn.LayerNorm / nn.RMSNorm over the last dimension"""

    def __init__(self, kind, weight=None, bias=None, eps=1e-5):
        if kind not in _KINDS:
            raise ValueError("norm kind %r: 'layer' or 'rms'" % (kind,))
        if not eps >= 0:
            raise ValueError("eps %r" % (eps,))
        self.kind, self.weight, self.bias, self.eps = kind, weight, bias, float(eps)

    @classmethod
    def of(cls, module):
        if len(module.normalized_shape) != 1:
            raise ValueError("a norm over the last dimension only is needed (normalized_shape %s)" % (tuple(module.normalized_shape),))
        if isinstance(module, nn.LayerNorm):
            return cls("layer", module.weight, module.bias, module.eps)
        if isinstance(module, nn.RMSNorm):
            if module.eps is None:  # torch's default there: the input type's eps
                raise ValueError("nn.RMSNorm without an eps: give one")
            return cls("rms", module.weight, None, module.eps)
        raise TypeError("nn.LayerNorm or nn.RMSNorm needed, got %s" % type(module).__name__)


class DropoutState(object):
    """(seed, step) of a training program's dropout, on the device, and the number of the next call within the step.  The kernels read seed and step
    when they run: a captured training step that ends with advance() draws new masks at every replay.  advance() comes after the backward pass
    of everything drawn before it (an eager backward that finds another step raises, as after any in-place change of a saved tensor).  A graph keeps the call
    numbers of its capture; eager work between its replays takes a state of its own, or it may draw what the graph draws.  Under activation checkpointing
    each dropout is given its `call`: a forward pass repeated inside the backward pass that asks for the next number raises."""

    def __init__(self, seed, device="cuda", step=0):
        self.tensor = torch.tensor([int(seed), int(step)], dtype=torch.int64, device=device)
        self.calls = 0

    def next_call(self):
        if torch._C._current_graph_task_id() != -1:  # (activation checkpointing: the forward pass is repeated and would count on, its masks not those of the first time)
            raise RuntimeError("a dropout inside a backward pass (activation checkpointing) needs its `call` given")
        n = self.calls
        self.calls += 1
        return n

    def advance(self):
        self.tensor[1:].add_(1)
        self.calls = 0

    def state_dict(self):
        return {"state": self.tensor.clone(), "calls": self.calls}

    def load_state_dict(self, sd):
        self.tensor.copy_(sd["state"])
        self.calls = int(sd["calls"])


def _dtype_ok(t, what):
    if t.dtype not in _TYPES:
        raise TypeError("%s: float32, bfloat16 or float16 needed, got %s" % (what, t.dtype))


def _on_device(t, what):
    if not (t.is_cuda or ops._SIM):
        raise RuntimeError("%s: lidarseg3d_amd ops need tensors on the MI355X (got a %s tensor); there is no CPU fallback" % (what, t.device))


def _number(v, what):
    if torch.is_tensor(v) and v.requires_grad:
        raise TypeError("%s is a number: a tensor that requires a gradient would not get one" % what)


def _draw(p, state, call):
    """-> (p, state tensor, call) of a dropout"""
    if p == 0.0:
        return 0.0, None, 0
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout probability %r" % (p,))
    if isinstance(state, DropoutState):
        call = state.next_call() if call is None else call
        state = state.tensor
    if not torch.is_tensor(state) or state.dtype != torch.int64 or state.shape != (2,) or not state.is_contiguous():
        raise ValueError("dropout needs a DropoutState, or its int64 (seed, step) tensor")
    if call is None:
        raise ValueError("`call`, the number of this dropout within the step, is needed with a bare state tensor")
    if not 0 <= int(call) < 1 << 32:
        raise ValueError("call %r is not in [0, 2^32)" % (call,))
    return p, state, int(call)


# ---------------------------------------------------------------------------------------------- dropout
def dropout(x, p, state, call=None, relu=False):
    """dropout(x) - relu: dropout(relu(x)) - over the last dimension's rows, the mask made from (seed, step, call, row, column) in the forward pass and
    again in the backward pass: it is never stored (relu: one bit per element says where x was positive and kept).
    p is resolved to 1 / 65536 and what is kept is scaled by the inverse of the resolved probability.  state: a DropoutState, or its tensor together with
    `call`; two dropouts of one step need different calls.  A dropped element is zero whatever stood there."""
    if not x.is_cuda:
        _on_device(x, "dropout")
    if x.dtype not in _TYPES:
        _dtype_ok(x, "dropout")
    p, state, call = _draw(p, state, call)
    if p == 0.0:
        return torch.relu(x) if relu else x
    if x.dim() == 0:
        return dropout(x.reshape(1), p, state, call, relu).reshape(())
    if x.numel() == 0:
        return x
    return _lib.host_module().dropout(x, p, state, call, relu)


class Dropout(nn.Dropout):
    """nn.Dropout on `dropout` with a DropoutState (None: torch's generator, as nn.Dropout); evaluation passes its input through"""
    converted = False  # an nn.Dropout that use_in_training put on the operator

    def __init__(self, p, state=None):
        super().__init__(p)
        self.state = state

    def forward(self, input):
        if self.state is None:
            return super().forward(input)
        if not self.training:
            return input
        out = dropout(input, self.p, self.state)
        return input.copy_(out) if self.inplace and out is not input else out


# ---------------------------------------------------------------------------------------------- residual, dropout, gate and norms
def _norm_arguments(nm, c, what):
    """-> weight, bias, kind, eps of a Norm, checked against rows of c values"""
    if not isinstance(nm, Norm):
        raise TypeError("%s: a blocks.Norm needed, got %s" % (what, type(nm).__name__))
    out = []
    for t in (nm.weight, nm.bias):
        if t is not None:
            if t.dtype not in _TYPES:
                _dtype_ok(t, what + " parameter")
            if t.dim() != 1 or t.shape[0] != c:
                raise ValueError("%s: weight and bias of shape [%d] needed, got %s" % (what, c, tuple(t.shape)))
            if not t.is_contiguous():
                t = t.contiguous()
        out.append(t)
    return out[0], out[1], _KINDS[nm.kind], nm.eps


def residual_norm(x, residual=None, norm=None, norm_in=None, gate=None, alpha=1.0, p=0.0, state=None, call=None, return_sum=False):
    """One pass over a block's output x [..., c] and the residual stream:

        t = norm_in(x);  s = alpha * residual + gate * dropout(t);  y = norm(s)      -> y;  (y, s) with return_sum;  s without a norm

    norm / norm_in: a Norm (layer or RMS) or None.  gate: None, a single value, one per channel [c], or one per element (x's shape and type).
    residual: x's shape, of x's type or float32 (s has its type).  p / state / call: as in `dropout`; p = 0 outside training.  c <= 8192."""
    if not x.is_cuda:
        _on_device(x, "residual_norm")
    if x.dtype not in _TYPES:
        _dtype_ok(x, "residual_norm")
    shape = x.shape
    if not shape:
        raise ValueError("residual_norm needs at least one dimension")
    c = shape[-1]
    if c > 8192:
        raise ValueError("residual_norm takes rows of up to 8192 values, got %d" % c)
    if residual is not None:
        if residual.shape != shape:
            raise ValueError("residual %s does not match x %s" % (tuple(residual.shape), tuple(shape)))
        if residual.dtype != x.dtype and residual.dtype != torch.float32:
            raise TypeError("residual: %s or float32 needed, got %s" % (x.dtype, residual.dtype))
    if gate is not None:
        _dtype_ok(gate, "gate")
        if gate.shape == shape and gate.dim() > 1 and gate.numel() != 1:
            if gate.dtype != x.dtype:
                raise TypeError("a gate for each element has x's type (%s), got %s" % (x.dtype, gate.dtype))
        elif gate.numel() == 1 or gate.shape == (c,):
            gate = gate if gate.shape == (c,) else gate.reshape(1).float().expand(c)  # (float: its gradient is the sum of c channels', rounded once at the end)
            if not gate.is_contiguous():
                gate = gate.contiguous()
        else:
            raise ValueError("gate %s: one value, [%d] or %s" % (tuple(gate.shape), c, tuple(shape)))
    _number(alpha, "alpha")
    w_in, b_in, kind_in, eps_in = _NO_NORM if norm_in is None else _norm_arguments(norm_in, c, "norm_in")
    w_out, b_out, kind_out, eps_out = _NO_NORM if norm is None else _norm_arguments(norm, c, "norm")
    p, state, call = _draw(p, state, call)
    out = _lib.host_module().residual_norm(x, residual, gate, w_in, b_in, w_out, b_out, state, kind_in, eps_in, kind_out, eps_out, alpha, p, call, return_sum)
    return out[0] if len(out) == 1 else tuple(out)


# ---------------------------------------------------------------------------------------------- row lookup
def embedding(table, idx, weight=None, scale=1.0, padding_idx=None, bag=False):
    """scale * table[idx] of a table [rows, c]; idx int32 / int64 of any shape.  bag: the sum over idx's last dimension [..., k], with `weight` (float32, idx's
    shape) the weighted sum, scale * sum_j weight[..., j] * table[idx[..., j]].  An index outside [0, rows) - -1 by custom - names no row: it reads as zero and takes no
    gradient.  padding_idx: a row that is read but takes no gradient.  The table's gradient is dense; its entries are sorted by row and
    added in input order: the same bits every time, for one frequent token as for many rare ones."""
    if not table.is_cuda:
        _on_device(table, "embedding")
    if table.dtype not in _TYPES:
        _dtype_ok(table, "embedding")
    if table.dim() != 2:
        raise ValueError("embedding: a table [rows, c] needed, got %s" % (tuple(table.shape),))
    if idx.dtype != torch.int64 and idx.dtype != torch.int32:
        raise TypeError("embedding: int32 or int64 indices needed, got %s" % idx.dtype)
    if weight is not None:
        if weight.dtype != torch.float32:
            raise TypeError("embedding: float32 weights needed, got %s" % weight.dtype)
        if weight.shape != idx.shape or idx.dim() < 1:
            raise ValueError("embedding: weights %s do not match the indices %s" % (tuple(weight.shape), tuple(idx.shape)))
        bag = True
    if bag and (idx.dim() < 1 or idx.shape[-1] == 0):
        raise ValueError("embedding: no indices to sum over")
    _number(scale, "scale")
    if padding_idx is not None and not -table.shape[0] <= padding_idx < table.shape[0]:
        raise ValueError("padding_idx %r outside a table of %d rows" % (padding_idx, table.shape[0]))
    padding = -1 if padding_idx is None else int(padding_idx) % table.shape[0]
    lead, k = (idx.shape[:-1], idx.shape[-1]) if bag else (idx.shape, 1)
    if not bag and idx.dim() == 1 and idx.is_contiguous():
        idx = idx.unsqueeze(1)
    elif idx.dim() != 2 or not bag or not idx.is_contiguous():
        idx = idx.reshape(-1, k).contiguous()
    if weight is not None and (weight.dim() != 2 or not weight.is_contiguous()):
        weight = weight.reshape(-1, k).contiguous()
    out = _lib.host_module().embedding(table, weight, idx, scale, padding)
    return out if len(lead) == 1 else out.reshape(*lead, table.shape[1])


# ---------------------------------------------------------------------------------------------- the models' training forward
def training_state(module):
    """the DropoutState that use_in_training gave a module of this package; None in evaluation, also where evaluation is differentiated"""
    return module.block_state if module.training else None


def use_in_training(model, state):
    """Puts the training forward of a model of this package on the operators above: the SF-Phase decoder's and the TransVFE layers' residuals, dropouts and
    norms in one pass each, dropout (the decoder's and the heads' nn.Dropout) from `state`, a DropoutState, and the camera features' sampling on one
    weighted lookup.  The masks differ from torch's generator's (which still draws the class tokens' attention dropout inside nn.MultiheadAttention), everything
    else agrees to rounding; a module in evaluation mode is not touched, with gradients or without.  The training loop
    calls state.advance() after each backward pass.  state None: back to the torch composition.  -> model"""
    if state is not None and not isinstance(state, DropoutState):
        raise TypeError("use_in_training: a DropoutState or None needed, got %s" % type(state).__name__)
    for module in model.modules():
        if hasattr(type(module), "block_state"):
            module.block_state = state
        if type(module) is nn.Dropout and state is not None:  # the same object: its hooks and every other place that holds it stay with it
            module.__class__, module.converted = Dropout, True
        if isinstance(module, Dropout):
            module.state = state
            if state is None and module.converted:
                module.__class__, module.converted = nn.Dropout, False
    return model
