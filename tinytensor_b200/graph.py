"""Graph builders with the reference API (python/tinytensor/graph.py), producing the
node table the C ABI compiles (tt_graph in include/tt_cuda.h).

Shape rules and the exceptions they raise follow the reference builders
(src/graph/graph.cpp:51-200): NumPy broadcasting for binary ops, the batched matmul
rule, transpose axis normalisation, and reductions with optional keepdims.
Additional builders for ops the reference lacks: exp, neg, tanh, reduce_max, and the
sequence operators gated_scan, scan_last, token_logprob, policy_loss, preference_loss.
"""

import builtins
import ctypes
from collections.abc import Sequence

import numpy as np

from . import _lib
from ._lib import BroadcastError, DimensionError, IRError, ShapeError, TypeError

float32 = "float32"
float64 = "float64"
int32 = "int32"  # token ids: graph inputs read by the token operators
_DTYPE_CODE = {float32: 0, float64: 1, int32: 2}

__all__ = [
    "Graph", "Node", "float32", "float64", "int32", "add", "sub", "mul", "div", "relu", "sigmoid",
    "matmul", "sum", "mean", "max", "transpose", "exp", "neg", "tanh",
    "gated_scan", "scan_last", "token_logprob", "policy_loss", "preference_loss",
]


def broadcast_shapes(a, b):
    """Tensor::broadcast_shapes (src/core/tensor.cpp:189-215)."""
    r = builtins.max(len(a), len(b))
    out = []
    for i in range(r):
        da = a[i - (r - len(a))] if i >= r - len(a) else 1
        db = b[i - (r - len(b))] if i >= r - len(b) else 1
        if da != db and da != 1 and db != 1:
            raise BroadcastError(f"Shapes {list(a)} and {list(b)} are not broadcastable")
        out.append(db if da == 1 else da)
    return out


class Node:
    """A graph node (the Python face of tinytensor::Node)."""

    __slots__ = ("_graph", "index", "op", "shape", "dtype", "inputs", "id", "name", "dim0", "dim1",
                 "axes", "keepdims", "data", "expr", "attrs")

    def __init__(self, graph, op, shape, dtype, inputs=(), name=""):
        self._graph = graph
        self.index = len(graph._nodes)
        self.op = op
        self.shape = [int(d) for d in shape]
        self.dtype = dtype
        self.inputs = list(inputs)
        self.id = graph._next_id
        self.name = name
        self.dim0 = self.dim1 = 0
        self.axes = []
        self.keepdims = False
        self.data = None
        self.expr = None
        self.attrs = None  # sequence operators: their numbers (tt_op_attrs.f)

    def __add__(self, other):
        return self._graph.add(self, other)

    def __radd__(self, other):
        return self._graph.add(other, self)

    def __sub__(self, other):
        return self._graph.sub(self, other)

    def __rsub__(self, other):
        return self._graph.sub(other, self)

    def __mul__(self, other):
        return self._graph.mul(self, other)

    def __rmul__(self, other):
        return self._graph.mul(other, self)

    def __truediv__(self, other):
        return self._graph.div(self, other)

    def __rtruediv__(self, other):
        return self._graph.div(other, self)

    def __matmul__(self, other):
        return self._graph.matmul(self, other)

    def __neg__(self):
        return self._graph.neg(self)

    def __hash__(self):
        return id(self)

    def __eq__(self, other):
        return self is other

    def __repr__(self):
        return f"Node(id={self.id}, name='{self.name}', shape={self.shape}, dtype={self.dtype})"


class Graph:
    """Computation graph with the reference builder API."""

    def __init__(self):
        self._nodes = []
        self._inputs = []
        self._outputs = []
        self._next_id = 0
        self._version = 0

    # -- construction ------------------------------------------------------------------
    def _add(self, node):
        self._nodes.append(node)
        self._next_id = node.id + 1
        self._version += 1
        return node

    def _ensure(self, x):
        if isinstance(x, Node):
            if x._graph is not self:
                raise IRError("Node belongs to a different graph")
            return x
        return self.constant(x)

    def input(self, shape: Sequence[int], dtype=float32, name: str = "") -> Node:
        if dtype not in _DTYPE_CODE:
            raise TypeError(f"Unsupported dtype {dtype}")
        if any(int(d) < 0 for d in shape):
            raise IRError("Input shape has a negative dimension")
        if not name:
            name = f"input_{len(self._inputs)}"  # Graph::create_input (graph.cpp:22-33)
        n = self._add(Node(self, _lib.OP_INPUT, shape, dtype, name=name))
        self._inputs.append(n)
        return n

    def constant(self, value, name: str = "") -> Node:
        arr = np.array(value, dtype=np.float32, order="C")  # keeps 0-d scalars 0-d
        n = Node(self, _lib.OP_CONSTANT, arr.shape, float32, name=name or f"const_{self._next_id}")
        n.data = arr
        return self._add(n)

    def _binary(self, op, a, b):
        a, b = self._ensure(a), self._ensure(b)
        if a.dtype != b.dtype:
            raise TypeError(f"DType mismatch in {_OPNAME[op]}")
        return self._add(Node(self, op, broadcast_shapes(a.shape, b.shape), a.dtype, [a, b]))

    def _unary(self, op, a):
        a = self._ensure(a)
        return self._add(Node(self, op, a.shape, a.dtype, [a]))

    def add(self, a, b) -> Node:
        return self._binary(_lib.OP_ADD, a, b)

    def sub(self, a, b) -> Node:
        return self._binary(_lib.OP_SUB, a, b)

    def mul(self, a, b) -> Node:
        return self._binary(_lib.OP_MUL, a, b)

    def div(self, a, b) -> Node:
        return self._binary(_lib.OP_DIV, a, b)

    def relu(self, a) -> Node:
        return self._unary(_lib.OP_RELU, a)

    def sigmoid(self, a) -> Node:
        return self._unary(_lib.OP_SIGMOID, a)

    def exp(self, a) -> Node:
        return self._unary(_lib.OP_EXP, a)

    def neg(self, a) -> Node:
        return self._unary(_lib.OP_NEG, a)

    def tanh(self, a) -> Node:
        return self._unary(_lib.OP_TANH, a)

    def matmul(self, a, b) -> Node:
        """Graph::matmul shape rule (graph.cpp:89-127)."""
        a, b = self._ensure(a), self._ensure(b)
        if a.dtype != b.dtype:
            raise TypeError("DType mismatch in matmul")
        if len(a.shape) < 2 or len(b.shape) < 2:
            raise DimensionError("Unsupported ranks for matmul")
        ka, kb = a.shape[-1], b.shape[-2]
        if ka != kb:
            raise ShapeError(f"Matmul inner dimensions mismatch: {ka} vs {kb}")
        batch = []
        if len(a.shape) > 2 or len(b.shape) > 2:
            batch = broadcast_shapes(a.shape[:-2], b.shape[:-2])
        return self._add(Node(self, _lib.OP_MATMUL, batch + [a.shape[-2], b.shape[-1]], a.dtype, [a, b]))

    def transpose(self, a, dim0: int, dim1: int) -> Node:
        a = self._ensure(a)
        r = len(a.shape)
        d0 = dim0 + r if dim0 < 0 else dim0
        d1 = dim1 + r if dim1 < 0 else dim1
        if not (0 <= d0 < r and 0 <= d1 < r):
            raise DimensionError(f"Invalid transpose axes for rank {r}")
        shape = list(a.shape)
        shape[d0], shape[d1] = shape[d1], shape[d0]
        n = Node(self, _lib.OP_TRANSPOSE, shape, a.dtype, [a])
        n.dim0, n.dim1 = d0, d1
        return self._add(n)

    def _reduce(self, op, a, axes, keepdims):
        a = self._ensure(a)
        r = len(a.shape)
        axes = [] if axes is None else [int(x) for x in axes]
        if not axes:
            norm = set(range(r))
        else:
            norm = set()
            for ax in axes:
                x = ax + r if ax < 0 else ax
                if not 0 <= x < r:
                    raise DimensionError(f"Axis out of range in {_OPNAME[op]}")
                norm.add(x)
        shape = []
        for i in range(r):
            if i in norm:
                if keepdims:
                    shape.append(1)
            else:
                shape.append(a.shape[i])
        n = Node(self, op, shape, a.dtype, [a])
        n.axes = axes
        n.keepdims = bool(keepdims)
        return self._add(n)

    def reduce_sum(self, a, axes=None, keepdims: bool = False) -> Node:
        return self._reduce(_lib.OP_REDUCE_SUM, a, axes, keepdims)

    def reduce_mean(self, a, axes=None, keepdims: bool = False) -> Node:
        return self._reduce(_lib.OP_REDUCE_MEAN, a, axes, keepdims)

    def reduce_max(self, a, axes=None, keepdims: bool = False) -> Node:
        return self._reduce(_lib.OP_REDUCE_MAX, a, axes, keepdims)

    def _expand(self, a, shape):
        a = self._ensure(a)
        if a.shape == shape:
            return a
        if broadcast_shapes(a.shape, shape) != shape:
            raise BroadcastError(f"Shape {a.shape} does not broadcast to {shape}")
        return self._add(Node(self, _lib.OP_EXPAND, shape, a.dtype, [a]))

    def _float32(self, what, *nodes):
        for n in nodes:
            if n.dtype != float32:
                raise TypeError(f"{what} takes float32 operands, got {n.dtype}")

    def gated_scan(self, gate, x, init=None, axis: int = -2) -> Node:
        """Gated linear recurrence h[t] = gate[t] * h[t-1] + x[t] along `axis`, from h[-1] = init
        (zeros when None).  gate and x broadcast together; init broadcasts to their shape
        without the axis.  The gradient reaches all three.  One step (an axis of size 1)
        with the last state as init is the form for serving one token at a time; a gate
        of 0 starts anew there, e.g. at a document's first token.  A state that is NaN stays
        NaN, an infinite one infinite or NaN, through gates of 0 too (0 * inf).  Gates may have any
        size; where their products overflow, or underflow beside states above 10^6, the lanes
        are walked step by step, which is slower."""
        gate, x = self._ensure(gate), self._ensure(x)
        self._float32("gated_scan", gate, x)
        shape = broadcast_shapes(gate.shape, x.shape)
        r = len(shape)
        ax = axis + r if axis < 0 else axis
        if not 0 <= ax < r:
            raise DimensionError(f"Invalid gated_scan axis {axis} for rank {r}")
        ins = [self._expand(gate, shape), self._expand(x, shape)]
        if init is not None:
            init = self._ensure(init)
            self._float32("gated_scan", init)
            ins.append(self._expand(init, shape[:ax] + shape[ax + 1:]))
        n = Node(self, _lib.OP_GATED_SCAN, shape, float32, ins)
        n.dim0 = ax
        n.attrs = ()
        return self._add(n)

    def scan_last(self, h) -> Node:
        """The state after the last step of gated_scan's result `h` (init, or zeros, when there
        are no steps): the next window's init.  When only it is used, the states in between
        are not stored."""
        h = self._ensure(h)
        if h.op != _lib.OP_GATED_SCAN:
            raise IRError("scan_last takes the result of a gated_scan")
        return self._add(Node(self, _lib.OP_SCAN_LAST, h.shape[:h.dim0] + h.shape[h.dim0 + 1:], h.dtype, [h]))

    def _token_operands(self, what, logits, tokens, rank=None):
        logits, tokens = self._ensure(logits), self._ensure(tokens)
        self._float32(what, logits)
        if tokens.dtype != int32:
            raise TypeError(f"{what} takes int32 tokens, got {tokens.dtype}")
        if not logits.shape:
            raise DimensionError(f"{what} needs logits of rank 1 or more")
        if logits.shape[-1] == 0:
            raise ShapeError(f"{what} needs a vocabulary of at least one token")
        if logits.shape[-1] > 2**30:
            raise ShapeError(f"{what} takes a vocabulary of at most 2^30 tokens")
        if rank is not None and (len(logits.shape) != rank or logits.shape[-3] != 2):
            raise ShapeError(f"{what} needs logits [pairs, 2, tokens, vocabulary], got {logits.shape}")
        if tokens.shape != logits.shape[:-1]:
            raise ShapeError(f"{what}: tokens {tokens.shape} do not go with logits {logits.shape}")
        return logits, tokens

    def _token_node(self, op, shape, ins, attrs):
        n = Node(self, op, shape, float32, ins)
        n.attrs = tuple(float(a) for a in attrs)
        return self._add(n)

    def token_logprob(self, logits, tokens) -> Node:
        """log softmax(logits)[token] for logits [..., V] and int32 tokens [...].

        Padding is a negative token: its logits are not read (whatever they hold), its value
        and its gradient are 0.  A token of V or more gives NaN and DeviceStatusError.  With
        seed = -weights it is the cross-entropy's gradient.  Programs with a gradient and without
        one round differently: the same value from both differs in its last bits."""
        logits, tokens = self._token_operands("token_logprob", logits, tokens)
        return self._token_node(_lib.OP_TOKEN_LOGPROB, tokens.shape, [logits, tokens], ())

    def policy_loss(self, logits, tokens, old_logp, advantage, ref_logp=None, clip=(0.2, 0.2), kl: float = 0.0) -> Node:
        """Clipped policy loss of every token, with a KL term to a reference policy:

            r = exp(p - old_logp),  p = token_logprob(logits, tokens)
            -min(r * advantage, clamp(r, 1 - clip[0], 1 + clip[1]) * advantage)
              + kl * (exp(ref_logp - p) - (ref_logp - p) - 1)

        old_logp, advantage and ref_logp broadcast to the tokens' shape and count as data:
        the gradient reaches the logits only.  kl > 0 takes ref_logp, kl = 0 does not.  With
        old_logp from a program of its own, r of the same policy is 1 up to that rounding.
        Padding as in token_logprob, whatever the other operands hold there."""
        logits, tokens = self._token_operands("policy_loss", logits, tokens)
        if len(clip) != 2 or not 0.0 <= clip[0] <= 1.0 or not 0.0 <= clip[1] < float("inf"):
            raise ValueError("clip must be (lower in [0, 1], upper >= 0)")
        if not 0.0 <= kl < float("inf"):
            raise ValueError("kl must be finite and not negative")
        if (ctypes.c_float(kl).value > 0.0) != (ref_logp is not None):
            raise ValueError("ref_logp goes with kl > 0, and only with it")
        data = [old_logp, advantage] + ([] if ref_logp is None else [ref_logp])
        data = [self._ensure(d) for d in data]
        self._float32("policy_loss", *data)
        ins = [logits, tokens] + [self._expand(d, tokens.shape) for d in data]
        return self._token_node(_lib.OP_POLICY_LOSS, tokens.shape, ins, (clip[0], clip[1], kl))

    def preference_loss(self, logits, tokens, ref_logp, beta: float = 0.1, smoothing: float = 0.0) -> Node:
        """Preference loss of answer pairs: logits [N, 2, T, V] and tokens [N, 2, T] of the chosen
        (0) and the rejected (1) answer, ref_logp (broadcast to the tokens' shape) the tokens'
        log-probabilities under the reference.  Per pair, with S(j) the sum of token_logprob -
        ref_logp over answer j's tokens and z = beta * (S(0) - S(1)):

            -(1 - smoothing) * log sigmoid(z) - smoothing * log sigmoid(-z)

        The gradient reaches the logits only.  Padding as in token_logprob; an answer of
        padding alone has S = 0."""
        logits, tokens = self._token_operands("preference_loss", logits, tokens, rank=4)
        if not 0.0 < beta < float("inf"):
            raise ValueError("beta must be finite and positive")
        if not 0.0 <= smoothing <= 0.5:
            raise ValueError("smoothing must lie in [0, 0.5]")
        ref = self._ensure(ref_logp)
        self._float32("preference_loss", ref)
        ins = [logits, tokens, self._expand(ref, tokens.shape)]
        return self._token_node(_lib.OP_PREFERENCE_LOSS, tokens.shape[:1], ins, (beta, smoothing))

    def mark_output(self, node: Node) -> None:
        if node is None:
            raise IRError("Cannot mark null node as output")
        if node not in self._outputs:
            self._outputs.append(node)
            self._version += 1

    @property
    def inputs(self):
        return list(self._inputs)

    @property
    def outputs(self):
        return list(self._outputs)

    @property
    def nodes(self):
        return list(self._nodes)

    # -- C ABI image ---------------------------------------------------------------------
    def _to_c(self, outputs=None):
        """Returns (TTGraph, keepalive) describing this graph for the C ABI."""
        nodes = (_lib.TTNode * builtins.max(1, len(self._nodes)))()
        keep = []
        for i, n in enumerate(self._nodes):
            c = nodes[i]
            c.op = n.op
            c.dtype = _DTYPE_CODE[n.dtype]
            c.num_inputs = len(n.inputs)
            for k, q in enumerate(n.inputs[:_lib.TT_MAX_NODE_INPUTS]):
                c.inputs[k] = q.index
            if n.attrs is not None:
                at = _lib.TTOpAttrs()
                for k, q in enumerate(n.inputs[_lib.TT_MAX_NODE_INPUTS:]):
                    at.more_inputs[k] = q.index
                for k, f in enumerate(n.attrs):
                    at.f[k] = f
                keep.append(at)
                c.data = ctypes.addressof(at)
            if len(n.shape) > _lib.TT_MAX_RANK:
                raise DimensionError(f"rank {len(n.shape)} exceeds {_lib.TT_MAX_RANK}")
            c.rank = len(n.shape)
            for k, d in enumerate(n.shape):
                c.shape[k] = d
            c.id = n.id
            c.dim0, c.dim1 = n.dim0, n.dim1
            c.num_axes = len(n.axes)
            for k, ax in enumerate(n.axes):
                c.axes[k] = ax
            c.keepdims = int(n.keepdims)
            if n.data is not None:
                keep.append(n.data)
                c.data = n.data.ctypes.data
            if n.name:
                b = n.name.encode()
                keep.append(b)
                c.name = b
            if n.expr:
                b = n.expr.encode()
                keep.append(b)
                c.expr = b
        outs = self._outputs if outputs is None else outputs
        ins = (ctypes.c_int32 * builtins.max(1, len(self._inputs)))(*[n.index for n in self._inputs])
        outa = (ctypes.c_int32 * builtins.max(1, len(outs)))(*[n.index for n in outs])
        keep += [nodes, ins, outa]
        g = _lib.TTGraph(len(self._nodes), nodes, len(self._inputs), ins, len(outs), outa)
        return g, keep

    def to_ir(self) -> str:
        """Canonical IR text (IRPrinter::to_string format)."""
        g, keep = self._to_c()
        return _lib.cstr(_lib.lib.tt_graph_ir, ctypes.byref(g))


_OPNAME = {
    _lib.OP_ADD: "add", _lib.OP_SUB: "sub", _lib.OP_MUL: "mul", _lib.OP_DIV: "div",
    _lib.OP_REDUCE_SUM: "reduce_sum", _lib.OP_REDUCE_MEAN: "reduce_mean", _lib.OP_REDUCE_MAX: "reduce_max",
}


def _graph_of(a, b=None):
    if isinstance(a, Node):
        return a._graph
    if isinstance(b, Node):
        return b._graph
    raise TypeError("At least one operand must be a Node")


def add(a, b):
    return _graph_of(a, b).add(a, b)


def sub(a, b):
    return _graph_of(a, b).sub(a, b)


def mul(a, b):
    return _graph_of(a, b).mul(a, b)


def div(a, b):
    return _graph_of(a, b).div(a, b)


def matmul(a, b):
    return _graph_of(a, b).matmul(a, b)


def _unary_node(a):
    if not isinstance(a, Node):
        raise TypeError("Operand must be a Node")
    return a._graph


def relu(a):
    return _unary_node(a).relu(a)


def sigmoid(a):
    return _unary_node(a).sigmoid(a)


def exp(a):
    return _unary_node(a).exp(a)


def neg(a):
    return _unary_node(a).neg(a)


def tanh(a):
    return _unary_node(a).tanh(a)


def sum(a, axes=None, keepdims=False):  # noqa: A001 - reference name
    return _unary_node(a).reduce_sum(a, axes, keepdims)


def mean(a, axes=None, keepdims=False):
    return _unary_node(a).reduce_mean(a, axes, keepdims)


def max(a, axes=None, keepdims=False):  # noqa: A001 - mirrors sum/mean
    return _unary_node(a).reduce_max(a, axes, keepdims)


def transpose(a, dim0, dim1):
    return _unary_node(a).transpose(a, dim0, dim1)


def gated_scan(gate, x, init=None, axis=-2):
    return _graph_of(gate, x).gated_scan(gate, x, init, axis)


def scan_last(h):
    return _unary_node(h).scan_last(h)


def token_logprob(logits, tokens):
    return _graph_of(logits, tokens).token_logprob(logits, tokens)


def policy_loss(logits, tokens, old_logp, advantage, ref_logp=None, clip=(0.2, 0.2), kl=0.0):
    return _graph_of(logits, tokens).policy_loss(logits, tokens, old_logp, advantage, ref_logp, clip, kl)


def preference_loss(logits, tokens, ref_logp, beta=0.1, smoothing=0.0):
    return _graph_of(logits, tokens).preference_loss(logits, tokens, ref_logp, beta, smoothing)
