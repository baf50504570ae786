"""Symbolic graph layer: the TF-1.x graph-building calls the reference scripts make.

This is deliberately NOT a dataflow engine.  A ``Graph`` records variables,
placeholders and a small expression DAG so that (a) scripts written against the
reference's API (tfdist_between.py:33-75) build the same objects, names and
placements, and (b) the session can recognise the MLP training pattern and run
it on the fused HIP pipeline; everything else is evaluated op by op with
PyTorch (the soft-placement path).

Names follow TensorFlow: ``name_scope("weights")`` + ``Variable(...)`` gives
``weights/Variable`` then ``weights/Variable_1``; tensors are ``<op>:0``.
"""
from __future__ import annotations

import contextlib
import threading
from typing import Any, Callable, Dict, List, Optional, Sequence, Tuple, Union

import numpy as np

from .placement import DeviceSpec, ReplicaDeviceSetter
from .variables import VarSpec

float32 = "float32"
float64 = "float64"
int32 = "int32"
int64 = "int64"
bool_ = "bool"

_DTYPE_ALIASES = {float: float32, int: int32, bool: bool_, np.float32: float32, np.float64: float64,
                  np.int32: int32, np.int64: int64, "float": float32}


def as_dtype(d) -> str:
    if d is None:
        return float32
    return _DTYPE_ALIASES.get(d, d if isinstance(d, str) else str(np.dtype(d)))


class GraphKeys:
    GLOBAL_VARIABLES = "variables"
    TRAINABLE_VARIABLES = "trainable_variables"
    SUMMARIES = "summaries"
    GLOBAL_STEP = "global_step"


class Graph:
    def __init__(self):
        self.nodes: List["Tensor"] = []
        self.variables: List["Variable"] = []
        self.collections: Dict[str, list] = {}
        self.seed: Optional[int] = None
        self._name_counts: Dict[str, int] = {}
        self._scope: List[str] = []
        self._devices: List[Union[str, Callable]] = []
        self._lock = threading.Lock()
        self.finalized = False

    # -- naming -----------------------------------------------------------------
    def scope_prefix(self) -> str:
        return "/".join(self._scope) + "/" if self._scope else ""

    def unique_name(self, base: str, scoped: bool = True) -> str:
        full = (self.scope_prefix() if scoped else "") + base
        with self._lock:
            n = self._name_counts.get(full, 0)
            self._name_counts[full] = n + 1
        return full if n == 0 else f"{full}_{n}"

    # -- devices ------------------------------------------------------------------
    def device_for(self, kind: str, name: str, nbytes: int = 0) -> str:
        spec = DeviceSpec()
        for d in reversed(self._devices):   # innermost first
            if d is None:
                continue
            if isinstance(d, ReplicaDeviceSetter):
                s = DeviceSpec.from_string(d(kind, name, nbytes))
            elif callable(d):
                s = DeviceSpec.from_string(d(kind))
            else:
                s = DeviceSpec.from_string(d)
            spec = spec.merged_over(s)
        return spec.to_string()

    def add_to_collection(self, key: str, value):
        self.collections.setdefault(key, []).append(value)

    def get_collection(self, key: str) -> list:
        return list(self.collections.get(key, []))

    @contextlib.contextmanager
    def as_default(self):
        _graph_stack.append(self)
        try:
            yield self
        finally:
            _graph_stack.pop()

    def as_graph_def_bytes(self) -> bytes:
        """Minimal serialized GraphDef (NodeDef name/op/input/device) for the TensorBoard graph tab."""
        from .summary import encode_graph_def

        return encode_graph_def(self)


_graph_stack: List[Graph] = [Graph()]


def get_default_graph() -> Graph:
    return _graph_stack[-1]


def reset_default_graph():
    _graph_stack[-1] = Graph()


class Tensor:
    """A node of the expression DAG (one output)."""

    def __init__(self, op: str, inputs: Sequence["Tensor"] = (), attrs: Optional[Dict[str, Any]] = None,
                 name: Optional[str] = None, dtype: str = float32, shape: Optional[Tuple] = None,
                 graph: Optional[Graph] = None, kind: str = "op"):
        g = graph or (inputs[0].graph if inputs else get_default_graph())
        self.graph = g
        self.op = op
        self.inputs = tuple(inputs)
        self.attrs = attrs or {}
        self.op_name = g.unique_name(name or _default_op_name(op))
        self.dtype = dtype
        self.shape = None if shape is None else tuple(shape)
        self.device = g.device_for(kind, self.op_name, 0)
        self.id = len(g.nodes)
        g.nodes.append(self)

    @property
    def name(self) -> str:
        return self.op_name + ":0"

    def get_shape(self):
        return self.shape

    def __repr__(self):
        return f"<Tensor {self.name} op={self.op} shape={self.shape} dtype={self.dtype} device={self.device!r}>"

    def __hash__(self):
        return id(self)

    def __eq__(self, other):   # identity, like tf.Tensor
        return self is other

    # arithmetic sugar
    def __add__(self, o): return add(self, o)
    def __radd__(self, o): return add(o, self)
    def __sub__(self, o): return subtract(self, o)
    def __rsub__(self, o): return subtract(o, self)
    def __mul__(self, o): return multiply(self, o)
    def __rmul__(self, o): return multiply(o, self)
    def __truediv__(self, o): return divide(self, o)
    def __rtruediv__(self, o): return divide(o, self)
    def __neg__(self): return negative(self)
    def __matmul__(self, o): return matmul(self, o)

    def eval(self, feed_dict=None, session=None):
        from .session import get_default_session

        s = session or get_default_session()
        if s is None:
            raise RuntimeError("no default session")
        return s.run(self, feed_dict=feed_dict)


_OP_NAMES = {"const": "Const", "placeholder": "Placeholder", "random_normal": "random_normal", "zeros": "zeros",
             "ones": "ones", "matmul": "MatMul", "add": "Add", "sub": "Sub", "mul": "Mul", "div": "truediv",
             "neg": "Neg", "log": "Log", "exp": "Exp", "sigmoid": "Sigmoid", "relu": "Relu", "tanh": "Tanh",
             "softmax": "Softmax", "log_softmax": "LogSoftmax", "reduce_sum": "Sum", "reduce_mean": "Mean",
             "reduce_max": "Max", "argmax": "ArgMax", "equal": "Equal", "cast": "Cast", "square": "Square",
             "sqrt": "Sqrt", "reshape": "Reshape", "transpose": "transpose", "identity": "Identity",
             "softmax_xent": "SoftmaxCrossEntropyWithLogits", "variable": "Variable", "init_all": "init",
             "init_vars": "init", "group": "group_deps", "no_op": "NoOp", "train": "GradientDescent",
             "scalar_summary": "ScalarSummary", "merge_summary": "Merge/MergeSummary", "assign": "Assign",
             "assign_add": "AssignAdd", "stop_gradient": "StopGradient", "maximum": "Maximum", "minimum": "Minimum",
             "abs": "Abs", "greater": "Greater", "less": "Less", "embedding_lookup": "embedding_lookup",
             "sparse_softmax_xent": "SparseSoftmaxCrossEntropyWithLogits"}


def _default_op_name(op: str) -> str:
    return _OP_NAMES.get(op, op)


def convert_to_tensor(v, dtype=None) -> Tensor:
    if isinstance(v, Tensor):
        return v
    arr = np.asarray(v)
    if dtype is not None:
        arr = arr.astype(np.dtype(as_dtype(dtype)))
    elif arr.dtype == np.float64:
        arr = arr.astype(np.float32)
    return Tensor("const", (), {"value": arr}, dtype=str(arr.dtype), shape=arr.shape)


def constant(value, dtype=None, shape=None, name=None) -> Tensor:
    arr = np.asarray(value)
    if dtype is not None:
        arr = arr.astype(np.dtype(as_dtype(dtype)))
    elif arr.dtype == np.float64:
        arr = arr.astype(np.float32)
    if shape is not None:
        arr = np.broadcast_to(arr, shape).copy()
    return Tensor("const", (), {"value": arr}, name=name, dtype=str(arr.dtype), shape=arr.shape)


def placeholder(dtype=float32, shape=None, name=None) -> Tensor:
    return Tensor("placeholder", (), {}, name=name, dtype=as_dtype(dtype),
                  shape=None if shape is None else tuple(shape))


# -- scopes ------------------------------------------------------------------------
@contextlib.contextmanager
def name_scope(name: Optional[str], default_name=None, values=None):
    g = get_default_graph()
    if not name:
        yield ""
        return
    scope = name
    # TensorFlow uniquifies repeated scopes (weights, weights_1, ...)
    base = g.scope_prefix() + scope
    with g._lock:
        n = g._name_counts.get("scope:" + base, 0)
        g._name_counts["scope:" + base] = n + 1
    if n:
        scope = f"{scope}_{n}"
    g._scope.append(scope)
    try:
        yield g.scope_prefix()
    finally:
        g._scope.pop()


variable_scope = name_scope


@contextlib.contextmanager
def device(device_name_or_function):
    g = get_default_graph()
    g._devices.append(device_name_or_function)
    try:
        yield
    finally:
        g._devices.pop()


def set_random_seed(seed: Optional[int]):
    get_default_graph().seed = seed


# -- initial values / initializers ----------------------------------------------------
def random_normal(shape, mean=0.0, stddev=1.0, dtype=float32, seed=None, name=None) -> Tensor:
    return Tensor("random_normal", (), {"shape": tuple(int(s) for s in shape), "mean": float(mean),
                                        "stddev": float(stddev), "seed": seed}, name=name,
                  dtype=as_dtype(dtype), shape=tuple(shape))


def zeros(shape, dtype=float32, name=None) -> Tensor:
    return Tensor("zeros", (), {"shape": tuple(int(s) for s in shape)}, name=name, dtype=as_dtype(dtype),
                  shape=tuple(shape))


def ones(shape, dtype=float32, name=None) -> Tensor:
    return Tensor("ones", (), {"shape": tuple(int(s) for s in shape)}, name=name, dtype=as_dtype(dtype),
                  shape=tuple(shape))


class _Initializer:
    def __init__(self, spec: Tuple):
        self.spec = spec


def constant_initializer(value=0.0, dtype=float32):
    return _Initializer(("constant", float(value)))


def zeros_initializer(dtype=float32):
    return _Initializer(("zeros",))


def random_normal_initializer(mean=0.0, stddev=1.0, seed=None, dtype=float32):
    return _Initializer(("normal", float(mean), float(stddev)))


class Variable(Tensor):
    """A mutable tensor living on a parameter-server shard (or locally)."""

    def __init__(self, initial_value=None, trainable: bool = True, name: Optional[str] = None, dtype=None,
                 _init_spec: Optional[Tuple] = None, _shape: Optional[Tuple] = None, _scoped: bool = True):
        g = get_default_graph()
        if _init_spec is None:
            iv = convert_to_tensor(initial_value, dtype)
            if iv.op == "random_normal":
                _init_spec = ("normal", iv.attrs["mean"], iv.attrs["stddev"])
            elif iv.op == "zeros":
                _init_spec = ("zeros",)
            elif iv.op == "ones":
                _init_spec = ("constant", 1.0)
            elif iv.op == "const" and iv.attrs["value"].size == 1:
                _init_spec = ("constant", float(iv.attrs["value"].reshape(-1)[0]))
            elif iv.op == "const":
                _init_spec = ("value", iv.attrs["value"].astype(np.float32))
            else:
                raise ValueError(f"unsupported initial value op {iv.op!r} for a Variable")
            _shape = iv.shape
        if _shape is None:
            raise ValueError("variable shape must be known")
        self.graph = g
        self.op = "variable"
        self.inputs = ()
        self.attrs = {}
        base = name or "Variable"
        self.op_name = g.unique_name(base, scoped=_scoped)
        self.dtype = float32
        self.shape = tuple(int(s) for s in _shape)
        numel = int(np.prod(self.shape)) if self.shape else 1
        self.device = g.device_for("variable", self.op_name, 4 * numel)
        self.id = len(g.nodes)
        g.nodes.append(self)
        self.trainable = bool(trainable)
        self.spec = VarSpec(self.op_name, self.shape, _init_spec, self.trainable, index=len(g.variables),
                            device=self.device)
        dev = DeviceSpec.from_string(self.device)
        self.spec.shard = dev.task if (dev.job == "ps" and dev.task is not None) else 0
        g.variables.append(self)
        g.add_to_collection(GraphKeys.GLOBAL_VARIABLES, self)
        if self.trainable:
            g.add_to_collection(GraphKeys.TRAINABLE_VARIABLES, self)
        self.initializer = Tensor("init_vars", (), {"variables": [self]}, name=self.op_name.split("/")[-1] + "/Assign",
                                  kind="variable_init")

    def initialized_value(self):
        return self

    def assign(self, value):
        return assign(self, value)

    def assign_add(self, delta):
        return assign_add(self, delta)

    def read_value(self):
        return identity(self)


def get_variable(name: str, shape=None, dtype=float32, initializer=None, trainable: bool = True) -> Variable:
    g = get_default_graph()
    for v in g.variables:
        if v.op_name == name:
            return v
    if initializer is None:
        initializer = _Initializer(("normal", 0.0, 1.0)) if shape else _Initializer(("zeros",))
    if isinstance(initializer, Tensor):
        return Variable(initializer, trainable=trainable, name=name, _scoped=False)
    return Variable(trainable=trainable, name=name, _init_spec=initializer.spec,
                    _shape=tuple(shape or ()), _scoped=False)


def global_variables() -> List[Variable]:
    return list(get_default_graph().variables)


all_variables = global_variables


def trainable_variables() -> List[Variable]:
    return [v for v in get_default_graph().variables if v.trainable]


def global_variables_initializer() -> Tensor:
    return Tensor("init_all", (), {"variables": list(get_default_graph().variables)}, name="init",
                  kind="variable_init")


initialize_all_variables = global_variables_initializer


def variables_initializer(var_list, name="init") -> Tensor:
    return Tensor("init_vars", (), {"variables": list(var_list)}, name=name, kind="variable_init")


# -- ops ---------------------------------------------------------------------------------
def _t(x) -> Tensor:
    return convert_to_tensor(x)


def _bshape(a: Tensor, b: Tensor):
    if a.shape is None or b.shape is None:
        return None
    try:
        return tuple(np.broadcast_shapes(tuple(1 if d is None else d for d in a.shape),
                                         tuple(1 if d is None else d for d in b.shape)))
    except ValueError:
        return None


def matmul(a, b, transpose_a=False, transpose_b=False, name=None) -> Tensor:
    a, b = _t(a), _t(b)
    shape = None
    if a.shape is not None and b.shape is not None and len(a.shape) == 2 and len(b.shape) == 2:
        m = a.shape[1] if transpose_a else a.shape[0]
        n = b.shape[0] if transpose_b else b.shape[1]
        shape = (m, n)
    return Tensor("matmul", (a, b), {"transpose_a": transpose_a, "transpose_b": transpose_b}, name=name, shape=shape)


def _binary(op):
    def f(x, y, name=None) -> Tensor:
        x, y = _t(x), _t(y)
        out_dtype = bool_ if op in ("equal", "greater", "less") else x.dtype
        return Tensor(op, (x, y), {}, name=name, dtype=out_dtype, shape=_bshape(x, y))
    f.__name__ = op
    return f


add = _binary("add")
subtract = _binary("sub")
multiply = _binary("mul")
divide = _binary("div")
equal = _binary("equal")
greater = _binary("greater")
less = _binary("less")
maximum = _binary("maximum")
minimum = _binary("minimum")
sub, mul, div = subtract, multiply, divide


def _unary(op):
    def f(x, name=None) -> Tensor:
        x = _t(x)
        return Tensor(op, (x,), {}, name=name, dtype=x.dtype, shape=x.shape)
    f.__name__ = op
    return f


negative = _unary("neg")
neg = negative
log = _unary("log")
exp = _unary("exp")
sqrt = _unary("sqrt")
square = _unary("square")
abs = _unary("abs")  # noqa: A001
sigmoid = _unary("sigmoid")
tanh = _unary("tanh")
relu = _unary("relu")
identity = _unary("identity")
stop_gradient = _unary("stop_gradient")


def softmax(logits, dim=-1, name=None) -> Tensor:
    x = _t(logits)
    return Tensor("softmax", (x,), {"axis": dim}, name=name, dtype=x.dtype, shape=x.shape)


def log_softmax(logits, dim=-1, name=None) -> Tensor:
    x = _t(logits)
    return Tensor("log_softmax", (x,), {"axis": dim}, name=name, dtype=x.dtype, shape=x.shape)


def softmax_cross_entropy_with_logits(_sentinel=None, labels=None, logits=None, dim=-1, name=None) -> Tensor:
    labels, logits = _t(labels), _t(logits)
    shape = None if logits.shape is None else tuple(logits.shape[:-1])
    return Tensor("softmax_xent", (labels, logits), {}, name=name, dtype=logits.dtype, shape=shape)


def embedding_lookup(params, ids, name=None, scale: float = 1.0) -> Tensor:
    """``scale * params[ids]``: rows of a 2-D table for ids of any shape.  An id outside the table gives a row of zeros and has no
    gradient (padding).  ``params``: one table, or a list of one."""
    if isinstance(params, (list, tuple)):
        if len(params) != 1:
            raise ValueError("embedding_lookup: one table (a table dealt over several variables is not supported)")
        params = params[0]
    table, ids = _t(params), _t(ids)
    if table.shape is not None and len(table.shape) != 2:
        raise ValueError(f"embedding_lookup: the table must be a matrix, got shape {table.shape}")
    if ids.dtype not in (int32, int64):
        raise ValueError(f"embedding_lookup: ids must be int32 or int64, got {ids.dtype}")
    shape = None if table.shape is None or ids.shape is None else tuple(ids.shape) + (table.shape[1],)
    return Tensor("embedding_lookup", (table, ids), {"scale": float(scale)}, name=name, dtype=table.dtype, shape=shape)


def sparse_softmax_cross_entropy_with_logits(_sentinel=None, labels=None, logits=None, name=None) -> Tensor:
    """Loss of every row of ``logits [..., classes]`` against integer ``labels [...]``.  A negative label is padding: loss and gradient
    0; a label that is no class gives NaN."""
    labels, logits = _t(labels), _t(logits)
    if labels.dtype not in (int32, int64):
        raise ValueError(f"sparse_softmax_cross_entropy_with_logits: labels must be int32 or int64, got {labels.dtype}")
    shape = None if logits.shape is None else tuple(logits.shape[:-1])
    return Tensor("sparse_softmax_xent", (labels, logits), {}, name=name, dtype=logits.dtype, shape=shape)


def _axes(axis, reduction_indices):
    ax = axis if axis is not None else reduction_indices
    if ax is None:
        return None
    if isinstance(ax, (list, tuple)):
        return tuple(int(a) for a in ax)
    return (int(ax),)


def _reduce(op):
    def f(input_tensor, axis=None, keep_dims=False, name=None, reduction_indices=None, keepdims=None) -> Tensor:
        x = _t(input_tensor)
        kd = bool(keep_dims if keepdims is None else keepdims)
        return Tensor(op, (x,), {"axis": _axes(axis, reduction_indices), "keep_dims": kd}, name=name, dtype=x.dtype)
    f.__name__ = op
    return f


reduce_sum = _reduce("reduce_sum")
reduce_mean = _reduce("reduce_mean")
reduce_max = _reduce("reduce_max")


def argmax(input, axis=None, name=None, dimension=None) -> Tensor:  # noqa: A002
    x = _t(input)
    ax = axis if axis is not None else (dimension if dimension is not None else 0)
    return Tensor("argmax", (x,), {"axis": int(ax)}, name=name, dtype=int64)


def cast(x, dtype, name=None) -> Tensor:
    x = _t(x)
    return Tensor("cast", (x,), {"dtype": as_dtype(dtype)}, name=name, dtype=as_dtype(dtype), shape=x.shape)


def to_float(x, name="ToFloat") -> Tensor:
    return cast(x, float32, name=name)


def reshape(tensor, shape, name=None) -> Tensor:
    x = _t(tensor)
    return Tensor("reshape", (x,), {"shape": tuple(int(s) for s in shape)}, name=name, dtype=x.dtype)


def transpose(a, perm=None, name=None) -> Tensor:
    x = _t(a)
    return Tensor("transpose", (x,), {"perm": None if perm is None else tuple(perm)}, name=name, dtype=x.dtype)


def assign(ref: Variable, value, name=None) -> Tensor:
    return Tensor("assign", (ref, _t(value)), {}, name=name, dtype=ref.dtype, shape=ref.shape)


def assign_add(ref: Variable, delta, name=None) -> Tensor:
    return Tensor("assign_add", (ref, _t(delta)), {}, name=name, dtype=ref.dtype, shape=ref.shape)


def group(*inputs, name=None) -> Tensor:
    return Tensor("group", tuple(i for i in inputs if i is not None), {}, name=name)


def no_op(name=None) -> Tensor:
    return Tensor("no_op", (), {}, name=name)


class _NN:
    sigmoid = staticmethod(sigmoid)
    relu = staticmethod(relu)
    tanh = staticmethod(tanh)
    softmax = staticmethod(softmax)
    log_softmax = staticmethod(log_softmax)
    softmax_cross_entropy_with_logits = staticmethod(softmax_cross_entropy_with_logits)
    sparse_softmax_cross_entropy_with_logits = staticmethod(sparse_softmax_cross_entropy_with_logits)
    embedding_lookup = staticmethod(embedding_lookup)


nn = _NN()
