"""Graph-building surface for the B200 transformer.

Mirrors the part of the reference's `ng.*` op surface that the hot path uses
(ngraph/__init__.py:23-89, ngraph/op_graph/op_graph.py, ngraph/op_graph/axes.py): named axes,
placeholders / variables / constants, elementwise ops with broadcasting by axis name,
reductions, dot, convolution, pooling, assign and sequential.  Names, argument meaning and error
behaviour follow the reference so that tests read like the reference's own; autodiff, serde and
the frontends are not part of this package.
"""
import itertools
import numbers

import numpy as np

_axis_counter = itertools.count()


class Axis(object):
    """A named dimension (ngraph/op_graph/axes.py: make_axis).  Two axes match when name and
    length are equal."""

    def __init__(self, length, name=None):
        if name is None:
            name = "Axis_%d" % next(_axis_counter)
        self.name = name
        self._length = None if length is None else int(length)

    @property
    def length(self):
        return self._length

    @length.setter
    def length(self, value):
        self._length = int(value)

    @property
    def is_batch(self):
        return self.name == "N"

    def named(self, name):
        return Axis(self.length, name)

    def __eq__(self, other):
        return isinstance(other, Axis) and self.name == other.name and self.length == other.length

    def __ne__(self, other):
        return not self == other

    def __hash__(self):
        return hash((self.name, self._length))

    def __repr__(self):
        return "Axis(%s: %s)" % (self.name, self._length)


def make_axis(length=None, name=None, **kw):
    return Axis(length, name)


class Axes(object):
    """An ordered collection of axes (ngraph/op_graph/axes.py: Axes)."""

    def __init__(self, axes=None):
        if axes is None:
            axes = ()
        elif isinstance(axes, Axis):
            axes = (axes,)
        elif isinstance(axes, Axes):
            axes = axes._axes
        axes = tuple(axes)
        for a in axes:
            if not isinstance(a, Axis):
                raise ValueError("Axes must contain Axis objects, got %r" % (a,))
        names = [a.name for a in axes]
        if len(set(names)) != len(names):
            raise ValueError("The axes labels of a tensor cannot contain duplicates: %s" % names)
        self._axes = axes

    def __iter__(self):
        return iter(self._axes)

    def __len__(self):
        return len(self._axes)

    def __getitem__(self, i):
        if isinstance(i, slice):
            return Axes(self._axes[i])
        return self._axes[i]

    def __add__(self, other):
        other = make_axes(other)
        return Axes(self._axes + tuple(a for a in other if a not in self._axes))

    def __sub__(self, other):
        other = make_axes(other)
        return Axes(a for a in self._axes if a not in other._axes)

    def __and__(self, other):
        other = make_axes(other)
        return Axes(a for a in self._axes if a in other._axes)

    def __eq__(self, other):
        return isinstance(other, Axes) and self._axes == other._axes

    def __ne__(self, other):
        return not self == other

    def __hash__(self):
        return hash(self._axes)

    def __contains__(self, a):
        return a in self._axes

    def __repr__(self):
        return "Axes(%s)" % ", ".join("%s: %s" % (a.name, a.length) for a in self._axes)

    def index(self, a):
        return self._axes.index(a)

    def find_by_name(self, name):
        return Axes(a for a in self._axes if a.name == name)

    def is_equal_set(self, other):
        return set(self._axes) == set(make_axes(other)._axes)

    def is_sub_set(self, other):
        return set(self._axes) <= set(make_axes(other)._axes)

    @property
    def lengths(self):
        return tuple(a.length for a in self._axes)

    @property
    def size(self):
        return int(np.prod(self.lengths, dtype=np.int64)) if self._axes else 1

    def batch_axis(self):
        for a in self._axes:
            if a.is_batch:
                return a
        return None


def make_axes(axes=()):
    if isinstance(axes, Axes):
        return axes
    return Axes(axes)


# ---------------------------------------------------------------------------------------------
class Op(object):
    """Base of all graph nodes."""
    _counter = itertools.count()

    def __init__(self, args=(), axes=(), name=None, metadata=None):
        self.args = tuple(as_op(a) for a in args)
        self.axes = make_axes(axes)
        self.uid = next(Op._counter)
        self.name = name or "%s_%d" % (type(self).__name__, self.uid)
        self.metadata = dict(metadata or {})
        self.control_deps = []

    is_tensor_op = True
    is_device_op = True

    @property
    def shape(self):
        return self.axes.lengths

    def add_control_dep(self, op):
        if op is not self and op not in self.control_deps:
            self.control_deps.append(op)

    @property
    def all_deps(self):
        return list(self.args) + list(self.control_deps)

    # arithmetic sugar, as on the reference's TensorOp
    def __neg__(self):
        return negative(self)

    def __pos__(self):
        return self

    def __abs__(self):
        return absolute(self)

    def __add__(self, o):
        return add(self, o)

    def __radd__(self, o):
        return add(o, self)

    def __sub__(self, o):
        return subtract(self, o)

    def __rsub__(self, o):
        return subtract(o, self)

    def __mul__(self, o):
        return multiply(self, o)

    def __rmul__(self, o):
        return multiply(o, self)

    def __truediv__(self, o):
        return divide(self, o)

    def __rtruediv__(self, o):
        return divide(o, self)

    __div__ = __truediv__
    __rdiv__ = __rtruediv__

    def __pow__(self, o):
        return power(self, o)

    def __rpow__(self, o):
        return power(o, self)

    __hash__ = object.__hash__

    def __repr__(self):
        return "<%s %s %s>" % (type(self).__name__, self.name, self.axes)


class AssignableTensorOp(Op):
    """placeholder / variable / persistent tensor / constant
    (ngraph/op_graph/op_graph.py: AssignableTensorOp)."""
    is_device_op = False

    def __init__(self, axes, initial_value=None, is_input=False, is_persistent=False,
                 is_constant=False, is_trainable=False, is_placeholder=False, **kw):
        super(AssignableTensorOp, self).__init__((), axes, **kw)
        self.is_input = is_input
        self.is_persistent = is_persistent
        self.is_constant = is_constant
        self.is_trainable = is_trainable
        self.is_placeholder = is_placeholder
        if initial_value is not None and not callable(initial_value):
            initial_value = np.asarray(initial_value, dtype=np.float32)
            lengths = tuple(self.axes.lengths)
            if initial_value.shape not in ((), lengths):
                # the same elements up to axes of length 1, or a value that numpy broadcasts to
                # the axes (the reference hands initial values to numpy the same way)
                if tuple(n for n in initial_value.shape if n != 1) == \
                        tuple(n for n in lengths if n != 1):
                    initial_value = initial_value.reshape(lengths)
                else:
                    try:
                        initial_value = np.ascontiguousarray(np.broadcast_to(initial_value, lengths))
                    except ValueError:
                        raise ValueError("initial value shape %s does not match axes %s" %
                                         (initial_value.shape, self.axes))
        self.initial_value = initial_value

    @property
    def is_scalar_constant(self):
        return self.is_constant and len(self.axes) == 0

    def initial_array(self):
        v = self.initial_value
        if v is None:
            return None
        if callable(v):
            v = np.asarray(v(self.axes), dtype=np.float32)
        return np.ascontiguousarray(np.broadcast_to(v, self.axes.lengths), dtype=np.float32)


def placeholder(axes, dtype=None, initial_value=None, **kw):
    return AssignableTensorOp(make_axes(axes), initial_value, is_input=True, is_persistent=True,
                              is_placeholder=True, **kw)


def variable(axes, dtype=None, initial_value=None, **kw):
    return AssignableTensorOp(make_axes(axes), initial_value, is_input=True, is_persistent=True,
                              is_trainable=True, **kw)


def persistent_tensor(axes, dtype=None, initial_value=None, **kw):
    return AssignableTensorOp(make_axes(axes), initial_value, is_persistent=True, **kw)


def temporary(axes, dtype=None, initial_value=None, **kw):
    return AssignableTensorOp(make_axes(axes), initial_value, **kw)


def constant(const, axes=None, dtype=None, **kw):
    const = np.asarray(const, dtype=np.float32)
    if axes is None:
        if const.ndim:
            raise ValueError("a non-scalar constant needs axes")
        axes = ()
    return AssignableTensorOp(make_axes(axes), const, is_constant=True, is_persistent=True, **kw)


def as_op(x):
    if isinstance(x, Op):
        return x
    if isinstance(x, (numbers.Number, np.number, np.bool_)) or \
            (isinstance(x, np.ndarray) and x.ndim == 0):
        return constant(float(x))
    raise ValueError("cannot use %r as a graph op" % (x,))


def as_ops(xs):
    return tuple(as_op(x) for x in xs)


# ---- views ----------------------------------------------------------------------------------
class ViewOp(Op):
    """Ops that re-describe their argument's storage without moving data (the reference's
    IndexOp family, ngraph/op_graph/op_graph.py:1650-1715)."""
    is_device_op = False


class BroadcastOp(ViewOp):
    def __init__(self, x, axes, **kw):
        x = as_op(x)
        axes = make_axes(axes)
        if not x.axes.is_sub_set(axes):
            raise ValueError("The new axes %s are not a superset of the op's axes %s" %
                             (axes, x.axes))
        super(BroadcastOp, self).__init__((x,), axes, **kw)


class ReorderAxes(ViewOp):
    def __init__(self, x, axes, **kw):
        x = as_op(x)
        axes = make_axes(axes)
        if not x.axes.is_equal_set(axes):
            raise ValueError("The input axes %s and output axes %s must have the same members" %
                             (x.axes, axes))
        super(ReorderAxes, self).__init__((x,), axes, **kw)


class AxesCastOp(ViewOp):
    """Same storage, new axes position by position (ngraph/op_graph/op_graph.py: AxesCastOp)."""

    def __init__(self, x, axes, **kw):
        x = as_op(x)
        axes = make_axes(axes)
        if x.axes.lengths != axes.lengths:
            raise ValueError("casting axes {} must have the same length as original axes {}"
                             .format(axes, x.axes))
        super(AxesCastOp, self).__init__((x,), axes, **kw)


class ReshapeOp(ViewOp):
    """The same elements in the same order under other axes: neighbouring axes merged into one or
    one axis split into several (the reference's Flatten / Unflatten,
    ngraph/op_graph/op_graph.py:2221-2294, whose FlattenedAxis has the product of its members'
    lengths).  No data moves; the argument's storage must allow it (a dense tensor always does)."""

    def __init__(self, x, axes, **kw):
        x = as_op(x)
        axes = make_axes(axes)
        if x.axes.size != axes.size:
            raise ValueError("reshape from {} to {} changes the number of elements"
                             .format(x.axes, axes))
        super(ReshapeOp, self).__init__((x,), axes, **kw)


def reshape(x, axes):
    x = as_op(x)
    axes = make_axes(axes)
    if x.axes == axes:
        return x
    return ReshapeOp(x, axes)


class TensorSliceOp(ViewOp):
    """A sliced view: one slice or int per axis of x; an int drops the axis
    (ngraph/op_graph/op_graph.py:2067-2120).  Negative steps are not supported, as there."""

    def __init__(self, x, slices, axes=None, **kw):
        x = as_op(x)
        slices = tuple(slices)
        if len(slices) != len(x.axes):
            raise ValueError("There should be one slice in slices for each dimension in input "
                             "tensor.  Input tensor had {} dimensions, but slices has length {}."
                             .format(len(x.axes), len(slices)))
        kept, starts, steps = [], [], []
        for axis, sl in zip(x.axes, slices):
            if isinstance(sl, slice):
                if sl.step is not None and sl.step < 0:
                    raise ValueError("Negative slice steps are not supported.")
                start, stop, step = sl.indices(axis.length)
                n = -(-(stop - start) // step)        # (max / min are reductions in this module)
                n = n if n > 0 else 0
                kept.append(axis if (start, n, step) == (0, axis.length, 1)
                            else make_axis(n, name=axis.name))
                starts.append(start)
                steps.append(step)
            else:
                idx = int(sl)
                if idx < 0:
                    idx += axis.length
                if not 0 <= idx < axis.length:
                    raise ValueError("index %d is out of range for axis %s" % (int(sl), axis))
                starts.append(idx)
                steps.append(None)          # the axis is dropped
        if axes is None:
            axes = kept
        axes = make_axes(axes)
        if axes.lengths != make_axes(kept).lengths:
            raise ValueError("slice result has shape %s, the given axes %s"
                             % (make_axes(kept).lengths, axes.lengths))
        super(TensorSliceOp, self).__init__((x,), axes, **kw)
        self.slices = slices
        self.starts = tuple(starts)
        self.steps = tuple(steps)


def tensor_slice(x, slices, axes=None):
    return TensorSliceOp(x, slices, axes)


def cast_axes(tensor, axes):
    tensor = as_op(tensor)
    axes = make_axes(axes)
    if tensor.axes == axes:
        return tensor
    return AxesCastOp(tensor, axes)


def broadcast(x, axes):
    x = as_op(x)
    axes = make_axes(axes)
    if x.axes == axes:
        return x
    return BroadcastOp(x, axes)


def axes_with_order(x, axes):
    x = as_op(x)
    axes = make_axes(axes)
    if x.axes == axes:
        return x
    return ReorderAxes(x, axes)


# ---- elementwise ------------------------------------------------------------------------------
class ElementWiseOp(Op):
    def __init__(self, opname, args, **kw):
        args = as_ops(args)
        axes = Axes()
        for a in args:
            axes = axes + a.axes
        super(ElementWiseOp, self).__init__(args, axes, **kw)
        self.opname = opname


def _unary(opname):
    def build(x, **kw):
        return ElementWiseOp(opname, (x,), **kw)
    build.__name__ = opname
    return build


def _binary(opname):
    def build(x, y, dtype=None, **kw):
        return ElementWiseOp(opname, (x, y), **kw)
    build.__name__ = opname
    return build


negative = _unary("neg")
absolute = _unary("abs")
sin = _unary("sin")
cos = _unary("cos")
tanh = _unary("tanh")
exp = _unary("exp")
log = _unary("log")
reciprocal = _unary("rcp")
sign = _unary("sgn")
square = _unary("sqr")
sqrt = _unary("sqrt")
sigmoidAtomic = _unary("sig")

add = _binary("add")
subtract = _binary("sub")
multiply = _binary("mul")
divide = _binary("div")
floordivide = _binary("int_div")
mod = _binary("mod")
maximum = _binary("maximum")
minimum = _binary("minimum")
power = _binary("pow")
equal = _binary("eq")
not_equal = _binary("ne")
greater = _binary("gt")
less = _binary("lt")
greater_equal = _binary("ge")
less_equal = _binary("le")


safelog_cutoff = 50.0


def safelog(x, limit=-safelog_cutoff):
    """maximum(log(x + exp(limit)), limit) (ngraph/op_graph/op_graph.py:3067-3072)."""
    return maximum(log(x + float(np.exp(limit))), limit)


def sigmoid(x):
    """reciprocal(exp(-x) + 1), as the reference composes it
    (ngraph/op_graph/op_graph.py:4183-4199)."""
    return reciprocal(exp(negative(x)) + 1)


# ---- reductions -------------------------------------------------------------------------------
def compute_reduction_axes(x, reduction_axes, out_axes):
    """ngraph/op_graph/op_graph.py: compute_reduction_axes."""
    if reduction_axes is None and out_axes is None:
        reduction_axes = x.axes - x.axes.find_by_name("N")   # sample axes
        out_axes = x.axes - reduction_axes
    elif reduction_axes is None:
        out_axes = make_axes(out_axes)
        reduction_axes = x.axes - out_axes
    elif out_axes is None:
        reduction_axes = make_axes(reduction_axes)
        out_axes = x.axes - reduction_axes
    else:
        out_axes = make_axes(out_axes)
        reduction_axes = make_axes(reduction_axes)
    if not reduction_axes.is_sub_set(x.axes):
        raise ValueError("reduction axes %s are not axes of the operand %s" %
                         (reduction_axes, x.axes))
    return reduction_axes, out_axes


class ReductionOp(Op):
    def __init__(self, redop, x, reduction_axes=None, out_axes=None, **kw):
        x = as_op(x)
        reduction_axes, out_axes = compute_reduction_axes(x, reduction_axes, out_axes)
        super(ReductionOp, self).__init__((x,), out_axes, **kw)
        self.redop = redop
        self.reduction_axes = reduction_axes


def _reduction(redop):
    def build(x, reduction_axes=None, out_axes=None, dtype=None, **kw):
        return ReductionOp(redop, x, reduction_axes, out_axes, **kw)
    build.__name__ = redop
    return build


sum = _reduction("sum")          # noqa: A001  (the reference shadows the builtins the same way)
prod = _reduction("prod")
max = _reduction("max")          # noqa: A001
min = _reduction("min")          # noqa: A001
argmax = _reduction("argmax")
argmin = _reduction("argmin")


def mean(x, reduction_axes=None, out_axes=None):
    """ngraph/op_graph/op_graph.py:4252-4266."""
    x = as_op(x)
    reduction_axes, out_axes = compute_reduction_axes(x, reduction_axes, out_axes)
    return sum(x, reduction_axes=reduction_axes, out_axes=out_axes) / float(reduction_axes.size)


def variance(x, out_axes=None, reduction_axes=None):
    """ngraph/op_graph/op_graph.py:4007-4009: mean of the squared distance from the mean."""
    x = as_op(x)
    return mean(square(x - mean(x, reduction_axes=reduction_axes, out_axes=out_axes)),
                reduction_axes=reduction_axes, out_axes=out_axes)


def softmax(x, normalization_axes=None, **kw):
    """ngraph/op_graph/op_graph.py: SoftmaxOp -- exp(x - max) / sum(exp(x - max))."""
    x = as_op(x)
    if normalization_axes is None:
        normalization_axes = x.axes - x.axes.find_by_name("N")
    normalization_axes = make_axes(normalization_axes)
    e = exp(x - max(x, reduction_axes=normalization_axes))
    return e * reciprocal(sum(e, reduction_axes=normalization_axes))


# ---- contractions -------------------------------------------------------------------------------
class DotOp(Op):
    """Contracts the axes common to both operands (ngraph/op_graph/op_graph.py: DotOp)."""

    def __init__(self, x, y, **kw):
        x, y = as_op(x), as_op(y)
        self.reduction_axes = x.axes & y.axes
        self.x_out_axes = x.axes - self.reduction_axes
        self.y_out_axes = y.axes - self.reduction_axes
        super(DotOp, self).__init__((x, y), self.x_out_axes + self.y_out_axes, **kw)


def dot(x, y):
    return DotOp(x, y)


class ConvolutionOp(Op):
    """fprop: O[K,M,P,Q,N] = sum F[C,T,R,S,K] * I[C,D,H,W,N]
    (ngraph/op_graph/convolution.py:  ConvolutionOp)."""

    def __init__(self, conv_params, inputs, filters, axes, bias=None, activation=None,
                 residual=None, **kw):
        inputs, filters = as_op(inputs), as_op(filters)
        if len(inputs.axes) != 5:
            raise ValueError("convolution input shape must be length 5, found {}".format(
                len(inputs.axes.lengths)))
        if len(filters.axes) != 5:
            raise ValueError("convolution filter shape must be length 5, found {}".format(
                len(filters.axes.lengths)))
        if inputs.axes[0].length != filters.axes[0].length:
            raise ValueError("the first axis in input {inputs} and filter {filters} are not the "
                             "same.".format(inputs=inputs.axes[0], filters=filters.axes[0]))
        args = [inputs, filters]
        super(ConvolutionOp, self).__init__(args, axes, **kw)
        self.conv_params = dict(conv_params)


def convolution(conv_params, inputs, filters, axes, **kw):
    return ConvolutionOp(conv_params, inputs, filters, make_axes(axes), **kw)


class ConvDerivOp(Op):
    """Common part of the two convolution gradients: they carry the forward op, whose
    conv_params and tensor extents they share (ngraph/op_graph/convolution.py: ConvDerivOp)."""

    def __init__(self, args, fprop, axes, **kw):
        if not isinstance(fprop, ConvolutionOp):
            raise ValueError("fprop must be the forward ConvolutionOp")
        super(ConvDerivOp, self).__init__(args, axes, **kw)
        self.fprop = fprop
        self.conv_params = fprop.conv_params
        self.add_control_dep(fprop)


class update_conv(ConvDerivOp):
    """Filter gradient U[C,T,R,S,K] = sum_{p,q,n} I * delta
    (ngraph/op_graph/convolution.py: update_conv; args are (delta, inputs))."""

    def __init__(self, delta, inputs, filters, fprop, **kw):
        delta, inputs = as_op(delta), as_op(inputs)
        super(update_conv, self).__init__((delta, inputs), fprop, as_op(filters).axes, **kw)


class bprop_conv(ConvDerivOp):
    """Input gradient gI[C,D,H,W,N] = sum_{k,r,s} F * delta
    (ngraph/op_graph/convolution.py: bprop_conv; args are (delta, filters))."""

    def __init__(self, delta, inputs, filters, fprop, **kw):
        delta, filters = as_op(delta), as_op(filters)
        super(bprop_conv, self).__init__((delta, filters), fprop, as_op(inputs).axes, **kw)


class PoolingOp(Op):
    """ngraph/op_graph/pooling.py: PoolingOp; input C,D,H,W,N -> output C,M,P,Q,N."""

    def __init__(self, pool_params, inputs, axes, **kw):
        inputs = as_op(inputs)
        if len(inputs.axes) != 5:
            raise ValueError("pooling input shape must be length 5, found {}".format(
                len(inputs.axes.lengths)))
        if pool_params["op"] not in ("max", "avg"):
            raise ValueError("Unsupported pooling type: {pooltype}.  Only max and avg pooling "
                             "currently supported. ".format(pooltype=pool_params["op"]))
        super(PoolingOp, self).__init__((inputs,), axes, **kw)
        self.pool_params = dict(pool_params)


def pooling(pool_params, inputs, axes, **kw):
    return PoolingOp(pool_params, inputs, make_axes(axes), **kw)


class BpropPoolOp(Op):
    """Gradient of a PoolingOp with respect to its input (ngraph/op_graph/pooling.py:70-93):
    args (delta C,M,P,Q,N ; the pooled tensor C,D,H,W,N), result on the pooled tensor's axes."""

    def __init__(self, delta, inputs, fprop, **kw):
        delta, inputs = as_op(delta), as_op(inputs)
        if not isinstance(fprop, PoolingOp):
            raise ValueError("bprop_pool needs the forward PoolingOp, got {}".format(fprop))
        if delta.axes.lengths != fprop.axes.lengths:
            raise ValueError("bprop_pool: delta has shape %s, the pooling result %s"
                             % (delta.axes.lengths, fprop.axes.lengths))
        super(BpropPoolOp, self).__init__((delta, inputs), inputs.axes, **kw)
        self.fprop = fprop

    @property
    def pool_params(self):
        return self.fprop.pool_params


def bprop_pool(delta, inputs, fprop):
    return BpropPoolOp(delta, inputs, fprop)


class LookupTableOp(Op):
    """out = lut.take(idx, axis) (ngraph/op_graph/lookuptable.py:55-118): lut is 2-d, idx 1-d;
    the output axes name the index axis in place of the lut axis that is looked up."""

    def __init__(self, lut, idx, axes, update=True, pad_idx=None, **kw):
        lut, idx = as_op(lut), as_op(idx)
        axes = make_axes(axes)
        if len(lut.axes) != 2:
            raise ValueError("lookup table shape must be length 2, found {}".format(len(lut.axes)))
        if len(idx.axes) != 1:
            raise ValueError("index shape must be length 1, found {}".format(len(idx.axes)))
        if not (lut.axes[0] in axes or lut.axes[1] in axes):
            raise ValueError("Output axes must indicate which axis to do lookup.  None of the "
                             "output axes is from lookup table.")
        if idx.axes[0] not in axes:
            raise ValueError("Output axes must index axes.")
        self.lut_axis = 0 if lut.axes[1] in axes else 1
        self.pad_idx = pad_idx
        self.update = update
        if axes[self.lut_axis] != idx.axes[0]:
            raise ValueError("Cannot transpose lut axes implicitly")
        super(LookupTableOp, self).__init__((lut, idx), axes, **kw)


def lookuptable(lut, idx, axes, update=True, pad_idx=None, **kw):
    return LookupTableOp(lut, idx, axes, update=True, pad_idx=pad_idx)


class update_lut(Op):    # noqa: N801  (the reference's name)
    """Gradient of the table: args (delta, idx), result on the table's axes
    (ngraph/op_graph/lookuptable.py:160-175)."""

    def __init__(self, delta, lut, idx, fprop, **kw):
        delta, lut, idx = as_op(delta), as_op(lut), as_op(idx)
        if not isinstance(fprop, LookupTableOp):
            raise ValueError("update_lut needs the forward LookupTableOp, got {}".format(fprop))
        if delta.axes.lengths != fprop.axes.lengths:
            raise ValueError("update_lut: delta has shape %s, the lookup result %s"
                             % (delta.axes.lengths, fprop.axes.lengths))
        super(update_lut, self).__init__((delta, idx), lut.axes, **kw)
        self.fprop = fprop

    @property
    def lut_axis(self):
        return self.fprop.lut_axis

    @property
    def pad_idx(self):
        return self.fprop.pad_idx


def lookuptable_update(delta, lut, idx, fprop_op):
    return update_lut(delta, lut, idx, fprop_op)


# ---- operators of a language model's training step ----------------------------------------------
# (The reference has no counterpart; they stand beside its lookup table, batch normalisation and
# optimizers.  Gradients are ops of their own, like those of convolutions.)
class ResultOp(Op):
    """One of several results of an op."""

    def __init__(self, of, which, axes, **kw):
        super(ResultOp, self).__init__((of,), axes, **kw)
        self.which = which


def _check_operand(what, op, axes):
    if not op.axes.is_equal_set(axes):
        raise ValueError("%s has the axes %s where %s are expected" % (what, op.axes, axes))


class EmbeddingOp(Op):
    """scale * table[idx]: args (table, idx), result on the axes of idx and the table's second."""

    def __init__(self, table, idx, scale=1.0, pad_idx=None, **kw):
        table, idx = as_op(table), as_op(idx)
        if len(table.axes) != 2:
            raise ValueError("embedding table shape must be length 2, found {}".format(len(table.axes)))
        if len(idx.axes) == 0:
            raise ValueError("embedding index needs an axis")
        if table.axes[1] in idx.axes or table.axes[1].name in [a.name for a in idx.axes]:
            raise ValueError("the table's axis %s is an axis of the index" % table.axes[1])
        super(EmbeddingOp, self).__init__((table, idx), list(idx.axes) + [table.axes[1]], **kw)
        self.scale = float(scale)
        self.pad_idx = None if pad_idx is None else int(pad_idx)

    def layouts(self):
        """(argument, its axes in the order of memory, how many of them may lie apart)"""
        return [(self.args[0], self.args[0].axes, 0), (self.args[1], self.args[1].axes, 0)]


def embedding(table, idx, scale=1.0, pad_idx=None):
    """Rows of `table` [tokens, features] looked up at `idx` (any axes) and scaled.  Indices outside
    the table, and NaN, read as zero; the gradient of row pad_idx is zero."""
    return EmbeddingOp(table, idx, scale, pad_idx)


class EmbeddingGradOp(Op):
    """The table's gradient: args (delta, idx); rows of delta added up per token in their order."""

    def __init__(self, delta, fprop, **kw):
        delta = as_op(delta)
        if not isinstance(fprop, EmbeddingOp):
            raise ValueError("embedding_grad needs the forward EmbeddingOp, got {}".format(fprop))
        _check_operand("delta", delta, fprop.axes)
        self.fprop = fprop
        super(EmbeddingGradOp, self).__init__((delta, fprop.args[1]), fprop.args[0].axes, **kw)

    def layouts(self):
        return [(self.args[0], self.fprop.axes, 0), (self.args[1], self.args[1].axes, 0)]


def embedding_grad(delta, fprop):
    """Gradient of the table that the embedding `fprop` looks up, from that of its result."""
    return EmbeddingGradOp(delta, fprop)


class ResidualNormOp(Op):
    """stream = residual_scale * residual + gate * (rms(block) * post_weight),
    out = rms(stream) * weight, with rms(x) = x / sqrt(mean(x^2) + eps) over `axes`."""

    def __init__(self, residual, block, weight, axes, post_weight=None, gate=None, residual_scale=1.0,
                 eps=1e-6, **kw):
        residual = as_op(residual)
        self.norm_axes = make_axes(axes)
        if not len(self.norm_axes) or not self.norm_axes.is_sub_set(residual.axes):
            raise ValueError("the axes %s are not axes of the operand %s" % (self.norm_axes, residual.axes))
        self.row_axes = residual.axes - self.norm_axes
        both = self.row_axes + self.norm_axes
        optional = lambda x: None if x is None else as_op(x)  # noqa: E731
        self.residual, self.block, self.weight = residual, optional(block), optional(weight)
        self.post_weight, self.gate = optional(post_weight), optional(gate)
        if self.block is None and (self.gate is not None or self.post_weight is not None or float(residual_scale) != 1.0):
            raise ValueError("a gate, a weight or a scale without a block")
        if self.block is None and self.weight is None:
            raise ValueError("nothing to compute: neither a block nor a weight")
        if self.block is not None:
            _check_operand("block", self.block, both)
        for what, w in (("weight", self.weight), ("post_weight", self.post_weight)):
            if w is not None:
                _check_operand(what, w, self.norm_axes)
        self.gate_kind = 0
        if self.gate is not None:
            kinds = [k for k, ax in ((1, self.norm_axes), (2, self.row_axes), (3, both))
                     if len(ax) and self.gate.axes.is_equal_set(ax)]
            if not kinds:
                raise ValueError("a gate has the axes %s, %s or %s, not %s" %
                                 (self.norm_axes, self.row_axes, both, self.gate.axes))
            self.gate_kind = kinds[0]
        self.residual_scale, self.eps = float(residual_scale), float(eps)
        if not self.eps >= 0:
            raise ValueError("eps is not negative: %r" % (eps,))
        operands = [x for x in (self.residual, self.block, self.gate, self.post_weight, self.weight) if x is not None]
        super(ResidualNormOp, self).__init__(operands, both, **kw)
        self.results = {}
        if self.block is not None:
            self.results["stream"] = ResultOp(self, "stream", both)
        if self.weight is not None:
            self.results["out"] = ResultOp(self, "out", both)
            self.results["stream_rstd"] = ResultOp(self, "stream_rstd", self.row_axes)
        if self.post_weight is not None:
            self.results["block_rstd"] = ResultOp(self, "block_rstd", self.row_axes)

    @property
    def gate_axes(self):
        return (None, self.norm_axes, self.row_axes, self.row_axes + self.norm_axes)[self.gate_kind]

    def layouts(self):
        both, rows = self.row_axes + self.norm_axes, len(self.row_axes)
        found = [(x, both, rows) for x in (self.residual, self.block) if x is not None]
        found += [(x, self.norm_axes, 0) for x in (self.post_weight, self.weight) if x is not None]
        if self.gate is not None:
            found.append((self.gate, self.gate_axes, rows if self.gate_kind == 3 else 0))
        return found


def residual_norm(residual, block, weight, axes, post_weight=None, gate=None, residual_scale=1.0, eps=1e-6):
    """The edge between two blocks of a residual network: (stream, out) with
    stream = residual_scale * residual + gate * (rms(block) * post_weight) and out = rms(stream) * weight.
    gate (per feature, per row or for every value) and post_weight may be None; weight None: out is None."""
    op = ResidualNormOp(residual, block, weight, axes, post_weight, gate, residual_scale, eps)
    return op.results.get("stream"), op.results.get("out")


def rms_norm(x, weight, axes, eps=1e-6):
    """x / sqrt(mean(x^2) + eps) * weight over `axes`."""
    return ResidualNormOp(x, None, weight, axes, eps=eps).results["out"]


class ResidualNormGradOp(Op):
    """All gradients of a ResidualNormOp in one step."""

    def __init__(self, fprop, d_out=None, d_stream=None, **kw):
        if isinstance(fprop, ResultOp):
            fprop = fprop.args[0]
        if not isinstance(fprop, ResidualNormOp):
            raise ValueError("residual_norm_grad needs a result of the forward op, got {}".format(fprop))
        if (d_out is None) != (fprop.weight is None):
            raise ValueError("the gradient of out and a weight go together")
        if d_out is None and d_stream is None:
            raise ValueError("no gradient to start from")
        both = fprop.row_axes + fprop.norm_axes
        self.fprop = fprop
        self.d_out, self.d_stream = [None if d is None else as_op(d) for d in (d_out, d_stream)]
        for what, d in (("d_out", self.d_out), ("d_stream", self.d_stream)):
            if d is not None:
                _check_operand(what, d, both)
        self.reads = dict(d_out=self.d_out, d_stream=self.d_stream, block=fprop.block, gate=fprop.gate,
                          post_weight=fprop.post_weight, weight=fprop.weight,
                          stream=fprop.results.get("stream", fprop.residual) if fprop.weight is not None else None,
                          stream_rstd=fprop.results.get("stream_rstd"), block_rstd=fprop.results.get("block_rstd"))
        self.reads = {k: v for k, v in self.reads.items() if v is not None}
        super(ResidualNormGradOp, self).__init__(list(self.reads.values()), both, **kw)
        self.results = {"residual": ResultOp(self, "residual", both)}
        if fprop.block is not None:
            self.results["block"] = ResultOp(self, "block", both)
        for name, ax in (("gate", fprop.gate_axes), ("post_weight", fprop.norm_axes), ("weight", fprop.norm_axes)):
            if getattr(fprop, name) is not None:
                self.results[name] = ResultOp(self, name, ax)

    def layouts(self):
        f = self.fprop
        both, rows = f.row_axes + f.norm_axes, len(f.row_axes)
        axes = dict(post_weight=(f.norm_axes, 0), weight=(f.norm_axes, 0), stream_rstd=(f.row_axes, 0), block_rstd=(f.row_axes, 0),
                    gate=(f.gate_axes, rows if f.gate_kind == 3 else 0))
        return [(x,) + axes.get(k, (both, rows)) for k, x in self.reads.items()]


def residual_norm_grad(fprop, d_out=None, d_stream=None):
    """Gradients of residual_norm or rms_norm (`fprop` is one of its results) from those of `out` and, where
    later blocks read it, of `stream`: a dict of residual, block, gate, post_weight and weight, those of them
    that the forward op has.  The gradient of rms_norm's operand is `residual`."""
    return dict(ResidualNormGradOp(fprop, d_out, d_stream).results)


class AdamWOp(Op):
    """One AdamW step over all of `variables` (see adamw).  Its value is the number of steps made."""
    is_tensor_op = False

    def __init__(self, variables, gradients, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, no_decay=(),
                 state_bits=32, grad_scale=None, seed=0, **kw):
        variables, gradients = as_ops(variables), as_ops(gradients)
        if len(variables) != len(gradients):
            raise ValueError("%d variables and %d gradients" % (len(variables), len(gradients)))
        if len(set(variables)) != len(variables):
            raise ValueError("a variable occurs twice")
        for v, g in zip(variables, gradients):
            if not isinstance(v, AssignableTensorOp) or v.is_constant:
                raise ValueError("{} is not assignable.".format(v))
            _check_operand("the gradient of %s" % v, g, v.axes)
        if state_bits not in (8, 32):
            raise ValueError("moments are held in 32 or 8 bits, not in %r" % (state_bits,))
        for x in no_decay:
            if x not in variables:
                raise ValueError("{} is not among the variables".format(x))
        self.variables, self.gradients = variables, gradients
        self.rates = dict(beta1=float(beta1), beta2=float(beta2), eps=float(eps), weight_decay=float(weight_decay))
        if not (0 <= self.rates["beta1"] < 1 and 0 <= self.rates["beta2"] < 1 and self.rates["eps"] >= 0):
            raise ValueError("bad rates: %s" % self.rates)
        self.state_bits, self.seed = state_bits, int(seed) & 0xffffffff
        self.decayed = [v not in no_decay for v in variables]
        # (numbers stay as they are: an op of one would be rounded to fp32)
        self.lr = float(lr) if isinstance(lr, numbers.Number) else as_op(lr)
        self.grad_scale = float(grad_scale) if isinstance(grad_scale, numbers.Number) else None if grad_scale is None else as_op(grad_scale)
        for what, x in (("lr", self.lr), ("grad_scale", self.grad_scale)):
            if isinstance(x, Op) and x.axes.size != 1:
                raise ValueError("%s is a number, not a tensor with axes %s" % (what, x.axes))
        self.count = persistent_tensor([make_axis(1, name="steps")], initial_value=0.0)
        # 32 bits: (m, v).  8: bytes of m and of sqrt(v), four to a word, and the scales of 256 values each
        words = lambda n, per, name: persistent_tensor([make_axis(-(-n // per), name="words")], initial_value=0.0, name=name)  # noqa: E731
        self.states = []
        for v in variables:
            n = v.axes.size
            if state_bits == 32:
                self.states.append(tuple(persistent_tensor(v.axes, initial_value=0.0, name="%s_%s" % (v.name, m)) for m in "mv"))
            else:
                self.states.append((words(n, 4, v.name + "_m"), words(n, 4, v.name + "_v"), words(n, 256, v.name + "_m_scales"),
                                    words(n, 256, v.name + "_v_scales")))
        args = list(variables) + list(gradients) + [s for x in self.states for s in x] + [self.count]
        super(AdamWOp, self).__init__(args + [x for x in (self.lr, self.grad_scale) if isinstance(x, Op)], self.count.axes, **kw)

    def layouts(self):
        return [(g, v.axes, 0) for v, g in zip(self.variables, self.gradients)] + \
            [(x, x.axes, 0) for x in (self.lr, self.grad_scale) if isinstance(x, Op)]

    def written(self):
        return list(self.variables) + [s for x in self.states for s in x] + [self.count]


def adamw(variables, gradients, lr, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=0.01, no_decay=(), state_bits=32,
          grad_scale=None, seed=0):
    """One AdamW step over many variables at once.  lr, and grad_scale, which multiplies every gradient, are
    numbers or ops whose value is one.  no_decay: the variables without weight decay.  state_bits 8: moments as
    e4m3 bytes with a scale for every 256, rounded at random (from `seed`, the position and the step).  The
    moments (op.states) and the number of steps (op.count) are persistent tensors, zero before the first."""
    return AdamWOp(variables, gradients, lr, beta1, beta2, eps, weight_decay, no_decay, state_bits, grad_scale, seed)


# ---- communication ----------------------------------------------------------------------------
class AllReduceOp(Op):
    """Sum (or mean) of a tensor over all data-parallel replicas; every replica gets the result
    (ngraph/op_graph/comm_nodes.py:347-383 GPUCudaAllReduceOp; inserted by hetr wherever an
    argument carries reduce_func and its consumer does not,
    ngraph/factory/comm_node_factory.py:298-341)."""

    def __init__(self, x, reduce_func="sum", **kw):
        x = as_op(x)
        if reduce_func not in ("sum", "mean"):
            raise ValueError("unsupported reduce_func %r" % (reduce_func,))
        super(AllReduceOp, self).__init__((x,), x.axes, **kw)
        self.reduce_func = reduce_func


class RngOp(Op):
    """A tensor with the axes of x, filled with fresh random numbers on every execution
    (ngraph/op_graph/op_graph.py:2786-2870; x only supplies the axes, as in the reference's
    kernels, ngraph/transformers/gpu/tensor_ops.py:621-661)."""

    def __init__(self, distribution, params, x, **kw):
        if distribution not in ("uniform", "normal"):
            raise ValueError("unsupported distribution: {}".format(distribution))
        x = as_op(x)
        self.distribution = distribution
        self.params = dict(params)
        super(RngOp, self).__init__((x,), x.axes, **kw)


def uniform(x, low=0.0, high=1.0):
    return RngOp("uniform", dict(low=low, high=high), x)


def normal(x, loc=0.0, scale=1.0):
    return RngOp("normal", dict(loc=loc, scale=scale), x)


def allreduce(x, reduce_func="sum"):
    return AllReduceOp(x, reduce_func)


# ---- state and control ------------------------------------------------------------------------
class AssignOp(Op):
    """tensor <- value (ngraph/op_graph/op_graph.py: AssignOp)."""
    is_tensor_op = False

    def __init__(self, tensor, val, **kw):
        tensor, val = as_op(tensor), as_op(val)
        base = tensor
        while isinstance(base, ViewOp):              # a view of an assignable tensor is assignable
            base = base.args[0]
        if not isinstance(base, AssignableTensorOp):
            raise ValueError("{} is not assignable.".format(tensor))
        if not val.axes.is_sub_set(tensor.axes):
            raise ValueError("cannot assign axes %s to a tensor with axes %s" %
                             (val.axes, tensor.axes))
        super(AssignOp, self).__init__((tensor, val), tensor.axes, **kw)


def assign(lvalue, rvalue):
    return AssignOp(lvalue, rvalue)


class SequentialOp(Op):
    """Runs `ops` in order; its value is the last one (ngraph/op_graph/op_graph.py:
    SequentialOp)."""
    is_device_op = False

    def __init__(self, ops, **kw):
        ops = as_ops(ops)
        if not ops:
            raise ValueError("sequential needs at least one op")
        super(SequentialOp, self).__init__(ops, ops[-1].axes, **kw)
        self.ops = ops

    @property
    def value_tensor(self):
        return self.ops[-1]


def sequential(ops=None):
    return SequentialOp(ops)


def value_of(tensor):
    """A copy of the tensor's current value (ngraph/op_graph/op_graph.py: value_of)."""
    return ElementWiseOp("assign", (tensor,))
