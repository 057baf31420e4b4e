"""Operators of transformer layers as graph ops: what stands around attention and the plain linear layers.

Each is a call of the library (include/mjt.h) with one or several results, a core.KernelOp for each of them; the functions that
programs use are in nn.py.  Their gradients are calls of the same kind.  Second derivatives of norms of heads and of gated projections are not
there: they are refused when they are asked for.
"""
import copy
import ctypes
import itertools
import numbers
import weakref

import numpy as np

from . import _graph
from . import _lib
from . import core
from .core import KernelOp, Var

_FLOATS = ("float32", "bfloat16", "float16")


_numbers, _next = {}, itertools.count()            # (name, options) -> its number


class Call:
    """What is called and with which options; shared by the ops of its results."""
    __slots__ = ("name", "options", "number", "kept")

    def __init__(self, name, *options):
        self.name, self.options, self.number = name, options, None
        self.kept = None                                       # weakly, a result that gradients read and nobody else has

    def key(self):
        """A number for name and options: a graph's key is worked out and looked up for every execution."""
        if self.number is None:
            self.number = _numbers.get((self.name, self.options))
            if self.number is None:
                if len(_numbers) >= 4096:                      # (options that change with every step; a number is never given twice)
                    _numbers.clear()
                self.number = _numbers[self.name, self.options] = next(_next)
        return self.number


def _result(call, index, inputs, shape, dtype):
    return _graph.kernel_var(KernelOp, call, index, inputs, shape, dtype)


def _float_var(who, v, name="x"):
    v = core._as_var(v)
    if v.dtype not in _FLOATS:
        raise TypeError("%s: %s is %s, not one of %s" % (who, name, v.dtype, ", ".join(_FLOATS)))
    return v


# ---- dropout ------------------------------------------------------------------------------------------------------
class _Generator:
    """The key and the number of the next call of a dropout without a seed of its own; jt.set_seed starts it anew."""

    def __init__(self):
        self.seed(0)

    def seed(self, seed):
        if not isinstance(seed, numbers.Integral):             # what else numpy makes a generator of: a copy's first number, the generator itself goes on from where it is
            seed = copy.deepcopy(np.random.default_rng(seed)).integers(1 << 63)
        self.state = int(seed), itertools.count()              # (one object: threads that draw at the same time get numbers of one key)

    def next(self):
        key, calls = self.state
        return key, next(calls)


generator = _Generator()


def _number(value, name):
    """64 bits that go into the kernel by value."""
    if not isinstance(value, numbers.Integral):
        raise TypeError("dropout: %s has to be an integer, got %r" % (name, value))
    value = int(value) & (1 << 64) - 1
    return _graph.number_var(np.array([value - (value >> 63 << 64)], np.int64), "int64")


def dropout(x, p, is_train, seed, offset, residual):
    x = _float_var("dropout", x)
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("dropout: p has to be between 0 and 1, got %r" % p)
    if residual is not None:
        residual = core._as_var(residual)
        if residual.dtype != x.dtype or list(residual.shape) != list(x.shape):
            raise ValueError("dropout: x is %s %s, the residual %s %s" % (x.dtype, list(x.shape), residual.dtype, list(residual.shape)))
    if seed is None and offset is not None:
        raise ValueError("dropout: an offset belongs to a seed")
    if not is_train or p == 0.0:
        if residual is None:
            return x
        p, seed, offset = 0.0, 0, 0                            # (the sum alone, rounded as in training)
    numbered = seed is not None                                # by the program; otherwise by numbers that no seed and offset of a program's give
    if not numbered:
        seed, offset = generator.next()
    key = [_number(seed, "the seed"), _number(offset or 0, "the offset")]
    inputs = [x] + ([] if residual is None else [residual]) + key
    return _result(Call("dropout", p, residual is not None, numbered), 0, inputs, list(x.shape), x.dtype)


def _launch_dropout(ex, options, inputs, outs):
    p, added, numbered = options
    x, y = inputs[0], outs[0]
    scalars = [(_lib.FusedVar * 1)(_lib.FusedVar(_lib.VAR_SCALAR, _lib.DTYPE_CODE["int64"], None, 0.0, int(u._host.reshape(-1)[0]))) for u in inputs[-2:]]
    if ex._cap is not None:
        ex._cap.scalars += [(s, 0, u) for s, u in zip(scalars, inputs[-2:])]
    tx, ty = ex._tensor_of(x), ex._tensor(ex._alloc_out(y), y.dtype, y.shape)
    res = ctypes.byref(ex._tensor_of(inputs[1])) if added else None
    lib = ex._libh()
    _lib.check((lib.mjt_dropout if numbered else lib.mjt_dropout_unnumbered)(ctypes.byref(tx), res, ctypes.byref(ty), p, *scalars))


def _dropout_gradients(op, inputs, douts, wanted):
    p, added, numbered = op.call.options
    dy = douts[0]
    grads = [None] * len(inputs)
    if wanted[0]:
        grads[0] = _result(Call("dropout", p, False, numbered), 0, [dy] + list(inputs[-2:]), list(dy.shape), dy.dtype) if p else dy
    if added and wanted[1]:
        grads[1] = dy
    return grads


# ---- norms of heads and the rotation of positions -------------------------------------------------------------------
def rope_table(n, dim, base=10000.0):
    if dim < 2 or dim % 2 or n < 1:
        raise ValueError("rope_table: %r positions of %r rotated elements (an even number)" % (n, dim))
    angle = np.arange(n, dtype=np.float64)[:, None] * float(base) ** (-np.arange(0, dim, 2, dtype=np.float64) / dim)
    return core.array(np.stack([np.cos(angle), np.sin(angle)], -1).astype(np.float32), "float32")


def head_norm_rope(who, x, counts, scales, table, positions, sections, eps, interleaved, heads_first):
    """The results for the heads counts = (queries, keys, values) of x; none for a count of 0."""
    x = _float_var(who, x)
    if x.ndim < 3:
        raise ValueError("%s: x has to be [.., tokens, heads, dim], got %s" % (who, list(x.shape)))
    lead, (S, H, D) = list(x.shape[:-3]), x.shape[-3:]
    if min(counts) < 0 or sum(counts) != H:
        raise ValueError("%s: %d queries, %d keys and %d values in %d heads" % ((who,) + tuple(counts) + (H,)))
    if D < 2 or D % 2:
        raise ValueError("%s: heads of %d elements (an even number is needed)" % (who, D))
    inputs = [x]
    if scales is not None:
        q, k = _float_var(who, scales[0], "a scale"), _float_var(who, scales[1], "a scale")
        if q.num != D or k.num != D or q.dtype != k.dtype:
            raise ValueError("%s: scales of %s elements for heads of %d, of one dtype" % (who, [q.num, k.num], D))
        inputs += q, k
    elif table is None:
        raise ValueError("%s: neither scales nor a table: nothing to do" % who)
    if table is not None:
        table = core._as_var(table)
        if table.dtype != "float32" or table.ndim != 3 or table.shape[2] != 2 or not 1 <= table.shape[1] <= D // 2 or table.shape[0] < 1:
            raise ValueError("%s: the table has to be float32 [positions, pairs, 2] with at most %d pairs, got %s %s" % (who, D // 2, table.dtype, list(table.shape)))
        inputs.append(table)
    if sections is not None:
        sections = tuple(int(s) for s in sections)
        if table is None or positions is None:
            raise ValueError("%s: sections need a table and positions" % who)
        if not 1 <= len(sections) <= _lib.MOST_AXES or min(sections) < 0 or sum(sections) != table.shape[1]:
            raise ValueError("%s: sections %s of a table of %d pairs (up to %d axes)" % (who, list(sections), table.shape[1], _lib.MOST_AXES))
    if positions is not None:
        positions = core._as_var(positions)
        if table is None or positions.dtype != "int32":
            raise ValueError("%s: positions are int32 and need a table, got %s" % (who, positions.dtype))
        axes = [] if sections is None else [len(sections)]
        at = list(positions.shape)
        if at != axes + lead + [S] and at != axes + [S]:
            raise ValueError("%s: positions %s for tokens %s%s" % (who, at, lead + [S], " with %d axes" % axes[0] if axes else ""))
        inputs.append(positions)
    elif table is not None and S > table.shape[0]:
        raise ValueError("%s: %d tokens and a table of %d positions" % (who, S, table.shape[0]))
    if not float(eps) >= 0.0:
        raise ValueError("%s: eps has to be at least 0, got %r" % (who, eps))
    call = Call("head_norm_rope", tuple(map(int, counts)), scales is not None, table is not None, positions is not None, sections, float(eps), bool(interleaved), bool(heads_first))
    return [_result(call, i, inputs, lead + ([n, S, D] if heads_first else [S, n, D]), x.dtype) for i, n in enumerate(counts) if n]


def _head_norm(options, inputs):
    """The C parameters and the inputs by role."""
    counts, scaled, tabled, placed, sections, eps, interleaved, heads_first = options
    p = _lib.HeadNorm(counts[0], counts[1], counts[2], interleaved, heads_first, 0 if sections is None else len(sections), (ctypes.c_int32 * _lib.MOST_AXES)(*(sections or ())), eps)
    rest = list(inputs[1:])
    q_scale, k_scale = (rest.pop(0), rest.pop(0)) if scaled else (None, None)
    return p, [inputs[0], q_scale, k_scale, rest.pop(0) if tabled else None, rest.pop(0) if placed else None], rest


def _refs(ex, vs):
    return [None if v is None else ctypes.byref(ex._tensor_of(v)) for v in vs]


def _out_refs(ex, outs, n):
    return [ctypes.byref(ex._tensor(ex._alloc_out(outs[i]), outs[i].dtype, outs[i].shape)) if i in outs else None for i in range(n)]


def _launch_head_norm(ex, options, inputs, outs):
    p, roles, _ = _head_norm(options, inputs)
    _lib.check(ex._libh().mjt_head_norm_rope(*_refs(ex, roles), ctypes.byref(p), *_out_refs(ex, outs, 3)))


def _launch_head_norm_grad(ex, options, inputs, outs):
    p, roles, rest = _head_norm(options[:-1], inputs)
    given = [rest.pop(0) if there else None for there in options[-1]]
    _lib.check(ex._libh().mjt_head_norm_rope_grad(*_refs(ex, roles), ctypes.byref(p), *_refs(ex, given), *_out_refs(ex, outs, 3)))


def _head_norm_gradients(op, inputs, douts, wanted):
    given = tuple(i in douts for i in range(3))
    call = Call("head_norm_rope_grad", *op.call.options, given)
    ins = list(inputs) + [douts[i] for i in range(3) if given[i]]
    scaled, tabled = op.call.options[1:3]
    if tabled and wanted[3 if scaled else 1]:
        raise NotImplementedError("head_norm_rope: the gradient of a table of angles")
    return [_result(call, i, ins, list(u.shape), u.dtype) if want and i < (3 if scaled else 1) else None for i, (u, want) in enumerate(zip(inputs, wanted))]


# ---- gated projections ------------------------------------------------------------------------------------------------
def gated_linear(x, weight, activation):
    x, weight = _float_var("gated_linear", x), _float_var("gated_linear", weight, "the weight")
    if activation not in _lib.ACTIVATIONS:
        raise ValueError("gated_linear: activation %r is not one of %s" % (activation, ", ".join(_lib.ACTIVATIONS)))
    if weight.ndim != 2 or weight.shape[0] % 2 or x.shape[-1] != weight.shape[1] or x.dtype != weight.dtype:
        raise ValueError("gated_linear: x %s %s and weight %s %s have to be [.., k] and [2 f, k]" % (x.dtype, list(x.shape), weight.dtype, list(weight.shape)))
    return _result(Call("gated_linear", activation), 0, [x, weight], list(x.shape[:-1]) + [weight.shape[0] // 2], x.dtype)


def _flat(ex, v, out=False):
    """A Var as rows of its last axis."""
    n = v.shape[-1]
    rows = 1
    for s in v.shape[:-1]:
        rows *= s
    return ctypes.byref(ex._tensor(ex._alloc_out(v) if out else ex._ptr_of(v), v.dtype, [rows, n]))


def _launch_gated(ex, options, inputs, outs):
    x, w = inputs
    _lib.check(ex._libh().mjt_gated_linear(_flat(ex, x), _flat(ex, w), _lib.ACTIVATIONS.index(options[0]), *[_flat(ex, outs[i], True) if i in outs else None for i in range(2)]))


def _launch_gated_grad(ex, options, inputs, outs):
    dy, both = inputs
    _lib.check(ex._libh().mjt_gated_linear_grad(_flat(ex, dy), _flat(ex, both), _lib.ACTIVATIONS.index(options[0]), _flat(ex, outs[0], True)))


def _launch_product(ex, options, inputs, outs):
    a, b = inputs
    _lib.check(ex._libh().mjt_matmul_nearest(_flat(ex, a), _flat(ex, b), _flat(ex, outs[0], True), int(options[0]), int(options[1])))


def _gated_gradients(op, inputs, douts, wanted):
    x, w = inputs
    dy = douts[0]
    f2 = w.shape[0]
    # the products of the forward pass in 32 bits: written by the same launch where the two passes run together, made again otherwise.  Gradients that
    # are taken one after the other share them for as long as any that reads them waits.
    both = op.call.kept() if op.call.kept is not None else None
    if both is None:
        both = _result(op.call, 1, list(inputs), list(x.shape[:-1]) + [f2], "float32")
        op.call.kept = weakref.ref(both)
    d = _result(Call("gated_linear_grad", *op.call.options), 0, [dy, both], list(x.shape[:-1]) + [f2], dy.dtype)
    return [_result(Call("product", False, False), 0, [d, w], list(x.shape), x.dtype) if wanted[0] else None,
            _result(Call("product", True, False), 0, [d, x], list(w.shape), w.dtype) if wanted[1] else None]


def down_projection(x, weight):
    """x * weight^T for bfloat16, rounded to nearest even like what the other operators here write, gradients too; the ordinary product truncates."""
    if weight.ndim != 2 or x.shape[-1] != weight.shape[1]:
        raise ValueError("gated_ffn: the second weight %s has to be [n, %d]" % (list(weight.shape), x.shape[-1]))
    return _result(Call("product", False, True), 0, [x, weight], list(x.shape[:-1]) + [weight.shape[0]], x.dtype)


def _product_gradients(op, inputs, douts, wanted):
    (a, b), dc = inputs, douts[0]
    trans_a, trans_b = op.call.options
    da = ((b, dc) if trans_a else (dc, b)), (False, trans_a or not trans_b)                  # a^T b: b dc^T;  a b^T: dc b;  a b: dc b^T
    db = ((dc, a) if trans_b else (a, dc)), (not trans_a, False)                             #        a dc;           dc^T a;        a^T dc
    return [_result(Call("product", *trans), 0, list(ops), list(u.shape), u.dtype) if want else None for u, (ops, trans), want in zip(inputs, (da, db), wanted)]


# ---- what the executor and grad() call ------------------------------------------------------------------------------------
_LAUNCH = {"dropout": _launch_dropout, "head_norm_rope": _launch_head_norm, "head_norm_rope_grad": _launch_head_norm_grad, "gated_linear": _launch_gated,
           "gated_linear_grad": _launch_gated_grad, "product": _launch_product}
_GRADIENTS = {"dropout": _dropout_gradients, "head_norm_rope": _head_norm_gradients, "gated_linear": _gated_gradients, "product": _product_gradients}


def launch(ex, ops):
    """One call for the pending results `ops` of it; ex: the executor."""
    call = ops[0].call
    ex.stats["launches"] += 1
    _LAUNCH[call.name](ex, call.options, ops[0].inputs, {op.index: op.out for op in ops})


def gradients(op, inputs, out, douts, wanted):
    """The gradients of the inputs of op's call (None: not wanted, or none) from those of its results by index."""
    f = _GRADIENTS.get(op.call.name)
    if f is None:
        raise NotImplementedError("the gradient of %s (a second derivative)" % op.call.name)
    # a gradient arrives in its result's type, except from ops that compute in another
    douts = {i: d if d.dtype == out.dtype else core.unary(d, out.dtype) for i, d in douts.items()}
    return f(op, inputs, douts, wanted)
