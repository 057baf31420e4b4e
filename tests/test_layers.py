"""Operators of transformer layers without a GPU: the plain forms that the GPU tests compare with, refusals, kernels that build for every
type, the ops that gradients are made of."""
import ctypes
import gc

import numpy as np
import pytest

import jittor_amd as jt
from jittor_amd import _lib as L
from jittor_amd import core, executor, layers
import layers_plain as P

B = ctypes.byref


# ---- the plain forms --------------------------------------------------------------------------------------------------
def test_philox_gives_the_published_known_answers():
    """The known-answer vectors of Philox4x32-10 that its authors publish."""
    assert P.philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert P.philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert P.philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def _slope(f, at, along, h=1e-6):
    return (f(at + h * along) - f(at - h * along)) / (2 * h)


@pytest.mark.parametrize("paired", [False, True])
@pytest.mark.parametrize("scaled", [False, True])
def test_gradient_formula_of_head_norms_against_differences(paired, scaled):
    rng = np.random.default_rng(1)
    x, dy, along = (rng.standard_normal((5, 3, 8)) for _ in range(3))
    scale, turned = (rng.uniform(0.5, 1.5, 8), rng.standard_normal(8)) if scaled else (None, None)
    angle = rng.uniform(0, 6, (5, 3))
    cos, sin = np.cos(angle), np.sin(angle)
    f = lambda v, s: (P.head_norm(v, s, cos, sin, 1e-3, paired) * dy).sum()
    dx, ds, _, _ = P.head_norm_grad(x, scale, cos, sin, 1e-3, paired, dy)
    assert abs(_slope(lambda v: f(v, scale), x, along) - (dx * along).sum()) < 1e-7
    if scaled:
        assert abs(_slope(lambda s: f(x, s), scale, turned) - (ds * turned).sum()) < 1e-7


@pytest.mark.parametrize("name", L.ACTIVATIONS)
def test_gradient_formula_of_gated_projections_against_differences(name):
    rng = np.random.default_rng(2)
    x, w, dy = rng.standard_normal((6, 5)), rng.standard_normal((14, 5)), rng.standard_normal((6, 7))
    ax, aw = rng.standard_normal(x.shape), rng.standard_normal(w.shape)
    (dx, _), (dw, _) = P.gated_grad(x, w, name, dy, "float32")
    assert abs(_slope(lambda v: (P.gated(v, w, name)[0] * dy).sum(), x, ax) - (dx * ax).sum()) < 1e-6
    assert abs(_slope(lambda v: (P.gated(x, v, name)[0] * dy).sum(), w, aw) - (dw * aw).sum()) < 1e-6


def test_rope_table_is_worked_out_in_64_bits():
    t = jt.nn.rope_table(5000, 6, 500.0).numpy().astype(np.float64)
    angle = np.arange(5000)[:, None] * 500.0 ** (-np.arange(3) / 3)
    assert t.shape == (5000, 3, 2) and np.abs(t - np.stack([np.cos(angle), np.sin(angle)], -1)).max() <= 2.0 ** -24
    for n, dim in ((0, 4), (4, 3), (4, 0)):
        with pytest.raises(ValueError):
            jt.nn.rope_table(n, dim)


# ---- refusals -----------------------------------------------------------------------------------------------------------
def _x(*shape, dtype="float32"):
    return jt.array(np.zeros(shape, np.float32), dtype)


def test_dropout_refuses():
    x = _x(3, 4)
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(ValueError):
            jt.nn.dropout(x, p, True)
    with pytest.raises(TypeError):
        jt.nn.dropout(jt.array(np.arange(6)), 0.5, True)
    with pytest.raises(TypeError):
        jt.nn.dropout(x, 0.5, True, seed=1.5)
    with pytest.raises(ValueError):
        jt.nn.dropout(x, 0.5, True, offset=3)
    with pytest.raises(ValueError):
        jt.nn.dropout(x, 0.5, True, residual=_x(4, 3))
    with pytest.raises(ValueError):
        jt.nn.dropout(x, 0.5, True, residual=_x(3, 4, dtype="float16"))


def test_dropout_without_training_is_the_input():
    x = _x(3, 4)
    assert jt.nn.dropout(x, 0.5) is x and jt.nn.dropout(x, 0.0, True) is x


def test_a_seed_numbers_the_calls_without_one():
    def keys(n):
        return [tuple(int(u._host[0]) for u in jt.nn.dropout(_x(4), 0.5, True)._op.inputs[1:]) for _ in range(n)]
    jt.set_seed(7)
    a = keys(3)
    jt.set_seed(7)
    assert keys(3) == a == [(7, 0), (7, 1), (7, 2)]
    jt.set_seed(0)


def test_numbers_of_calls_without_a_seed_are_not_those_of_one(launches):
    """The key and number of a call without a seed may be a program's own seed and offset: its numbers, and its gradient's, are others."""
    jt.set_seed(0)
    x, taken = _there(4, 4), []
    for y in (jt.nn.dropout(x, 0.5, True), jt.nn.dropout(x, 0.5, True, seed=0)):
        dx = jt.grad((y * _there(4, 4)).sum(), x)
        taken.append({(op.call.name, op.call.options, tuple(int(u._host[0]) for u in op.inputs[1:])) for op in _calls([y, dx])})
        jt.sync([y, dx])
    assert all(len(t) == 1 and next(iter(t))[2] == (0, 0) for t in taken) and taken[0] != taken[1]


@pytest.mark.parametrize("seed", [lambda: None, lambda: [1, 2], lambda: np.random.SeedSequence(4), lambda: np.random.default_rng(3), lambda: np.random.PCG64(3), lambda: np.uint64(1 << 63)],
                         ids=["none", "list", "sequence", "generator", "bits", "uint64"])
def test_seeds_are_what_numpy_takes(seed):
    """jt.random's numbers are numpy's for the seed; dropout numbers its calls anew, the same again where the seed says what the numbers are."""
    def draws(s):
        jt.set_seed(s)
        return jt.random([5]).numpy(), [tuple(int(u._host[0]) for u in jt.nn.dropout(_x(4), 0.5, True)._op.inputs[1:]) for _ in range(2)]
    (r, (first, second)), (again, calls) = draws(seed()), draws(seed())
    jt.set_seed(0)
    assert first[1:] == (0,) and second == (first[0], 1)
    if seed() is None:
        assert not np.array_equal(r, again) and calls[0] != first
    else:
        assert np.array_equal(r, np.random.default_rng(seed()).random(5).astype(np.float32)) and np.array_equal(r, again) and calls == [first, second]


@pytest.mark.parametrize("case", [
    dict(qkv=(4, 8)), dict(qkv=(2, 4, 7, 8)), dict(qkv=(2, 4, 6, 7)), dict(heads=0), dict(kv=0), dict(k_scale=False), dict(q_scale=False), dict(scale=(9,)), dict(scale_dtype="float16"),
    dict(table=(10, 5, 2)), dict(table=(10, 4, 3)), dict(table=(0, 4, 2)), dict(table_dtype="float16"), dict(positions=(2, 3)), dict(positions_dtype="float32"),
    dict(sections=[2, 1]), dict(sections=[4], positions=None), dict(sections=[5, -1], positions=(2, 2, 4)), dict(sections=[4] + [0] * 8, positions=(9, 2, 4)), dict(eps=-1.0), dict(eps=float("nan")),
    dict(table=(3, 4, 2), positions=None), dict(q_scale=False, k_scale=False, table=None, positions=None), dict(dtype="int32")])
def test_qkv_norm_rope_refuses(case):
    c = dict(dict(qkv=(2, 4, 6, 8), heads=2, kv=2, q_scale=True, k_scale=True, scale=(8,), scale_dtype="float32", table=(10, 4, 2), table_dtype="float32", positions=(2, 4), positions_dtype="int32",
                  sections=None, eps=1e-6, dtype="float32"), **case)
    scale = _x(*c["scale"], dtype=c["scale_dtype"])
    other = _x(*c["scale"]) if case.get("scale_dtype") else scale
    with pytest.raises((ValueError, TypeError)):
        jt.nn.qkv_norm_rope(_x(*c["qkv"], dtype=c["dtype"]), c["heads"], c["kv"], scale if c["q_scale"] else None, other if c["k_scale"] else None,
                            None if c["table"] is None else _x(*c["table"], dtype=c["table_dtype"]), None if c["positions"] is None else _x(*c["positions"], dtype=c["positions_dtype"]),
                            sections=c["sections"], eps=c["eps"])


def test_gradients_that_are_refused():
    """Those of a table of angles, and second ones."""
    x, table = jt.array(np.ones((1, 3, 3, 4), np.float32)), jt.nn.rope_table(8, 4)
    q, k, v = jt.nn.qkv_norm_rope(x, 1, 1, None, None, table)
    assert len(jt.grad((q * q).sum(), [x])) == 1
    with pytest.raises(NotImplementedError, match="table"):
        jt.grad((q * q).sum(), [x, table])
    (d,) = jt.grad((q * q).sum(), [x])
    with pytest.raises(NotImplementedError, match="second"):
        jt.grad(d.sum(), [x])


def test_gradient_of_the_sum_alone_is_what_arrives():
    """Nothing is dropped with p = 0: both gradients are the one of the sum, without a launch."""
    x, r, g = (jt.array(np.full((3, 4), v, np.float32)) for v in (1, 2, 3))
    y = jt.nn.dropout(x, 0.0, True, residual=r)
    dx, dr = jt.grad((y * g).sum(), [x, r])
    assert not any(isinstance(d._op, core.KernelOp) for d in (dx, dr))


def test_gradients_of_many_calls_in_one_graph():
    """Every call's gradient reads the one behind it, and the results of a call are found whatever stands between them."""
    x = y = jt.array(np.ones((2, 4), np.float32))
    for i in range(300):
        y = jt.nn.dropout(y * 2.0, 0.5, True, seed=1, offset=i, residual=y)
    (d,) = jt.grad(y.sum(), [x])
    calls, left = set(), [d]
    seen = set()
    while left:
        u = left.pop()
        if u.id in seen or u._op is None:
            continue
        seen.add(u.id)
        if isinstance(u._op, core.KernelOp):
            calls.add(u._op.call)
        left += u._op.inputs
    assert len(calls) == 300


def test_gated_linear_refuses():
    for x, w, act in ((_x(3, 4), _x(5, 4), "silu"), (_x(3, 4), _x(6, 5), "silu"), (_x(3, 4), _x(6, 4), "tanh"), (_x(3, 4), _x(6, 4, dtype="float16"), "silu"), (_x(3, 4), _x(2, 3, 4), "silu"),
                      (jt.array(np.arange(12).reshape(3, 4)), jt.array(np.arange(24).reshape(6, 4)), "silu")):
        with pytest.raises((ValueError, TypeError)):
            jt.nn.gated_linear(x, w, act)


# ---- the C boundary (nothing is launched) ---------------------------------------------------------------------------------
ADDRESS = 0x100000


def _t(dtype, *shape, ptr=ADDRESS):
    return L.tensor(ptr, dtype, shape)


def _scalar(v=3):
    return (L.FusedVar * 1)(L.FusedVar(L.VAR_SCALAR, L.DTYPE_CODE["int64"], None, 0.0, v))


def _params(q=4, k=2, v=2, paired=0, first=0, sections=(), eps=1e-6):
    return L.HeadNorm(q, k, v, paired, first, len(sections), (ctypes.c_int32 * 8)(*sections), eps)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_kernels_build_for_every_type(compile_only, dtype):
    lib = compile_only.load()
    L.check(lib.mjt_dropout(B(_t(dtype, 9, 5)), B(_t(dtype, 9, 5, ptr=ADDRESS + 2)), B(_t(dtype, 9, 5)), 0.1, _scalar(), _scalar()))
    for dim, rot, paired, first, sections in ((128, 128, 0, 1, ()), (80, 80, 1, 0, (8, 16, 16)), (6, 2, 0, 0, ()), (258, 130, 1, 1, ())):
        p = _params(paired=paired, first=first, sections=sections)
        x, q, v, s = _t(dtype, 2, 5, 8, dim), _t(dtype, 2, 5, 4, dim), _t(dtype, 2, 5, 2, dim), _t("float32", dim)
        table, at = _t("float32", 50, rot // 2, 2), _t("int32", max(1, len(sections)), 2, 5)
        L.check(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(table), B(at), B(p), B(q), B(v), B(v)))
        assert L.last_kernel().startswith("mjt_head_norm_rope_" + dtype)
        L.check(lib.mjt_head_norm_rope_grad(B(x), B(s), B(s), B(table), B(at), B(p), B(q), None, B(v), B(x), B(s), B(s)))
    for act in range(4):
        for rows, k, f in ((1, 256, 96), (40, 512, 128), (700, 640, 512), (33, 30, 7)):
            L.check(lib.mjt_gated_linear(B(_t(dtype, rows, k)), B(_t(dtype, 2 * f, k)), act, B(_t(dtype, rows, f)), B(_t("float32", rows, 2 * f))))
            L.check(lib.mjt_gated_linear_grad(B(_t(dtype, rows, f)), B(_t("float32", rows, 2 * f)), act, B(_t(dtype, rows, 2 * f))))
    L.check(lib.mjt_matmul_nearest(B(_t(dtype, 40, 30)), B(_t(dtype, 30, 20)), B(_t(dtype, 40, 20)), 0, 0))


def test_entry_points_refuse(compile_only):
    lib = compile_only.load()
    x = _t("float32", 2, 5, 8, 16)
    q, v, s, table = _t("float32", 2, 5, 4, 16), _t("float32", 2, 5, 2, 16), _t("float32", 16), _t("float32", 50, 8, 2)

    def refused(rc, *codes):
        assert rc in (codes or (L.ERR_INVALID,)), (rc, lib.mjt_last_error())

    one, at = _params(), _t("int32", 10)
    refused(lib.mjt_head_norm_rope(None, None, None, None, None, B(one), B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), None, B(table), B(at), B(one), B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(table), B(at), None, B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(table), B(at), B(_params(3)), B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(table), B(at), B(one), B(v), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(table), B(_t("int32", 7)), B(one), B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(table), B(_t("float32", 10)), B(one), B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(table), B(at), B(_params(sections=(3, 4))), B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(x), B(s), B(s), B(_t("float32", 50, 9, 2)), B(at), B(one), B(q), B(v), B(v)))
    refused(lib.mjt_head_norm_rope(B(_t("float64", 2, 5, 8, 16)), B(s), B(s), B(table), B(at), B(one), B(q), B(v), B(v)), L.ERR_UNSUPPORTED)
    refused(lib.mjt_head_norm_rope(B(_t("float32", 2, 5, 8, 30000)), None, None, B(table), B(at), B(one), None, None, None), L.ERR_UNSUPPORTED)
    refused(lib.mjt_head_norm_rope_grad(B(x), None, None, B(table), B(at), B(one), B(q), B(v), B(v), B(x), B(s), None))
    refused(lib.mjt_dropout(B(x), None, B(x), 1.5, _scalar(), _scalar()))
    refused(lib.mjt_dropout(B(x), None, B(q), 0.5, _scalar(), _scalar()))
    refused(lib.mjt_dropout(B(x), None, B(x), 0.5, None, _scalar()))
    refused(lib.mjt_dropout(B(_t("int32", 4)), None, B(_t("int32", 4)), 0.5, _scalar(), _scalar()), L.ERR_UNSUPPORTED)
    a, w, y = _t("float32", 3, 4), _t("float32", 6, 4), _t("float32", 3, 3)
    refused(lib.mjt_gated_linear(B(a), B(w), 4, B(y), None))
    refused(lib.mjt_gated_linear(B(a), B(w), 0, None, None))
    refused(lib.mjt_gated_linear(B(a), B(_t("float32", 5, 4)), 0, B(y), None))
    refused(lib.mjt_gated_linear(B(a), B(w), 0, B(a), None))
    refused(lib.mjt_gated_linear(B(a), B(w), 0, B(y), B(y)))
    refused(lib.mjt_gated_linear_grad(B(y), B(y), 0, B(w)))


def test_products_are_cut_into_whole_rounds_only_where_those_run_on_large_tiles(compile_only, monkeypatch):
    """40960 x 336 counts 320 tiles of 256 x 256, more than a round of them, but a third of each row of tiles would be empty: the product runs whole on the
    tiles that it has where nothing is cut.  What is left of a cut product runs on a kernel of its own (here the ring of four stages of one tile each)."""
    monkeypatch.setenv("MJT_NO_DISK_CACHE", "1")
    lib = compile_only.load()

    def kernel(f, m, n, k):
        L.check(f(B(_t("bfloat16", m, k)), B(_t("bfloat16", k, n)), B(_t("bfloat16", m, n)), 0, 0))
        return L.last_kernel().replace("_nearest", "")

    whole, rest = kernel(lib.mjt_matmul, 40960, 336, 1024), kernel(lib.mjt_matmul, 8192, 336, 1024)
    assert whole != rest and kernel(lib.mjt_matmul_nearest, 40960, 336, 1024) == whole
    monkeypatch.setenv("MJT_GEMM_NO_DMA", "1")               # nor without the kernel of those tiles
    for n in (336, 512):
        assert kernel(lib.mjt_matmul_nearest, 40960, n, 1024) == kernel(lib.mjt_matmul, 40960, n, 1024)


# ---- graphs of gradients (built, not run) -----------------------------------------------------------------------------------
def _calls(vs):
    return [op for op in core._graph.pending_ops(vs) if isinstance(op, core.KernelOp)]


def test_results_of_one_call_have_their_gradients_taken_together():
    x, s = _x(2, 4, 6, 8), _x(8)
    q, k, v = jt.nn.qkv_norm_rope(x, 2, 2, s, s, _x(9, 4, 2))
    dx, ds = jt.grad((q * q).sum() + (v * 2.0).sum(), [x, s])
    grads = [op for op in _calls([dx, ds]) if op.call.name == "head_norm_rope_grad"]
    assert len({id(op.call) for op in grads}) == 1 and sorted(op.index for op in grads) == [0, 1, 2]      # both scales are the same Var
    assert grads[0].call.options[-1] == (True, False, True) and list(ds.shape) == [8]


def test_the_forward_products_are_the_same_call_as_the_result():
    x, w = _x(3, 4), _x(6, 4)
    y = jt.nn.gated_linear(x, w)
    dx, dw = jt.grad((y * y).sum(), [x, w])
    fwd = [op for op in _calls([y, dx, dw]) if op.call.name == "gated_linear"]
    assert sorted(op.index for op in fwd) == [0, 1] and fwd[0].call is fwd[1].call
    assert not [op for op in _calls([y]) if op.index == 1]


def test_second_derivatives_are_refused():
    x, w = _x(3, 4), _x(6, 4)
    dx = jt.grad(jt.nn.gated_linear(x, w).sum(), x)
    with pytest.raises(NotImplementedError):
        jt.grad(dx.sum(), w)


def test_a_key_tells_calls_apart():
    def key(**kw):
        q = jt.nn.qkv_norm_rope(_x(2, 4, 6, 8), 2, 2, _x(8), _x(8), _x(9, 4, 2), **kw)[0]
        return core._graph.signature(core._graph.pending_ops([q]), [q], jt.flags)
    assert key() == key() and len({key(), key(eps=1e-5), key(interleaved=True), key(heads_first=True)}) == 4


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_a_feed_forward_layer_keeps_its_type(dtype):
    x, w, o = _x(3, 4, dtype=dtype), _x(6, 4, dtype=dtype), _x(5, 3, dtype=dtype)
    y = jt.nn.gated_ffn(x, w, o)
    assert y.dtype == dtype and y.shape == [3, 5] and [g.dtype for g in jt.grad(y.sum(), [x, w, o])] == [dtype] * 3


# ---- graphs of gradients, executed up to the launches -------------------------------------------------------------------
@pytest.fixture
def launches(compile_only, monkeypatch):
    """Graphs are executed in compile-only mode on addresses that nothing is read from; what is launched is listed."""
    class Pool:
        at = 1 << 20

        def alloc(self, n):
            Pool.at += 1 << 20
            return Pool.at, n

        def free(self, ptr, size):
            pass

    listed, launch = [], layers.launch
    monkeypatch.setenv("MJT_NO_DISK_CACHE", "1")
    monkeypatch.setattr(core, "pool", Pool())
    monkeypatch.setattr(layers, "launch", lambda ex, ops: (listed.append((ops[0].call.name, sorted(op.index for op in ops))), launch(ex, ops)))
    yield listed
    executor._plans.clear()
    gc.collect()                                            # (buffers go back to the pool they are from)


def _there(*shape):
    v = core.Var(list(shape), "float32")
    v._buf = core.Buffer(4 * v.num)
    return v


def test_gradients_of_one_gated_result_taken_one_by_one(launches):
    """Two calls of grad() and one sync: both read the same products of the forward pass, which are made once."""
    x, w = _there(3, 4), _there(6, 4)
    y = jt.nn.gated_linear(x, w)
    loss = (y * _there(3, 3)).sum()
    gx, gw = jt.grad(loss, x), jt.grad(loss, w)
    jt.sync([gx, gw])
    assert gx._op is None and gw._op is None
    assert sorted(launches) == [("gated_linear", [1])] + 2 * [("gated_linear_grad", [0])] + 2 * [("product", [0])]


def test_two_losses_over_a_shared_gated_layer(launches):
    x, w = _there(3, 4), _there(6, 4)
    y = jt.nn.gated_linear(x, w)
    grads = [g for k in range(2) for g in jt.grad((y * _there(3, 3)).sum(), [x, w])]
    jt.sync([y] + grads)
    assert all(v._op is None for v in [y] + grads)
    assert sorted(launches) == [("gated_linear", [0, 1])] + 2 * [("gated_linear_grad", [0])] + 4 * [("product", [0])]


def test_a_result_that_was_asked_for_twice_is_made_twice(launches):
    """Whoever makes the same result of one call a second time gets it, whatever else is pending."""
    x, w = _there(3, 4), _there(6, 4)
    y = jt.nn.gated_linear(x, w)
    again = [layers._result(y._op.call, 1, [x, w], [3, 6], "float32") for _ in range(2)]
    jt.sync([y] + again)
    assert y._op is None and all(v._op is None and v._buf is not None for v in again)
    assert sorted(launches) == [("gated_linear", [0, 1]), ("gated_linear", [1])]


def test_a_feed_forward_layer_in_bfloat16_is_rounded_to_nearest_throughout(launches):
    """Its second product and that product's gradients are the operators' own, not the ordinary product, which truncates."""
    x, w, o = (core.Var(list(n), "bfloat16") for n in ((3, 5, 8), (12, 8), (7, 6)))
    for v in (x, w, o):
        v._buf = core.Buffer(2 * v.num)
    y = jt.nn.gated_ffn(x, w, o)
    grads = jt.grad((y * 2.0).sum(), [x, w, o])
    assert [g.shape for g in [y] + grads] == [[3, 5, 7], [3, 5, 8], [12, 8], [7, 6]] and {g.dtype for g in [y] + grads} == {"bfloat16"}
    jt.sync([y] + grads)
    assert sorted(launches) == [("gated_linear", [0, 1]), ("gated_linear_grad", [0])] + 5 * [("product", [0])]
    with pytest.raises(ValueError):
        jt.nn.gated_ffn(x, w, _x(7, 5, dtype="bfloat16"))


@pytest.mark.parametrize("trans_a,trans_b", [(False, False), (False, True), (True, False)])
def test_gradients_of_a_product_are_products(trans_a, trans_b):
    """sum(dc * A' B') moves with a and b as the products that are taken for its gradients say."""
    rng = np.random.default_rng(4)
    m, n, k = 3, 4, 5
    shapes = [(k, m) if trans_a else (m, k), (n, k) if trans_b else (k, n), (m, n)]
    values = {}

    def var(shape):
        v = _x(*shape)
        values[v.id] = rng.standard_normal(shape)
        return v

    def times(a, b, ta, tb):
        return (a.T if ta else a) @ (b.T if tb else b)

    a, b, dc = map(var, shapes)
    c = layers._result(layers.Call("product", trans_a, trans_b), 0, [a, b], [m, n], "float32")
    got = [times(*(values[u.id] for u in g._op.inputs), *g._op.call.options) for g in layers._product_gradients(c._op, [a, b], {0: dc}, [True, True])]
    for i, (v, g) in enumerate(zip((a, b), got)):
        along = rng.standard_normal(v.shape)
        moved = [along if j == i else values[u.id] for j, u in enumerate((a, b))]
        assert abs((times(*moved, trans_a, trans_b) * values[dc.id]).sum() - (g * along).sum()) < 1e-12
