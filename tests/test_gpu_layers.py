"""Operators of transformer layers on the GPU against the plain forms in 64 bits (layers_plain.py).

Tolerances: the result's own rounding (half a unit of its type), plus what 32-bit arithmetic may add: a bound derived for each operator
from the magnitudes of what is summed, E = 2^-24 relative for each operation."""
import numpy as np
import pytest

import jittor_amd as jt
from jittor_amd import core
from jittor_amd.dtypes import bf16_bits_to_f32
import layers_plain as P
from layers_plain import E, TINY, ULP

pytestmark = pytest.mark.gpu

DTYPES = ["float32", "bfloat16", "float16"]


def _make(rng, shape, dtype, scale=1.0, shift=0.0):
    """(Var, its exact values)"""
    raw, exact = P.to_type(rng.standard_normal(shape) * scale + shift, dtype)
    return jt.from_storage(raw, dtype), exact


def _got(v):
    return v.numpy().astype(np.float64)


def _check(got, want, bound, dtype, what):
    """|got - want| within the rounding of the result and `bound`; what is not finite has to be the same."""
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)), what
    assert np.array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)]), what
    off = np.abs(got - want)[fine]
    allowed = (np.broadcast_to(bound, want.shape)[fine]) * (1 + ULP[dtype]) + ULP[dtype] * np.abs(want[fine]) + TINY[dtype]
    worst = np.argmax(off - allowed) if off.size else 0
    assert not off.size or (off <= allowed).all(), (what, off.flat[worst], allowed.flat[worst])


# ---- dropout ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (3, 5, 11), (2, 1024), (1, 4099)])
@pytest.mark.parametrize("p", [0.5, 0.1, 0.999, 1.0, 1e-9])
def test_dropout(gpu, dtype, shape, p):
    rng = np.random.default_rng(len(shape))
    (x, xe), (r, re), (g, ge) = (_make(rng, shape, dtype) for _ in range(3))
    seed, offset = -3 * (1 << 60) + 5, (1 << 63) + 9
    keep = P.kept(x.num, p, seed, offset).reshape(shape)
    f = np.float64(np.float32(1.0 / (1.0 - p))) if p < 1 else 0.0
    for residual in (None, r):
        y = jt.nn.dropout(x, p, True, seed=seed, offset=offset, residual=residual)
        grads = jt.grad((y * g).sum(), [x] + ([] if residual is None else [r]))
        jt.sync([y] + grads)
        add = 0.0 if residual is None else re
        _check(_got(y), np.where(keep, xe * f, 0.0) + add, 2 * E * (np.abs(xe * f) + np.abs(add)), dtype, "y")
        _check(_got(grads[0]), np.where(keep, ge * f, 0.0), 2 * E * np.abs(ge * f), dtype, "dx")
        if residual is not None:
            assert np.array_equal(_got(grads[1]), ge)


@pytest.mark.parametrize("dtype", DTYPES)
def test_the_residual_is_added_without_dropout_too(gpu, dtype):
    rng = np.random.default_rng(2)
    (x, xe), (r, re) = _make(rng, (5, 77), dtype), _make(rng, (5, 77), dtype)
    for y in (jt.nn.dropout(x, 0.0, True, residual=r), jt.nn.dropout(x, 0.5, False, residual=r)):
        dx = jt.grad((y * r).sum(), x)
        _check(_got(y), xe + re, 2 * E * (np.abs(xe) + np.abs(re)), dtype, "y")
        assert np.array_equal(_got(dx), re)


def test_dropout_at_the_threshold(gpu):
    """p between two multiples of 2^-16: the lower halves of the numbers decide for one element in 65536, and have to."""
    n = 1 << 17
    u = P.numbers(n, 11, 2)
    at = u[np.argsort(np.abs(u.astype(np.int64) - (1 << 31)))[:64]]
    x = jt.array(np.ones(n, np.float32))
    for t in sorted({int(v) + d for v in at[:6] for d in (0, 1)}):
        y = jt.nn.dropout(x, t / 2.0 ** 32, True, seed=11, offset=2)
        assert np.array_equal(_got(y) != 0, u >= t), t


@pytest.mark.parametrize("p", [0.5, 0.3])
def test_calls_without_a_seed_have_numbers_of_their_own(gpu, p):
    """Neither the i-th call behind set_seed(s) nor its gradient has the mask of seed s and offset i: bit 28 of the counter's second word tells them apart."""
    n = 8 * 50
    x = jt.array(np.ones(n, np.float32))
    jt.set_seed(9)
    for call in range(3):
        y = jt.nn.dropout(x, p, True)
        dx = jt.grad(y.sum(), x)
        u = []
        for g in range(n // 8):
            hi, lo = (P.philox([g, 1 << 28 | block << 31, call, 0], [9, 0]) for block in (0, 1))
            u += [((hi[j // 2] >> 16 * (j % 2)) & 0xFFFF) << 16 | (lo[j // 2] >> 16 * (j % 2)) & 0xFFFF for j in range(8)]
        keep = np.array(u, np.uint64) >= round(p * 2.0 ** 32)
        assert np.array_equal(_got(y) != 0, keep) and np.array_equal(_got(dx) != 0, keep)
        assert not np.array_equal(keep, P.kept(n, p, 9, call))
    jt.set_seed(0)


def test_dropped_infinities_and_nan_are_zero(gpu):
    n, p = 4096, 0.3
    keep = P.kept(n, p, 1, 0)
    for bad in (np.inf, -np.inf, np.nan):
        y = _got(jt.nn.dropout(jt.array(np.full(n, bad, np.float32)), p, True, seed=1))
        assert (y[~keep] == 0).all() and (np.isnan(y[keep]) if np.isnan(bad) else y[keep] == bad).all()


def test_dropout_of_nothing(gpu):
    x = jt.array(np.zeros((0, 5), np.float32))
    y = jt.nn.dropout(x, 0.5, True, seed=1)
    assert y.numpy().shape == (0, 5) and jt.grad(y.sum(), x).numpy().shape == (0, 5)


def test_dropout_replays_with_other_seeds(gpu):
    """The same graph again and again: recorded launches take each call's seed, offset and buffers."""
    rng = np.random.default_rng(3)
    for turn in range(6):
        x, xe = _make(rng, (37, 29), "float32")
        h = x * 2.0
        y = jt.nn.dropout(h, 0.25, True, seed=100 + turn, offset=turn << 33)
        dx = jt.grad((y * y).sum(), x)
        jt.sync([y, dx])
        keep = P.kept(x.num, 0.25, 100 + turn, turn << 33).reshape(x.shape)
        f = np.float64(np.float32(4.0 / 3.0))
        _check(_got(y), np.where(keep, 2 * xe * f, 0.0), 4 * E * np.abs(xe), "float32", turn)
        _check(_got(dx), np.where(keep, 8 * xe * f * f, 0.0), 64 * E * np.abs(xe), "float32", turn)


def test_dropout_past_32_bits(gpu):
    """Elements behind 2^32: the counter's upper word."""
    n = (1 << 32) + 8 * 37
    x = core.Var([n], "float16")
    jt.sync([])
    buf = core.Buffer(2 * n)
    x._buf = buf
    gpu.check(gpu.load().mjt_fill_u32(buf.ptr, 0x3C003C00, n // 2))
    y = jt.nn.dropout(x, 0.5, True, seed=5, offset=1)
    y.sync()
    at = (1 << 32) - 64
    tail = gpu.d2h(y._buf.ptr + 2 * at, [n - at], np.float16)
    for k, v in enumerate(tail):
        e = at + k
        g = e // 8
        b = P.philox([g & 0xFFFFFFFF, g >> 32, 1, 0], [5, 0])
        assert v == (2.0 if (b[e % 8 // 2] >> 16 * (e % 2)) & 0xFFFF >= 0x8000 else 0.0), e


# ---- norms of heads and rotation ------------------------------------------------------------------------------------
def _table(rng, n, pairs):
    t = rng.uniform(0, 6.28, (n, pairs))
    t = np.stack([np.cos(t), np.sin(t)], -1).astype(np.float32)
    return jt.array(t), t.astype(np.float64)


def _laid(a, lead, first):
    """[tokens, heads, dim] as the operator writes it"""
    a = a.reshape(tuple(lead) + a.shape[1:])
    return np.swapaxes(a, -3, -2) if first else a


def _heads(dtype, lead, hq, hk, dim, pairs, paired, first, sections=None, scaled=True, scale_dtype=None, per_sequence=False, given=(True, True, True), seed=0, want=(True, True, True)):
    rng = np.random.default_rng(seed)
    tokens, S = int(np.prod(lead)), lead[-1]
    x, xe = _make(rng, tuple(lead) + (hq + 2 * hk, dim), dtype, 1.5)
    xe = xe.reshape(tokens, hq + 2 * hk, dim)
    sq = sk = sqe = ske = table = positions = cos = sin = None
    if scaled:
        (sq, sqe), (sk, ske) = (_make(rng, (dim,), scale_dtype or dtype, 0.3, 1.0) for _ in range(2))
    if pairs:
        rows = 40
        table, te = _table(rng, rows, pairs)
        axes = len(sections) if sections else 1
        at = rng.integers(0, rows, (axes, S if per_sequence else tokens)).astype(np.int32)
        positions = jt.array(at.reshape(([axes] if sections else []) + ([S] if per_sequence else list(lead))))
        whole = np.tile(at, (1, tokens // S)) if per_sequence and S else at
        cos, sin = P.angles_of(te, whole, sections or [pairs], lead)
    outs = jt.nn.qkv_norm_rope(x, hq, hk, sq, sk, table, positions, sections=sections, eps=1e-5, interleaved=paired, heads_first=first)
    parts = {"q": (slice(0, hq), sqe), "k": (slice(hq, hq + hk), ske), "v": (slice(hq + hk, None), None)}
    loss, gs = None, {}
    for name, o, use in zip("qkv", outs, given):
        if use:
            g, ge = _make(rng, tuple(o.shape), dtype)
            gs[name] = np.swapaxes(ge, -3, -2).reshape(tokens, -1, dim) if first else ge.reshape(tokens, -1, dim)
            term = (o * g).sum()
            loss = term if loss is None else loss + term
    targets = [x] + ([sq, sk] if scaled else [])
    grads = jt.grad(loss, targets) if loss is not None else []
    jt.sync(list(outs) + [d for d, w in zip(grads, want) if w])
    dx, sums = np.zeros_like(xe), {}
    dxs = np.zeros_like(xe)
    for name, o in zip("qkv", outs):
        rows_, scale = parts[name]
        part = xe[:, rows_]
        if name == "v":
            assert np.array_equal(_got(o), _laid(part, lead, first)), "v"
            if name in gs:
                dx[:, rows_] = gs[name]
            continue
        z = part / np.sqrt((part * part).mean(-1, keepdims=True) + 1e-5) * scale if scaled else part
        size = P.pair_size(z, cos, paired)
        # mean of squares, root and quotient: up to dim / 2 + 8 roundings; two more multiplications and the turn
        _check(_got(o), _laid(P.head_norm(part, scale, cos, sin, 1e-5, paired), lead, first), _laid((dim / 2 + 16) * E * size, lead, first), dtype, name)
        if name in gs:
            dx[:, rows_], ds, dxs[:, rows_], dss = P.head_norm_grad(part, scale, cos, sin, 1e-5, paired, gs[name])
            sums[name] = (ds, dss)
    if loss is None:
        return
    if want[0]:
        _check(_got(grads[0]).reshape(dx.shape), dx, (2 * dim + 32) * E * dxs, dtype, "dx")
    if scaled:
        for name, d, w in zip("qk", grads[1:], want[1:]):
            if not w:
                continue
            ds, dss = sums.get(name, (np.zeros(dim), np.zeros(dim)))
            _check(_got(d), ds, (tokens * (hq + 2 * hk) + dim + 32) * E * dss, scale_dtype or dtype, "d" + name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("paired", [False, True])
@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("lead,hq,hk,dim,pairs", [((1, 1), 1, 1, 2, 1), ((2, 5), 4, 2, 128, 64), ((3, 7), 3, 1, 80, 40), ((1, 33), 5, 5, 64, 16), ((2, 9), 2, 1, 6, 2), ((1, 4), 2, 1, 258, 65)])
def test_head_norms_and_rotation(gpu, dtype, paired, first, lead, hq, hk, dim, pairs):
    _heads(dtype, lead, hq, hk, dim, pairs, paired, first)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("sections,pairs", [([8, 16, 16], 40), ([3, 0, 5], 8), ([1] * 8, 8), ([4], 4)])
@pytest.mark.parametrize("per_sequence", [False, True])
def test_positions_on_several_axes(gpu, dtype, sections, pairs, per_sequence):
    for paired in (False, True):
        _heads(dtype, (2, 11), 3, 2, 80, pairs, paired, True, sections=sections, per_sequence=per_sequence, seed=len(sections))


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_tokens_and_heads(gpu, dtype):
    _heads(dtype, (3, 700), 16, 4, 128, 64, False, True, seed=4)
    _heads(dtype, (5000,), 1, 1, 64, 32, True, False, seed=5)
    _heads(dtype, (2, 3), 70, 10, 96, 48, False, True, seed=6)


@pytest.mark.parametrize("dtype", DTYPES)
def test_passes_larger_than_the_caches_keep(gpu, dtype):
    """Read and written by 32 MB and more, forward and backward: other loads and stores, the same results."""
    _heads(dtype, (2, 1750), 16, 4, 128, 64, False, True, seed=14)
    _heads(dtype, (2, 1801), 40, 5, 64, 32, True, True, sections=[8, 16, 8], seed=15)
    _heads(dtype, (1, 1003), 40, 3, 192, 48, False, True, seed=16)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("paired", [False, True])
@pytest.mark.parametrize("dim,pairs", [(128, 64), (128, 32), (256, 64), (128, 0), (64, 32)])
def test_layouts_of_large_passes(gpu, dtype, paired, dim, pairs):
    """Pieces of rows side by side and half a row apart, turned whole, in part and not at all."""
    _heads(dtype, (2, 190000 // dim), 16, 4, dim, pairs, paired, True, seed=dim + pairs)


def test_without_rotation_without_norm_and_with_scales_of_another_type(gpu):
    _heads("bfloat16", (2, 6), 4, 2, 64, 0, False, False)
    _heads("bfloat16", (2, 6), 4, 2, 64, 32, False, True, scaled=False)
    _heads("float16", (2, 6), 4, 2, 72, 36, True, True, scale_dtype="float32")
    _heads("float32", (2, 6), 4, 2, 72, 10, True, True, scale_dtype="bfloat16")


@pytest.mark.parametrize("given", [(True, False, False), (False, True, False), (False, False, True), (True, False, True)])
def test_gradients_of_some_of_the_results(gpu, given):
    _heads("float32", (2, 6), 4, 2, 64, 32, False, True, given=given)
    _heads("bfloat16", (2, 6), 4, 2, 64, 32, True, False, given=given, want=(False, True, False))
    _heads("bfloat16", (2, 6), 4, 2, 64, 32, True, False, given=given, want=(True, False, False))


def test_long_heads(gpu):
    _heads("float32", (2, 3), 2, 1, 1022, 511, False, True)
    _heads("bfloat16", (2, 3), 2, 1, 1024, 512, True, True)
    _heads("float32", (1, 2), 1, 1, 4096, 100, False, True)
    _heads("float16", (1, 2), 1, 1, 4096, 2048, True, False)


def test_heads_that_are_zero_or_not_finite(gpu):
    """A head of zeros stays zero; an infinity or NaN stays in its own head."""
    rng = np.random.default_rng(8)
    x = rng.standard_normal((1, 6, 4, 64)).astype(np.float32)
    x[0, 1, 0] = 0.0
    x[0, 2, 1, 5] = np.nan
    x[0, 3, 2, 7] = np.inf
    s = jt.array(np.ones(64, np.float32))
    t, _ = _table(rng, 6, 32)
    q, k, v = jt.nn.qkv_norm_rope(jt.array(x), 2, 1, s, s, t)
    good = x.copy()
    good[~np.isfinite(good)] = 1.0
    q1, k1, v1 = jt.nn.qkv_norm_rope(jt.array(good), 2, 1, s, s, t)
    q, k, v, q1, k1, v1 = (_got(u) for u in (q, k, v, q1, k1, v1))
    assert (q[0, 1, 0] == 0).all() and np.isnan(q[0, 2, 1]).all() and np.isnan(k[0, 3, 0]).any() and np.array_equal(v, x[:, :, 3:].astype(np.float64), equal_nan=True)
    q[0, 2, 1] = q1[0, 2, 1]
    k[0, 3, 0] = k1[0, 3, 0]
    assert np.array_equal(q, q1) and np.array_equal(k, k1)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("size", [1e-18, 1e-19, 1e-20])
def test_heads_whose_mean_square_is_subnormal(gpu, dtype, size):
    """Without eps.  Squares, their sum and its mean are each within half the least subnormal number, 2^-150, or E of their size; r has half the
    relative error of the mean."""
    rng = np.random.default_rng(31)
    (x, xe), (s, se), (g, ge) = _make(rng, (1, 5, 3, 64), dtype, size), _make(rng, (64,), dtype, 0.2, 1.0), _make(rng, (1, 5, 3, 64), dtype)
    y = jt.nn.head_norm_rope(x, s, eps=0.0)
    dx = jt.grad((y * g).sum(), x)
    mean = (xe[0] ** 2).mean(-1, keepdims=True)
    off = 64 * E + 3 * 2.0 ** -150 / mean
    want = P.head_norm(xe[0], se, None, None, 0.0, False)
    _check(_got(y)[0], want, off * np.abs(want), dtype, "y")
    want, _, sizes, _ = P.head_norm_grad(xe[0], se, None, None, 0.0, False, ge[0])
    _check(_got(dx)[0], want, 4 * off * sizes, dtype, "dx")


def test_positions_outside_the_table_make_nan_of_what_they_turn(gpu):
    rng = np.random.default_rng(9)
    x, g = (jt.array(rng.standard_normal((1, 5, 3, 16)).astype(np.float32)) for _ in range(2))
    s = jt.array(np.ones(16, np.float32))
    t, _ = _table(rng, 10, 4)
    at = np.array([[0, 10, -1, 9, 2 ** 31 - 1]], np.int32)
    q, k, v = jt.nn.qkv_norm_rope(x, 1, 1, s, s, t, jt.array(at))
    dx = jt.grad((q * g[:, :, :1]).sum(), x)
    bad = (at[0] < 0) | (at[0] >= 10)
    q, k, v, dx = _got(q), _got(k), _got(v), _got(dx)
    for y in (q, k):
        assert np.isnan(y[0, bad, :, :8]).all() and np.isfinite(y[0, bad, :, 8:]).all() and np.isfinite(y[0, ~bad]).all()
    assert np.isfinite(v).all() and np.isfinite(dx[0, ~bad]).all() and np.isnan(dx[0, bad][:, 0]).all() and (dx[0, :, 1:] == 0).all()


def test_positions_count_along_each_sequence_where_there_are_none(gpu):
    rng = np.random.default_rng(10)
    x = jt.array(rng.standard_normal((3, 7, 4, 8)).astype(np.float32))
    s = jt.array(np.ones(8, np.float32))
    t, _ = _table(rng, 9, 4)
    for first in (False, True):
        a = jt.nn.qkv_norm_rope(x, 2, 1, s, s, t, heads_first=first)
        b = jt.nn.qkv_norm_rope(x, 2, 1, s, s, t, jt.array(np.arange(7, dtype=np.int32)), heads_first=first)
        for u, w in zip(a, b):
            assert np.array_equal(_got(u), _got(w))


def test_no_tokens(gpu):
    s = jt.array(np.ones(8, np.float32))
    x = jt.array(np.zeros((2, 0, 4, 8), np.float32))
    outs = jt.nn.qkv_norm_rope(x, 2, 1, s, s)
    dx, ds = jt.grad(outs[0].sum() + outs[2].sum(), [x, s])
    assert outs[0].numpy().shape == (2, 0, 2, 8) and dx.numpy().shape == (2, 0, 4, 8) and (ds.numpy() == 0).all()


def test_heads_of_one_kind(gpu):
    rng = np.random.default_rng(11)
    x, xe = _make(rng, (2, 5, 3, 32), "bfloat16")
    s, se = _make(rng, (32,), "bfloat16", 0.3, 1.0)
    t, te = _table(rng, 5, 16)
    y = jt.nn.head_norm_rope(x, s, t, eps=1e-5)
    cos, sin = P.angles_of(te, np.tile(np.arange(5), 2)[None], [16], None)
    want = P.head_norm(xe.reshape(10, 3, 32), se, cos, sin, 1e-5, False)
    ds = jt.grad(y.sum(), s)
    _check(_got(y).reshape(10, 3, 32), want, 64 * E * P.pair_size(np.abs(want), cos, False) + 64 * E, "bfloat16", "y")
    _, dse, _, dss = P.head_norm_grad(xe.reshape(10, 3, 32), se, cos, sin, 1e-5, False, np.ones((10, 3, 32)))
    _check(_got(ds), dse, 128 * E * dss, "bfloat16", "ds")


def test_one_launch_for_three_results_and_replays(gpu):
    rng = np.random.default_rng(12)
    s = jt.array(np.ones(64, np.float32))
    t, te = _table(rng, 6, 32)
    cos, sin = P.angles_of(te, np.arange(6)[None], [32], None)
    for turn in range(5):
        x, xe = _make(rng, (1, 6, 4, 64), "float32")
        before = dict(jt.executor_stats)
        outs = jt.nn.qkv_norm_rope(x, 2, 1, s, s, t)
        dx = jt.grad((outs[0] * outs[0]).sum() + outs[1].sum(), x)
        jt.sync(list(outs) + [dx])
        if turn == 0:
            assert jt.executor_stats["launches"] - before["launches"] <= 4         # forward, the seeds' two groups, backward
        for o, rows in zip(outs[:2], (slice(0, 2), slice(2, 3))):
            want = P.head_norm(xe[0][:, rows], np.ones(64), cos, sin, 1e-6, False)
            _check(_got(o)[0], want, 64 * E * P.pair_size(np.abs(want), cos, False), "float32", turn)
        # a turn changes no length: sum q^2 = dim for every head whatever x, so dx of the queries is the eps's share alone
        assert np.abs(_got(dx)[0][:, :2]).max() < 1e-3


def _filled(gpu, shape, dtype, word):
    """A Var whose every 32 bits are `word`, without a copy of it in host memory."""
    v = core.Var(list(shape), dtype)
    v._buf = core.Buffer(v.nbytes)
    gpu.check(gpu.load().mjt_fill_u32(v._buf.ptr, word, v.nbytes // 4))
    return v


def test_heads_past_32_bits(gpu):
    """Elements behind 2^32: the last tokens of [2^19 + 3, 64, 128], forward and backward."""
    rng = np.random.default_rng(21)
    tokens, last = (1 << 19) + 3, 4
    x = _filled(gpu, (1, tokens, 64, 128), "float16", 0x3C003C00)
    raw, xe = P.to_type(rng.standard_normal((last, 64, 128)), "float16")
    gpu.h2d(x._buf.ptr + 2 * (tokens - last) * 64 * 128, raw)
    (s, se), (t, te) = _make(rng, (128,), "float16", 0.3, 1.0), _table(rng, 40, 64)
    at = (np.arange(tokens) % 40).astype(np.int32)
    cos, sin = P.angles_of(te, at[None, -last:], [64], (1, last))
    for first in (False, True):
        q, k, v = jt.nn.qkv_norm_rope(x, 62, 1, s, s, t, jt.array(at[None]), eps=1e-5, heads_first=first)
        dq = _filled(gpu, q.shape, "float16", 0x3C003C00)
        (dx,) = jt.grad((q * dq).sum(), [x])
        jt.sync([q, k, v, dx])
        def tail(u, heads):
            if not first:
                return gpu.d2h(u._buf.ptr + 2 * (tokens - last) * heads * 128, [last, heads, 128], np.float16).astype(np.float64)
            return np.stack([gpu.d2h(u._buf.ptr + 2 * ((h * tokens) + tokens - last) * 128, [last, 128], np.float16) for h in range(heads)], 1).astype(np.float64)
        for u, rows in ((q, slice(0, 62)), (k, slice(62, 63))):
            part = xe[:, rows]
            z = part / np.sqrt((part * part).mean(-1, keepdims=True) + 1e-5) * se
            _check(tail(u, part.shape[1]), P.head_norm(part, se, cos, sin, 1e-5, False), (64 + 16) * E * P.pair_size(z, cos, False), "float16", rows)
        assert np.array_equal(tail(v, 1), xe[:, 63:])
        want, _, off, _ = P.head_norm_grad(xe[:, :62], se, cos, sin, 1e-5, False, np.ones((last, 62, 128)))
        got = gpu.d2h(dx._buf.ptr + 2 * (tokens - last) * 64 * 128, [last, 64, 128], np.float16).astype(np.float64)
        _check(got[:, :62], want, (2 * 128 + 32) * E * off, "float16", "dx")
        assert (got[:, 62:] == 0).all()
        del q, k, v, dq, dx


@pytest.mark.parametrize("rows", [1, 24, 300])
def test_weights_past_32_bits(gpu, rows):
    """2^21 + 48 rows of 2048: the last columns of both halves on each of the routes."""
    k, f = 2048, (1 << 20) + 24
    w = _filled(gpu, (2 * f, k), "float16", 0x3C003C00)
    for row, value in ((f - 1, 2.0), (2 * f - 1, 3.0), (2 * f - 2, -1.0)):
        gpu.h2d(w._buf.ptr + 2 * row * k, np.full(k, value, np.float16))
    x = jt.array(np.full((rows, k), 1.0 / k, np.float16))
    y = jt.nn.gated_linear(x, w, "sigmoid")
    y.sync()
    s = lambda g: 1.0 / (1.0 + np.exp(-g))
    want = np.array([s(1.0)] * 6 + [-s(1.0), 3.0 * s(2.0)])
    for row in sorted({0, rows - 1}):
        got = gpu.d2h(y._buf.ptr + 2 * (row * f + f - 8), [8], np.float16).astype(np.float64)
        _check(got, want, 64 * E * np.abs(want), "float16", row)


# ---- gated projections ------------------------------------------------------------------------------------------------
def _gated(dtype, rows, k, f, act, lead=None, seed=0):
    rng = np.random.default_rng(seed)
    (x, xe), (w, we), (g, ge) = _make(rng, (rows, k), dtype), _make(rng, (2 * f, k), dtype, 1.5 / max(1, k) ** 0.5), _make(rng, (rows, f), dtype)
    y = jt.nn.gated_linear(x, w, act)
    want, off = P.gated(xe, we, act)
    _check(_got(y), want, off, dtype, "y alone")
    y = jt.nn.gated_linear(x, w, act)
    dx, dw = jt.grad((y * g).sum(), [x, w])
    jt.sync([y, dx, dw])
    _check(_got(y), want, off, dtype, "y")
    (dxe, dxo), (dwe, dwo) = P.gated_grad(xe, we, act, ge, dtype)
    _check(_got(dx), dxe, dxo, dtype, "dx")
    _check(_got(dw), dwe, dwo, dtype, "dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu", "sigmoid"])
@pytest.mark.parametrize("rows,k,f", [(1, 64, 16), (3, 40, 24), (17, 129, 33), (70, 256, 96)])
def test_gated_projections(gpu, dtype, act, rows, k, f):
    _gated(dtype, rows, k, f, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(1, 1, 1), (1, 4096, 48), (2, 72, 1), (16, 512, 640), (33, 2048, 16), (64, 8, 8), (65, 320, 100), (128, 64, 64), (129, 192, 260), (300, 448, 520), (1, 1000, 333),
                                      (260, 1024, 1030), (513, 128, 384)])
def test_gated_sizes(gpu, dtype, rows, k, f):
    _gated(dtype, rows, k, f, "silu", seed=rows + k)


def test_gated_large_tiles(gpu):
    _gated("bfloat16", 2100, 256, 4100, "gelu")
    _gated("float16", 2048, 512, 4096, "silu")


@pytest.mark.parametrize("act,ends", [("silu", (0.0, np.inf)), ("gelu", (0.0, np.inf)), ("relu", (0.0, np.inf)), ("sigmoid", (0.0, 1.0))])
@pytest.mark.parametrize("rows", [1, 200])
def test_gates_at_the_ends_of_the_range(gpu, act, ends, rows):
    """Gates of both infinities, of the type's extremes and NaN: the activation's limits, and gradients without NaN where it is flat."""
    values = np.array([-np.inf, np.inf, -3e38, 3e38, -200.0, 200.0, np.nan, 0.0], np.float32)
    x = np.zeros((rows, 8), np.float32)
    x[:, 0] = 1.0
    w = np.zeros((16, 8), np.float32)
    w[:8, 0] = values
    w[8:, 0] = 1.0
    x[:, 1:] = 0.0
    y = jt.nn.gated_linear(jt.array(x[:, :1].copy()), jt.array(w[:, :1].copy()), act)
    got = _got(y)
    low, high = ends
    assert (got[:, [0, 2]] == low).all() and (got[:, 1] == high).all() and np.isnan(got[:, 6]).all()
    assert np.allclose(got[:, 3], 3e38 if high == np.inf else 1.0, rtol=1e-6) and np.allclose(got[:, 5], 200.0 if high == np.inf else 1.0) and np.abs(got[:, 4]).max() < 1e-30
    v = jt.array(x[:, :1].copy())
    dw = _got(jt.grad(jt.nn.gated_linear(v, jt.array(w[:, :1].copy()), act).sum(), jt.array(w[:, :1].copy())))
    assert np.isfinite(dw).all()                      # (a weight that the result does not depend on)
    wv = jt.array(w[:, :1].copy())
    dw = _got(jt.grad(jt.nn.gated_linear(v, wv, act).sum(), wv))[:, 0]
    slope = 1.0 if high == np.inf else 0.0
    assert (dw[[0, 2, 4]] == 0).all() and (dw[[1, 3, 5]] == rows * slope).all()


def test_gated_of_nothing(gpu):
    for rows, k, f in ((0, 8, 4), (3, 8, 0), (3, 0, 4)):
        x, w = jt.array(np.zeros((rows, k), np.float32)), jt.array(np.zeros((2 * f, k), np.float32))
        y = jt.nn.gated_linear(x, w)
        dx, dw = jt.grad(y.sum(), [x, w])
        assert y.numpy().shape == (rows, f) and (y.numpy() == 0).all() and dx.numpy().shape == (rows, k) and dw.numpy().shape == (2 * f, k) and (dw.numpy() == 0).all()


def test_gated_keeps_leading_axes_and_runs_the_forward_product_once(gpu):
    rng = np.random.default_rng(5)
    (x, xe), (w, we) = _make(rng, (2, 3, 40, 64), "bfloat16"), _make(rng, (64, 64), "bfloat16", 0.2)
    y = jt.nn.gated_linear(x, w)
    dx, dw = jt.grad(y.sum(), [x, w])
    jt.sync([y, dx, dw])
    want, off = P.gated(xe.reshape(-1, 64), we, "silu")
    assert y.shape == [2, 3, 40, 32] and dx.shape == [2, 3, 40, 64]
    _check(_got(y).reshape(-1, 32), want, off, "bfloat16", "y")
    (dxe, dxo), (dwe, dwo) = P.gated_grad(xe.reshape(-1, 64), we, "silu", np.ones((240, 32)), "bfloat16")
    _check(_got(dx).reshape(-1, 64), dxe, dxo, "bfloat16", "dx")
    _check(_got(dw), dwe, dwo, "bfloat16", "dw")


def test_gradients_asked_for_after_the_result_has_been_computed(gpu):
    rng = np.random.default_rng(6)
    (x, xe), (w, we) = _make(rng, (130, 64), "float16"), _make(rng, (192, 64), "float16", 0.2)
    y = jt.nn.gated_linear(x, w, "gelu")
    y.sync()
    dx, dw = jt.grad((y * 2.0).sum(), [x, w])
    (dxe, dxo), (dwe, dwo) = P.gated_grad(xe, we, "gelu", np.full((130, 96), 2.0), "float16")
    _check(_got(dx), dxe, dxo, "float16", "dx")
    _check(_got(dw), dwe, dwo, "float16", "dw")


@pytest.mark.parametrize("replay", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_gradients_of_one_gated_layer_taken_one_by_one(gpu, replay, dtype):
    """Two calls of grad() over one layer, then one sync or two: the values of a single call, and of two losses each its own."""
    rng = np.random.default_rng(41)
    with jt.flag_scope(enable_replay=replay):
        for turn in range(4):
            (x, xe), (w, we) = _make(rng, (21, 40), dtype), _make(rng, (2 * 24, 40), dtype, 0.2)
            (g, ge), (h, he) = _make(rng, (21, 24), dtype), _make(rng, (21, 24), dtype)
            y = jt.nn.gated_linear(x, w)
            loss, other = (y * g).sum(), (y * h).sum()
            dx, dw = jt.grad(loss, x), jt.grad(loss, w)
            hx, hw = jt.grad(other, [x, w])
            if turn % 2:
                jt.sync([dw])
            jt.sync([hw, dx, dw, hx])
            for e, (ux, uw) in ((ge, (dx, dw)), (he, (hx, hw))):
                (want_x, off_x), (want_w, off_w) = P.gated_grad(xe, we, "silu", e, dtype)
                _check(_got(ux), want_x, off_x, dtype, ("dx", turn))
                _check(_got(uw), want_w, off_w, dtype, ("dw", turn))


def test_gated_replays(gpu):
    rng = np.random.default_rng(7)
    w, we = _make(rng, (256, 128), "bfloat16", 0.1)
    for turn in range(5):
        x, xe = _make(rng, (40, 128), "bfloat16")
        y = jt.nn.gated_linear(x, w)
        dx, dw = jt.grad((y * 1.0).sum(), [x, w])
        jt.sync([y, dx, dw])
        want, off = P.gated(xe, we, "silu")
        _check(_got(y), want, off, "bfloat16", turn)
        (dxe, dxo), (dwe, dwo) = P.gated_grad(xe, we, "silu", np.ones((40, 128)), "bfloat16")
        _check(_got(dx), dxe, dxo, "bfloat16", turn)
        _check(_got(dw), dwe, dwo, "bfloat16", turn)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f,n", [(1, 64, 48, 40), (37, 33, 21, 19), (200, 128, 96, 136)])
def test_feed_forward_layers(gpu, dtype, rows, k, f, n):
    """Both products and all gradients.  Beyond P.gated and P.gated_grad: what arrives at the second product has been rounded to the type, and so has
    the gradient that arrives at the first."""
    rng = np.random.default_rng(rows)
    (x, xe), (w, we), (o, oe), (g, ge) = (_make(rng, s, dtype, c) for s, c in (((rows, k), 1.0), ((2 * f, k), 0.2), ((n, f), 0.3), ((rows, n), 1.0)))
    y = jt.nn.gated_ffn(x, w, o)
    assert y.dtype == dtype
    dx, dw, do = jt.grad((y * g).sum(), [x, w, o])
    jt.sync([y, dx, dw, do])
    he, off = P.gated(xe, we, "silu")
    off = off * (1 + ULP[dtype]) + ULP[dtype] * np.abs(he) + TINY[dtype]
    size = np.abs(he) + off
    _check(_got(y), he @ oe.T, off @ np.abs(oe).T + 2 * f * E * (size @ np.abs(oe).T), dtype, "y")
    _check(_got(do), ge.T @ he, np.abs(ge).T @ off + 2 * rows * E * (np.abs(ge).T @ size), dtype, "dw_out")
    dh = ge @ oe
    edh = 2 * n * E * (np.abs(ge) @ np.abs(oe))
    edh = edh * (1 + ULP[dtype]) + ULP[dtype] * np.abs(dh) + TINY[dtype]
    (dxe, dxo), (dwe, dwo) = P.gated_grad(xe, we, "silu", dh, dtype)
    both = xe @ we.T
    a, da = P.activation("silu", both[:, :f])
    ed = 1.1 * np.concatenate([edh * np.abs(both[:, f:] * da), edh * np.abs(a)], 1) + 1e-5 * np.tile(edh, 2)      # (errors of a, da and up on top of edh's: far below a tenth)
    _check(_got(dx), dxe, dxo + ed @ np.abs(we), dtype, "dx")
    _check(_got(dw), dwe, dwo + ed.T @ np.abs(xe), dtype, "dw_in")


def test_a_feed_forward_layer_in_bfloat16_does_not_drift(gpu):
    """Truncated results are half a unit too small on average; rounded to nearest their errors cancel, also in the gradients."""
    rng = np.random.default_rng(8)
    (x, xe), (w, we), (o, oe), (g, ge) = (_make(rng, s, "bfloat16", c) for s, c in (((256, 64), 1.0), ((128, 64), 0.2), ((96, 64), 0.3), ((256, 96), 1.0)))
    h = jt.nn.gated_linear(x, w)
    y = jt.nn.gated_ffn(x, w, o)
    do = jt.grad((y * g).sum(), o)
    he = _got(h)
    for got, want in ((_got(y), he @ oe.T), (_got(do), ge.T @ he)):
        unit = 2.0 ** (np.floor(np.log2(np.abs(want))) - 7)
        # the mean of n errors, even over half a unit to either side, has a deviation of 0.29 / sqrt(n); truncated results are at -0.5
        assert abs(((np.abs(got) - np.abs(want)) / unit).mean()) < 6 * 0.29 / np.sqrt(want.size)


@pytest.mark.parametrize("m,k,n,ta,tb", [(40, 30, 20, 0, 0), (256, 512, 256, 0, 1), (512, 256, 512, 1, 0), (64, 4096, 64, 1, 0), (7, 33, 9, 0, 1), (9300, 1024, 2048, 1, 0), (9300, 1024, 2048, 0, 0)])
def test_products_rounded_to_nearest(gpu, m, k, n, ta, tb):
    """mjt_matmul_nearest on each of the product kernels' routes: whole, in slices, plain."""
    import ctypes
    from jittor_amd import _lib as L
    rng = np.random.default_rng(m)
    (a, ae), (b, be) = _make(rng, (k, m) if ta else (m, k), "bfloat16"), _make(rng, (n, k) if tb else (k, n), "bfloat16")
    c = core.Var([m, n], "bfloat16")
    jt.sync([a, b])
    c._buf = core.Buffer(c.nbytes)
    t = [L.tensor(v._device_ptr(), v.dtype, v.shape) for v in (a, b, c)]
    L.check(L.load().mjt_matmul_nearest(*[ctypes.byref(u) for u in t], ta, tb))
    x, y = ae.T if ta else ae, be.T if tb else be
    _check(bf16_bits_to_f32(L.d2h(c._buf.ptr, c.shape, np.uint16)).astype(np.float64), x @ y, (k + 2) * E * (np.abs(x) @ np.abs(y)), "bfloat16", "c")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("route,shapes", [("few", [(1, 8, 8), (16, 264, 100), (5, 4104, 24), (7, 512, 9)]),
                                          ("tiles", [(1, 64, 1), (130, 72, 70), (257, 320, 129), (90, 1000, 200)]),
                                          ("mfma", [(1, 8, 1), (65, 40, 33), (130, 200, 130), (200, 1032, 260), (64, 64, 64)]),
                                          ("product", [(3, 40, 24), (130, 264, 70)])])
def test_every_route_of_gated_projections(gpu, monkeypatch, dtype, route, shapes):
    """Each kernel on sizes that fill its tiles badly, whichever the sizes would go to."""
    monkeypatch.setenv("MJT_GATED", route)
    for tile in ("128", "256") if route == "tiles" else ("",):
        if tile:
            monkeypatch.setenv("MJT_GEMM_DMA", tile)
        for rows, k, f in shapes:
            k = max(k, 64) if route == "tiles" else k
            rng = np.random.default_rng(rows)
            (x, xe), (w, we) = _make(rng, (rows, k), dtype), _make(rng, (2 * f, k), dtype, 1.5 / k ** 0.5)
            want, off = P.gated(xe, we, "silu")
            y = jt.nn.gated_linear(x, w)
            _check(_got(y), want, off, dtype, (route, tile, rows, k, f))
            if route == "few" or route == "tiles" and dtype != "float32":
                assert gpu.last_kernel().startswith("mjt_gated_" + route), gpu.last_kernel()
            y = jt.nn.gated_linear(x, w)
            both = core._graph.kernel_var(core.KernelOp, y._op.call, 1, [x, w], [rows, 2 * f], "float32")
            both.sync()                                     # gate and up alone
            _check(_got(both), xe @ we.T, (k + 2) * E * (np.abs(xe) @ np.abs(we).T), "float32", (route, tile, rows, k, f))
            jt.sync([y])
            _check(_got(y), want, off, dtype, (route, tile, rows, k, f))


def test_gated_in_blocks_of_rows_without_memory_for_all(gpu):
    """An odd width goes to the plain product; gate and up of 2^25 values a block."""
    _gated("bfloat16", 70, 33, (1 << 19) + 3, "relu")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ta,tb", [(0, 0), (1, 0), (0, 1)])
@pytest.mark.parametrize("m,n,k", [(70, 9, 65), (9, 70, 400), (8, 8, 33), (5, 300, 77), (300, 7, 129), (129, 131, 127), (257, 385, 1001), (1, 1, 1), (3, 2, 9), (64, 71, 4099), (700, 1030, 61), (1027, 515, 901), (1030, 1099, 259),
                                    (2563, 1290, 133)])
def test_products_of_rows_of_any_length(gpu, dtype, ta, tb, m, n, k):
    """Operands whose rows are no whole 16-byte pieces, as they lie where they have k innermost or a piece of columns; an infinity behind the
    last element of each is no part of it."""
    import ctypes
    rng = np.random.default_rng(m + n + k)
    raws = [P.to_type(rng.standard_normal(shape), dtype) for shape in ((k, m) if ta else (m, k), (n, k) if tb else (k, n))]
    whole = [jt.from_storage(np.concatenate([raw.reshape(-1), np.full(64, P.to_type(np.array(np.inf), dtype)[0])]), dtype) for raw, _ in raws]
    whole.append(jt.from_storage(np.full(m * n + 64, P.to_type(np.array(7.0), dtype)[0]), dtype))
    pointers = [v.raw_ptr() for v in whole]
    t = [gpu.tensor(p, dtype, shape) for p, shape in zip(pointers, [raws[0][0].shape, raws[1][0].shape, (m, n)])]
    gpu.check(gpu.load().mjt_matmul_nearest(*[ctypes.byref(u) for u in t], ta, tb))
    wide = 4 if dtype == "float32" else 8
    if ((m if ta else k) % wide or (k if tb else n) % wide) and (ta == 0 or m >= wide) and (tb == 1 or n >= wide):
        assert "_ragged" in gpu.last_kernel()
    a, b = raws[0][1].T if ta else raws[0][1], raws[1][1].T if tb else raws[1][1]
    got = gpu.d2h(pointers[2], [m * n + 64], raws[0][0].dtype)               # (the Var still has what it was made from)
    got = (bf16_bits_to_f32(got) if dtype == "bfloat16" else got).astype(np.float64)
    _check(got[:m * n].reshape(m, n), a @ b, (k + 2) * E * (np.abs(a) @ np.abs(b)), dtype, (ta, tb))
    assert (got[m * n:] == 7.0).all()


@pytest.mark.parametrize("ta,tb", [(0, 0), (1, 0), (0, 1)])
@pytest.mark.parametrize("m,n,k", [(2563, 1290, 61), (2560, 1280, 64), (2048, 1412, 96), (1290, 2563, 33), (2100, 1300, 127)])
def test_short_sums_on_large_tiles(gpu, ta, tb, m, n, k):
    """Two to four stages of float32 as bfloat16 parts, and one value that needs the float32 loop."""
    import ctypes
    rng = np.random.default_rng(k)
    a, b = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    a[7, k - 1] = np.inf
    x, y = jt.array(a.T.copy() if ta else a), jt.array(b.T.copy() if tb else b)
    c = core.Var([m, n], "float32")
    c._buf = core.Buffer(c.nbytes)
    gpu.check(gpu.load().mjt_matmul_nearest(*[ctypes.byref(gpu.tensor(v.raw_ptr(), "float32", v.shape)) for v in (x, y)], ctypes.byref(gpu.tensor(c._buf.ptr, "float32", c.shape)), ta, tb))
    assert "128x128" in gpu.last_kernel() and "_parts" in gpu.last_kernel()
    got = gpu.d2h(c._buf.ptr, [m, n], np.float32).astype(np.float64)
    assert np.array_equal(got[7], np.copysign(np.inf, b[-1].astype(np.float64)))
    a[7, k - 1] = 0.0
    rows = np.arange(m) != 7
    a64, b64 = a[rows].astype(np.float64), b.astype(np.float64)
    _check(got[rows], a64 @ b64, (k + 2) * E * (np.abs(a64) @ np.abs(b64)), "float32", (ta, tb))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("ta,tb", [(0, 0), (1, 0), (0, 1)])
@pytest.mark.parametrize("m,n,k", [(131, 261, 1031), (1027, 515, 901)])
def test_infinities_stay_in_their_rows_and_columns(gpu, dtype, ta, tb, m, n, k):
    """Rows of any length with an infinity in the last place of one operand and a NaN in the other's: nothing else is touched."""
    import ctypes
    rng = np.random.default_rng(9)
    a, b = rng.standard_normal((m, k)), rng.standard_normal((k, n))
    a[m - 1, k - 1], b[0, n - 1] = np.inf, np.nan
    (ra, ae), (rb, be) = P.to_type(a.T.copy() if ta else a, dtype), P.to_type(b.T.copy() if tb else b, dtype)
    (x, y, c) = (jt.from_storage(r, dtype) for r in (ra, rb, P.to_type(np.zeros((m, n)), dtype)[0]))
    pc = c.raw_ptr()
    gpu.check(gpu.load().mjt_matmul_nearest(*[ctypes.byref(gpu.tensor(p, dtype, s)) for p, s in ((x.raw_ptr(), ra.shape), (y.raw_ptr(), rb.shape), (pc, (m, n)))], ta, tb))
    assert "_ragged" in gpu.last_kernel()
    got = gpu.d2h(pc, [m, n], ra.dtype)
    got = (bf16_bits_to_f32(got) if dtype == "bfloat16" else got).astype(np.float64)
    ae, be = ae.T if ta else ae, be.T if tb else be
    _check(got[:-1, :-1], ae[:-1] @ be[:, :-1], (k + 2) * E * (np.abs(ae[:-1]) @ np.abs(be[:, :-1])), dtype, (ta, tb))
    assert np.array_equal(got[-1, :-1], np.copysign(np.inf, be[-1, :-1])) and np.isnan(got[:, -1]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,k,f", [(2, 95, 40), (16, 1003, 24), (36, 46, 256), (24, 2231, 40), (90, 4099, 33), (600, 99, 500), (260, 515, 1030)])
def test_gated_rows_of_any_length(gpu, dtype, rows, k, f):
    _gated(dtype, rows, k, f, "silu", seed=rows + k)


# ---- in graphs --------------------------------------------------------------------------------------------------------------
def test_inputs_that_are_rebound_keep_their_value_in_what_was_built(gpu):
    rng = np.random.default_rng(20)
    (x, xe), (w, we), (s, se) = _make(rng, (2, 4, 4, 8), "float32"), _make(rng, (12, 8), "float32"), _make(rng, (8,), "float32", 0.1, 1.0)
    q, k, v = jt.nn.qkv_norm_rope(x, 2, 1, s, s)
    y = jt.nn.gated_linear(x, w)
    dw, ds = jt.grad(y.sum(), w), jt.grad(q.sum() + v.sum(), s)
    for u in (x, w, s):
        u.assign(u * 3.0)
    want, off = P.gated(xe.reshape(-1, 8), we, "silu")
    _check(_got(y).reshape(-1, 6), want, off, "float32", "y")
    (_, _), (dwe, dwo) = P.gated_grad(xe.reshape(-1, 8), we, "silu", np.ones((32, 6)), "float32")
    _check(_got(dw), dwe, dwo, "float32", "dw")
    part = xe.reshape(8, 4, 8)[:, :2]
    _check(_got(q).reshape(8, 2, 8), P.head_norm(part, se, None, None, 1e-6, False), 64 * E * np.abs(part) * 4, "float32", "q")
    _, dse, _, dss = P.head_norm_grad(part, se, None, None, 1e-6, False, np.ones(part.shape))
    _check(_got(ds), dse, 128 * E * dss, "float32", "ds")
    assert np.array_equal(_got(v).reshape(8, 1, 8), xe.reshape(8, 4, 8)[:, 3:])


def test_profiles_name_the_calls_and_change_nothing(gpu):
    rng = np.random.default_rng(21)
    (x, xe), (w, we) = _make(rng, (6, 8), "float32"), _make(rng, (12, 8), "float32")
    with jt.profile_scope() as rep:
        y = jt.nn.gated_linear(jt.nn.dropout(x, 0.5, True, seed=1), w)
        y.sync()
    keep = P.kept(48, 0.5, 1, 0).reshape(6, 8)
    want, off = P.gated(np.where(keep, 2 * xe, 0.0), we, "silu")
    _check(_got(y), want, off, "float32", "y")
    assert "gated_linear" in str(rep) and "dropout" in str(rep)


@pytest.mark.parametrize("replay", [True, False])
def test_results_of_a_call_one_after_the_other(gpu, replay):
    """q first, then k and v: each of them once, the ones that are there already left alone."""
    rng = np.random.default_rng(22)
    s = jt.array(np.ones(8, np.float32))
    with jt.flag_scope(enable_replay=replay):
        for _ in range(4):
            x, xe = _make(rng, (1, 4, 4, 8), "float32")
            q, k, v = jt.nn.qkv_norm_rope(x, 2, 1, s, s)
            q.sync()
            at = q._device_ptr()
            jt.sync([v, q, k])
            assert q._device_ptr() == at
            for o, rows in ((q, slice(0, 2)), (k, slice(2, 3))):
                _check(_got(o)[0], P.head_norm(xe[0][:, rows], np.ones(8), None, None, 1e-6, False), 64 * E * np.abs(xe[0][:, rows]) * 4, "float32", "q or k")
            assert np.array_equal(_got(v)[0], xe[0][:, 3:])


# ---- all of them in one model -----------------------------------------------------------------------------------------
def _example():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "decoder.py")
    spec = importlib.util.spec_from_file_location("decoder_example", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_example_learns_and_continues(gpu, dtype):
    ex = _example()
    model, losses, follows = ex.train(steps=60, dtype=dtype)
    assert losses[0] > 3.0 and losses[-1] < 0.3, (losses[0], losses[-1])
    out = model.generate(np.arange(4, dtype=np.int32)[:, None], 12)
    assert all(follows[a] == b for row in out for a, b in zip(row, row[1:]))


def test_the_example_token_by_token_is_the_example_at_once(gpu):
    ex = _example()
    model = ex.Decoder(seed=3)
    tokens = np.random.default_rng(0).integers(0, model.vocab, (3, 9))
    whole = _got(model.forward(tokens))
    cache = [None] * model.layers
    for i in range(9):
        step = _got(model.forward(tokens[:, i:i + 1], cache))
        # the same sums in other orders: relative to the logits' size, a few hundred roundings of 2^-24
        assert np.abs(step[:, 0] - whole[:, i]).max() < 512 * E * np.abs(whole).max(), i
