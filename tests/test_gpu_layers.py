"""Embedding and layer norm, with their gradients, on the GPU against plain implementations in 64
bits (80 for binary64 rows), at the sizes, strides and values where they can go wrong.

Tolerances. u is a rounding of the statistics' type (2^-24 binary32, 2^-53 binary64), U one of the
rows' type. A sum of n terms is off by at most u (n / 16 + 64) times the sum of their magnitudes: a
row is added up by 16 lanes or more, each taking every 16th vector at most (8 values of a vector one after
another), and at most 64 steps join the lanes, waves and workgroups; `_sum_u` is that factor. What
each test adds to it stands beside its bound. Outputs are rounded once more to their type.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "f64", "bf16", "f16"]
OUT_U = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 2.0 ** -149, "f64": 2.0 ** -1074, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}
WIDE = np.longdouble


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def _stored(pkg, x, dtype):
    """Values as an array of the type, and the values that it then holds."""
    x = np.asarray(x, dtype=np.float64)
    if dtype == "bf16":
        a = pkg.to_bfloat16(x.astype(np.float32))
        return a, pkg.from_bfloat16(a).astype(WIDE)
    a = x.astype({"f32": np.float32, "f64": np.float64, "f16": np.float16}[dtype])
    return a, a.astype(WIDE)


def _values(pkg, a):
    return (pkg.from_bfloat16(a) if a.dtype == pkg.bfloat16 else a).astype(WIDE)


def _bits(a):
    return np.ascontiguousarray(a).view({2: np.uint16, 4: np.uint32, 8: np.uint64}[a.dtype.itemsize])


def _u(dtype):
    return 2.0 ** -53 if dtype == "f64" else 2.0 ** -24


def _sum_u(dtype, n):
    return _u(dtype) * (n / 16 + 64)


def _near(got, want, bound, dtype, what=""):
    off = np.abs(got - want)
    limit = bound + OUT_U[dtype] * (np.abs(want) + bound) + LEAST[dtype]
    assert np.all(off <= limit), (what, float(np.max(off / limit)))


# ------------------------------------------------------------------------- embedding

EMBED_SHAPES = [(1, 1, 1), (0, 5, 8), (7, 3, 2), (64, 1000, 64), (65, 100, 33), (300, 257, 1000), (33, 50, 4099), (5, 9, 20000)]


def _scaled(pkg, table, scale, dtype):
    """scale * table, rounded once in the statistics' type and once to the table's."""
    if dtype == "f64":
        return table * np.float64(scale)
    wide = _values(pkg, table).astype(np.float32) * np.float32(scale)
    return pkg.to_bfloat16(wide) if dtype == "bf16" else wide.astype(table.dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,vocab,width", EMBED_SHAPES)
@pytest.mark.parametrize("scale", [1.0, 11.3137085])
def test_embedding_is_the_scaled_rows(ctx, pcu_pkg, count, vocab, width, scale, dtype):
    rng = np.random.default_rng(count + 3 * vocab + 7 * width)
    table, _ = _stored(pcu_pkg, rng.normal(0, 1, (vocab, width)), dtype)
    tokens = rng.integers(-1, vocab, count).astype(np.int32)
    if count:
        tokens[-1] = vocab - 1
    got = ctx.native_embedding(ctx.upload(table), ctx.upload(tokens), scale=scale).numpy()
    want = _bits(_scaled(pcu_pkg, table, scale, dtype))[np.maximum(tokens, 0)]
    want[tokens < 0] = 0
    np.testing.assert_array_equal(_bits(got).reshape(count, width), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_embedding_keeps_special_values(ctx, pcu_pkg, dtype):
    special = np.array([[np.inf, -np.inf, np.nan, 0.0, -0.0, 6e-8, -6e-8, 65504.0, 1.0]])
    table, _ = _stored(pcu_pkg, special, dtype)
    got = ctx.native_embedding(ctx.upload(table), ctx.upload(np.array([0, -1, 0], np.int32))).numpy()
    for r in (0, 2):
        nan = np.isnan(_values(pcu_pkg, table[0]).astype(np.float64))
        assert np.array_equal(np.isnan(_values(pcu_pkg, got[r]).astype(np.float64)), nan)
        np.testing.assert_array_equal(_bits(got[r])[~nan], _bits(table[0])[~nan])
    assert not np.any(_bits(got[1]))


def _strided(ctx, rows, cols, stride, lead, dtype, fill):
    """A device buffer of strided rows that begin `lead` elements into it; the whole and the pointer."""
    whole = np.full((lead + rows * stride,), fill).astype(dtype)
    dev = ctx.upload(whole)
    return dev, dev.ptr + lead * whole.dtype.itemsize


@pytest.mark.parametrize("dtype,code", [(np.float32, 0), (np.float64, 1), (np.float16, 3)])
@pytest.mark.parametrize("lead,width,stride", [(1, 37, 41), (3, 64, 65), (5, 1, 3), (0, 259, 300)])
def test_embedding_of_strided_rows(ctx, pcu_pkg, dtype, code, lead, width, stride):
    """Rows at every alignment of the type; what lies between the rows keeps its values."""
    from fusion_pcu_amd import _abi
    rng = np.random.default_rng(width)
    vocab, count = 19, 70
    host = np.zeros(lead + vocab * stride, dtype)
    host[:] = rng.normal(0, 1, host.shape)
    table = ctx.upload(host)
    view = host[lead:].reshape(vocab, stride)[:, :width]
    tokens = rng.integers(0, vocab, count).astype(np.int32)
    out, ptr = _strided(ctx, count, width, stride + 1, lead, dtype, 7)
    rows = _abi.Rows(table.ptr + lead * host.itemsize, code, 0, vocab, width, stride)
    f = _abi.Fault()
    assert ctx._lib.pcu_native_embedding(ctx.handle, ctypes.byref(rows), ctx.upload(tokens).ptr, count, 1.0, ptr,
                                         stride + 1, ctypes.byref(f)) == 0
    got = out.numpy()
    assert np.all(got[:lead] == 7)
    got = got[lead:].reshape(count, stride + 1)
    np.testing.assert_array_equal(got[:, :width], view[tokens])
    assert np.all(got[:, width:] == 7)
    # The gradient of the same rows, on a base and in its place.
    g = ctx.upload(np.ascontiguousarray(got))
    grad = _abi.Rows(g.ptr, code, 0, count, width, stride + 1)
    base = np.zeros_like(host)
    base[:] = rng.normal(0, 1, host.shape)
    change = ctx.upload(base)
    at = change.ptr + lead * host.itemsize
    assert ctx._lib.pcu_native_embedding_backward(ctx.handle, ctypes.byref(grad), ctx.upload(tokens).ptr, vocab, 0.5, at,
                                                  stride, at, stride, ctypes.byref(f)) == 0
    back = change.numpy()
    want = base.astype(np.float64)[lead:].reshape(vocab, stride).copy()
    size = np.abs(want[:, :width])
    np.add.at(want[:, :width], tokens, 0.5 * got[:, :width].astype(np.float64))
    np.add.at(size, tokens, 0.5 * np.abs(got[:, :width].astype(np.float64)))
    np.testing.assert_array_equal(back[:lead], base[:lead])
    back = back[lead:].reshape(vocab, stride)
    np.testing.assert_array_equal(back[:, width:], base[lead:].reshape(vocab, stride)[:, width:])
    name = {0: "f32", 1: "f64", 3: "f16"}[code]
    _near(back[:, :width].astype(np.float64), want[:, :width], (count + 4) * _u(name) * size, name)


BACK_SHAPES = [(1, 1, 1), (0, 9, 5), (5, 1, 8), (64, 1000, 64), (65, 1000, 63), (700, 3, 40), (511, 50257, 20),
               (4096, 100, 33), (4097, 100, 33), (5000, 40000, 17), (20000, 300000, 4), (9000, 65536, 9), (300, 70, 2500),
               (200, 4194304, 1), (1024, 17, 9), (1025, 17, 9), (1500, 100, 33), (2048, 50000, 12), (2049, 50000, 12),
               (1200, 4194304, 1)]


def _tokens(rng, count, vocab, how):
    if how == "one":
        return np.full(count, vocab // 2, np.int32)
    if how == "absent":
        return np.full(count, -1, np.int32)
    rank = np.exp(rng.random(count) * np.log(vocab + 1.0)).astype(np.int64) - 1
    t = np.minimum(rank * 7919 % vocab, vocab - 1).astype(np.int32)
    t[rng.random(count) < 0.1] = -1
    if count:
        t[-1] = vocab - 1
    return t


def _sum_in_order(pkg, g, tokens, vocab, base, scale, dtype):
    """The definition, each term added in its place, in the statistics' type."""
    stat = np.float64 if dtype == "f64" else np.float32
    acc = np.zeros((vocab, g.shape[1]), stat)
    with np.errstate(invalid="ignore"):
        np.add.at(acc, tokens[tokens >= 0], _values(pkg, g).astype(stat)[tokens >= 0])
        acc = acc * stat(scale)
        if base is not None:
            acc = _values(pkg, base).astype(stat) + acc
    return acc


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("count,vocab,width", BACK_SHAPES)
@pytest.mark.parametrize("how", ["text", "one", "absent"])
def test_embedding_backward_sums_each_tokens_rows(ctx, pcu_pkg, count, vocab, width, how, dtype):
    """Rows of at most 48 terms, and all rows of at most 1024 tokens, are added one after another: the
    same bits. Longer ones are off by at most one rounding a term (of a part, then of the parts), one for
    the scale and one for the base; the bound counts n + 4 of the magnitudes' sum."""
    rng = np.random.default_rng(count + vocab + width)
    tokens = _tokens(rng, count, vocab, how)
    g, gv = _stored(pcu_pkg, rng.normal(0, 1, (count, width)), dtype)
    scale = 1.75
    for base in (None, rng.normal(0, 1, (vocab, width)) if vocab * width < 1 << 21 else None):
        b, bv = _stored(pcu_pkg, base, dtype) if base is not None else (None, 0.0)
        dev_b = ctx.upload(b) if b is not None else None
        got = ctx.native_embedding_backward(ctx.upload(g), ctx.upload(tokens), vocab, scale=scale, base=dev_b).numpy()
        counts = np.bincount(tokens[tokens >= 0], minlength=vocab)
        want = _sum_in_order(pcu_pkg, g, tokens, vocab, b, scale, dtype)
        short = counts <= (1024 if count <= 1024 else 48)
        rounded, _ = _stored(pcu_pkg, want, dtype)
        np.testing.assert_array_equal(_bits(got)[short], _bits(rounded)[short])
        if not np.all(short):
            exact = np.zeros((vocab, width), WIDE)
            size = np.zeros((vocab, width), WIDE)
            np.add.at(exact, tokens[tokens >= 0], gv[tokens >= 0])
            np.add.at(size, tokens[tokens >= 0], np.abs(gv[tokens >= 0]))
            exact, size = exact * WIDE(scale) + bv, size * scale + np.abs(bv)
            bound = (counts[:, None] + 4) * _u(dtype) * size
            _near(_values(pcu_pkg, got)[~short], exact[~short], bound[~short], dtype)
        if base is not None:  # in the base's place
            ctx.native_embedding_backward(ctx.upload(g), ctx.upload(tokens), vocab, scale=scale, base=dev_b, out=dev_b)
            np.testing.assert_array_equal(_bits(dev_b.numpy()), _bits(got))


def test_embedding_backward_adds_in_the_terms_order(ctx):
    """Terms whose sum depends on the order: 2^24 and ones, the large one first, last and amid, in
    one part and in several."""
    for count in (40, 64, 65, 1000, 1500, 5000):
        for at in (0, count // 2, count - 1):
            g = np.ones((count, 3), np.float32)
            g[at] = 2.0 ** 24
            g[at - 1, 1] = -2.0 ** 24
            got = ctx.native_embedding_backward(ctx.upload(g), ctx.upload(np.zeros(count, np.int32)), 2).numpy()
            if count <= 1024:
                want = np.zeros(3, np.float32)
                for row in g:
                    want = want + row
                np.testing.assert_array_equal(got[0], want)
            else:
                exact = g.astype(np.float64).sum(0)
                assert np.all(np.abs(got[0] - exact) <= (count + 4) * 2.0 ** -24 * np.abs(g).astype(np.float64).sum(0))
            again = ctx.native_embedding_backward(ctx.upload(g), ctx.upload(np.zeros(count, np.int32)), 2).numpy()
            np.testing.assert_array_equal(got, again)
            assert not np.any(got[1])


@pytest.mark.parametrize("width", [3, 40, 300, 1100])
def test_embedding_backward_of_rows_at_the_parts_borders(ctx, pcu_pkg, width):
    """Rows of 46 to 51 terms (the longest of one wave has 48), of 95 to 98 and longer ones, at every
    offset to the parts of 48 terms that the others' numbers bring about; whole numbers, so any order
    gives the same sums."""
    rng = np.random.default_rng(width)
    lengths = [46, 47, 48, 49, 50, 51, 1, 2, 95, 96, 97, 98, 300, 1, 64, 16, 17, 15, 143, 144, 145, 3, 500, 48, 49, 48]
    for shift in range(0, 50, 7):
        order = rng.permutation(len(lengths))
        counts = np.array([shift] + [lengths[i] for i in order], np.int64)
        tokens = np.repeat(np.arange(len(counts)) * 2 + 1, counts).astype(np.int32)
        rng.shuffle(tokens)
        assert tokens.size > 1024
        g = rng.integers(-8, 9, (tokens.size, width)).astype(np.float32)
        vocab = 2 * len(counts) + 3
        want = np.zeros((vocab, width), np.float32)
        np.add.at(want, tokens, g)
        got = ctx.native_embedding_backward(ctx.upload(g), ctx.upload(tokens), vocab).numpy()
        np.testing.assert_array_equal(got, want)
        base = rng.integers(-8, 9, (vocab, width)).astype(np.float32)
        got = ctx.native_embedding_backward(ctx.upload(g), ctx.upload(tokens), vocab, base=ctx.upload(base)).numpy()
        np.testing.assert_array_equal(got, want + base)


def test_embedding_gradient_leaves_absent_rows_out(ctx):
    """NaN and infinities in rows of absent tokens reach nothing; in a row of a token, its row alone."""
    g = np.ones((6, 40), np.float32)
    g[1], g[4] = np.nan, np.inf
    tokens = np.array([2, -1, 0, 2, -5, 3], np.int32)
    got = ctx.native_embedding_backward(ctx.upload(g), ctx.upload(tokens), 5).numpy()
    want = np.zeros((5, 40), np.float32)
    want[[2, 0, 3]] = [[2], [1], [1]]
    np.testing.assert_array_equal(got, want)
    tokens[1] = 4
    got = ctx.native_embedding_backward(ctx.upload(g), ctx.upload(tokens), 5).numpy()
    assert np.all(np.isnan(got[4]))
    np.testing.assert_array_equal(got[:4], want[:4])


def test_tokens_out_of_range_are_faults(ctx, pcu_pkg):
    table = ctx.upload(np.ones((10, 8), np.float32))
    for count in (5, 200, 6000):
        tokens = np.zeros(count, np.int32)
        tokens[[3, count - 1]] = [10, 2 ** 31 - 1]
        for call in (lambda t: ctx.native_embedding(table, t),
                     lambda t: ctx.native_embedding_backward(ctx.upload(np.ones((count, 8), np.float32)), t, 10)):
            with pytest.raises(pcu_pkg.PcuExecutionError) as e:
                call(ctx.upload(tokens))
            assert e.value.tensor_fault.element_index == 3
            assert e.value.tensor_fault.kind == pcu_pkg.PcuExecutionFaultKind.InvalidFloatingOperand


def test_offsets_beyond_32_bits(ctx):
    """A table of 4.3 GB, whose last rows lie past 32-bit byte offsets."""
    rows, width = 1 << 22, 260
    table = ctx.empty((rows, width), np.float32)
    last = np.arange(width, dtype=np.float32)
    tokens = np.array([rows - 1, 3, rows - 1], np.int32)
    g = np.stack([last, 2 * last, 3 * last])
    ctx.native_embedding_backward(ctx.upload(g), ctx.upload(tokens), rows, out=table)
    got = ctx.native_embedding(table, ctx.upload(np.array([rows - 1, 3, 0, rows - 2, rows // 2], np.int32))).numpy()
    np.testing.assert_array_equal(got, np.stack([4 * last, 2 * last, 0 * last, 0 * last, 0 * last]))
    table.free()


# ------------------------------------------------------------------------- layer norm

NORM_SHAPES = [(1, 1), (0, 7), (3, 2), (64, 64), (65, 63), (17, 129), (70, 250), (5, 511), (130, 1000), (9, 1025), (4, 4097),
               (3, 8200), (2, 16391), (5, 33000), (2, 70001), (1000, 16), (2000, 5)]


def _norm_of(x, eps):
    m = np.mean(x, axis=1, keepdims=True)
    r = 1 / np.sqrt(np.mean((x - m) ** 2, axis=1, keepdims=True) + WIDE(eps))
    return m, r


def _forward_bounds(x, m, r, dtype):
    """Bounds of what the kernels' mean, 1 / deviation and normalised values are off by. The mean: its
    sum and the division. A difference: the mean's error and its own rounding. The mean square: twice
    the difference's error, its square, and the sum; half of that, relative, for its root's
    reciprocal, and three roundings."""
    n, u = x.shape[1], _u(dtype)
    d_mean = (_sum_u(dtype, n) + 2 * u) * np.mean(np.abs(x), axis=1, keepdims=True)
    d_diff = d_mean + u * (np.abs(x) + np.abs(m))
    square = np.mean((x - m) ** 2, axis=1, keepdims=True)
    d_square = np.mean(2 * np.abs(x - m) * d_diff + d_diff ** 2, axis=1, keepdims=True)
    d_square = d_square + (_sum_u(dtype, n) + 3 * u) * (square + d_square)
    d_r = r * (np.minimum(d_square * r ** 2, 1e9) / 2 * 1.1 + 4 * u)
    d_norm = d_diff * (r + d_r) + np.abs(x - m) * d_r + u * np.abs(x - m) * r
    return d_mean, d_r, d_norm


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", NORM_SHAPES)
@pytest.mark.parametrize("weights", ["own", "f32", "none", "weight", "bias"])
def test_layer_norm(ctx, pcu_pkg, rows, width, weights, dtype):
    if weights == "f32" and dtype in ("f32", "f64"):
        pytest.skip("16-bit rows alone take weights of another type")
    rng = np.random.default_rng(rows + 5 * width)
    a, x = _stored(pcu_pkg, rng.normal(0.5, 2, (rows, width)) * np.where(rng.random(width) < 0.02, 20, 1), dtype)
    wt = "f32" if weights == "f32" else dtype
    wa, w = _stored(pcu_pkg, rng.normal(1, 0.3, width), wt)
    ba, b = _stored(pcu_pkg, rng.normal(0, 0.3, width), wt)
    if weights in ("none", "bias"):
        wa, w = None, WIDE(1)
    if weights in ("none", "weight"):
        ba, b = None, WIDE(0)
    eps = 1e-5
    dev = ctx.upload(a)
    args = [ctx.upload(v) if v is not None else None for v in (wa, ba)]
    y, stats = ctx.native_layer_norm(dev, *args, eps=eps)
    if rows == 0:
        assert y.numpy().shape == (0, width)
        return
    eps_held = np.float64(eps) if dtype == "f64" else np.float32(eps)
    m, r = _norm_of(x, eps_held)
    d_mean, d_r, d_norm = _forward_bounds(x, m, r, dtype)
    got_s = stats.numpy().astype(WIDE)
    assert np.all(np.abs(got_s[:, :1] - m) <= d_mean) and np.all(np.abs(got_s[:, 1:] - r) <= d_r)
    want = (x - m) * r * w + b
    bound = d_norm * np.abs(w) + 3 * _u(dtype) * (np.abs((x - m) * r * w) + np.abs(b))
    got = _values(pcu_pkg, y.numpy())
    _near(got, want, bound, dtype)
    ctx.native_layer_norm(dev, *args, eps=eps, out=dev)  # in the rows' place
    np.testing.assert_array_equal(_bits(dev.numpy()), _bits(y.numpy()))


def test_layer_norm_of_hard_rows(ctx):
    """Equal values (the deviation is eps's alone), a large mean, infinities and NaN, which stay in their row."""
    width = 300
    rng = np.random.default_rng(1)
    x = rng.normal(0, 1, (70, width)).astype(np.float32)
    x[3], x[5] = 2.0, 0.0
    x[7] += 4096.0
    x[9, 17], x[11, 250] = np.nan, np.inf
    x[13] *= 1e18
    x[15] *= 1e-30
    y, stats = ctx.native_layer_norm(ctx.upload(x), eps=1e-5)
    y, stats = y.numpy(), stats.numpy()
    assert not np.any(y[[3, 5]]) and np.allclose(stats[[3, 5], 1], 1e-5 ** -0.5, rtol=1e-6)
    assert np.all(np.isnan(y[9])) and np.all(np.isnan(y[11]))
    fine = [r for r in range(70) if r not in (9, 11, 3, 5)]
    wide = x[fine].astype(WIDE)
    m, r = _norm_of(wide, np.float32(1e-5))
    _, _, d_norm = _forward_bounds(wide, m, r, "f32")
    _near(y[fine].astype(WIDE), (wide - m) * r, d_norm, "f32")
    zero, _ = ctx.native_layer_norm(ctx.upload(np.full((2, 9), 3.0, np.float32)), eps=0.0)
    assert np.all(np.isnan(zero.numpy()))  # 0 / 0, as the formula has it


def _norm_back(x, m, r, dy, w):
    near = (x - m) * r
    g = dy * w
    c0, c1 = np.mean(g, axis=1, keepdims=True), np.mean(g * near, axis=1, keepdims=True)
    return near, g, c0, c1, r * (g - c0 - near * c1), np.sum(dy * near, axis=0), np.sum(dy, axis=0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", NORM_SHAPES + [(3000, 100), (517, 700)])
@pytest.mark.parametrize("weights", ["own", "f32", "none"])
def test_layer_norm_backward(ctx, pcu_pkg, rows, width, weights, dtype):
    """A normalised value is off by 3 u of r (|x| + |m|); the means by their sums and one more
    rounding; dx by its parts' errors and 4 roundings. A weight's gradient is a sum over the rows."""
    if weights == "f32" and dtype in ("f32", "f64"):
        pytest.skip("16-bit rows alone take weights of another type")
    rng = np.random.default_rng(rows + 5 * width)
    a, x = _stored(pcu_pkg, rng.normal(0.5, 2, (rows, width)), dtype)
    da, dy = _stored(pcu_pkg, rng.normal(0, 1, (rows, width)), dtype)
    wt = "f32" if weights == "f32" else dtype
    wa, w = _stored(pcu_pkg, rng.normal(1, 0.3, width), wt)
    stat = np.float64 if dtype == "f64" else np.float32
    if rows:
        m, r = _norm_of(x, 1e-5)
        stats = np.concatenate([m, r], 1).astype(stat)
    else:
        stats = np.zeros((0, 2), stat)
    m, r = stats[:, :1].astype(WIDE), stats[:, 1:].astype(WIDE)
    dev = [ctx.upload(v) for v in (a, stats, da)]
    if weights == "none":
        w = WIDE(1)
        dx, none_w, none_b = ctx.native_layer_norm_backward(*dev)
        assert none_w is None and none_b is None
        dw = db = None
    else:
        dx, dw, db = ctx.native_layer_norm_backward(*dev, ctx.upload(wa))
    if rows == 0:
        if dw is not None:
            assert not np.any(_bits(dw.numpy())) and not np.any(_bits(db.numpy()))
        return
    u = _u(dtype)
    near, g, c0, c1, want, want_w, want_b = _norm_back(x, m, r, dy, w)
    d_near = 3 * u * r * (np.abs(x) + np.abs(m))
    d_c0 = (_sum_u(dtype, width) + 3 * u) * np.mean(np.abs(g), axis=1, keepdims=True)
    size = np.mean(np.abs(g) * (np.abs(near) + d_near), axis=1, keepdims=True)
    d_c1 = np.mean(np.abs(g) * d_near, axis=1, keepdims=True) + (_sum_u(dtype, width) + 4 * u) * size
    whole = np.abs(g) + np.abs(c0) + np.abs(near * c1)
    bound = r * (d_c0 + d_near * np.abs(c1) + (np.abs(near) + d_near) * d_c1 + 5 * u * whole)
    _near(_values(pcu_pkg, dx.numpy()), want, bound, dtype, "dx")
    if dw is not None:
        s = _sum_u(dtype, rows * 16) + 3 * u  # no fewer terms in a row of additions than the rows
        _near(_values(pcu_pkg, dw.numpy()), want_w, np.sum(np.abs(dy) * d_near, 0) + s * np.sum(np.abs(dy) * (np.abs(near) + d_near), 0), wt, "dw")
        _near(_values(pcu_pkg, db.numpy()), want_b, s * np.sum(np.abs(dy), 0), wt, "db")
        again = ctx.native_layer_norm_backward(*dev, ctx.upload(wa))
        for one, two in zip((dx, dw, db), again):
            np.testing.assert_array_equal(_bits(one.numpy()), _bits(two.numpy()))
    # In the upstream gradient's place, and in the rows'.
    kept = dx.numpy()
    for place in (2, 0):
        fresh = [ctx.upload(v) for v in (a, stats, da)]
        ctx.native_layer_norm_backward(*fresh, ctx.upload(wa) if weights != "none" else None, x_gradient=fresh[place])
        np.testing.assert_array_equal(_bits(fresh[place].numpy()), _bits(kept))


@pytest.mark.parametrize("rows,width", [(4, 33), (3, 300), (2, 9000)])
def test_layer_norm_gradient_is_the_differences(ctx, rows, width):
    """Central differences of L = sum(dy * y) along random directions in binary64. With steps of
    h = 2^-17 the differences' own error is about h^2 times a third derivative (of order 1 here)
    and 2^-53 |L| / h: 1e-8 of the sum of magnitudes covers both."""
    rng = np.random.default_rng(width)
    x, dy = rng.normal(0, 1, (rows, width)), rng.normal(0, 1, (rows, width))
    w, b = rng.normal(1, 0.3, width), rng.normal(0, 0.3, width)

    def loss(x, w, b):
        y, _ = ctx.native_layer_norm(ctx.upload(x), ctx.upload(w), ctx.upload(b), eps=1e-5)
        return float(np.sum(dy * y.numpy()))

    _, stats = ctx.native_layer_norm(ctx.upload(x), ctx.upload(w), ctx.upload(b), eps=1e-5)
    grads = ctx.native_layer_norm_backward(ctx.upload(x), stats, ctx.upload(dy), ctx.upload(w))
    h = 2.0 ** -17
    for k, grad in enumerate(grads):
        grad = grad.numpy()
        d = rng.normal(0, 1, grad.shape)
        args = [x, w, b]
        up, down = list(args), list(args)
        up[k], down[k] = args[k] + h * d, args[k] - h * d
        slope = (loss(*up) - loss(*down)) / (2 * h)
        assert abs(slope - np.sum(grad * d)) <= 1e-8 * (np.sum(np.abs(grad * d)) + np.sum(np.abs(dy)))


@pytest.mark.parametrize("dtype,code", [(np.float32, 0), (np.float64, 1), (np.float16, 3)])
@pytest.mark.parametrize("lead,width,stride", [(1, 37, 41), (3, 511, 515), (0, 2001, 2003), (1, 9001, 9004)])
def test_layer_norm_of_strided_rows(ctx, pcu_pkg, dtype, code, lead, width, stride):
    """Rows at every alignment give the bits of dense ones; what lies between them keeps its values."""
    from fusion_pcu_amd import _abi
    rng = np.random.default_rng(width)
    rows = 21
    x, dy = (rng.normal(0, 1, (rows, width)).astype(dtype) for _ in range(2))
    y, stats = ctx.native_layer_norm(ctx.upload(x))
    dx, dw, db = ctx.native_layer_norm_backward(ctx.upload(x), stats, ctx.upload(dy),
                                                weight_gradient=ctx.empty((width,), dtype), bias_gradient=ctx.empty((width,), dtype))

    def spread(v):
        host = np.full(lead + rows * stride, 9, dtype)
        host[lead:].reshape(rows, stride)[:, :width] = v
        dev = ctx.upload(host)
        return dev, dev.ptr + lead * host.itemsize

    (xd, xp), (gd, gp), (od, op) = spread(x), spread(dy), spread(np.zeros_like(x))
    st = ctx.empty(stats.shape, stats.dtype)
    r = _abi.Rows(xp, code, 0, rows, width, stride)
    assert ctx._lib.pcu_native_layer_norm(ctx.handle, ctypes.byref(r), None, None, code, 1e-5, op, stride, st.ptr) == 0

    def check(dev, want):
        host = dev.numpy()
        assert np.all(host[:lead] == 9)
        host = host[lead:].reshape(rows, stride)
        assert np.all(host[:, width:] == 9)
        np.testing.assert_array_equal(host[:, :width], want)

    check(od, y.numpy())
    np.testing.assert_array_equal(st.numpy(), stats.numpy())
    wd, bd = ctx.empty((width,), dtype), ctx.empty((width,), dtype)
    assert ctx._lib.pcu_native_layer_norm_backward(ctx.handle, ctypes.byref(r), st.ptr, gp, stride, None, code, op, stride,
                                                   wd.ptr, bd.ptr) == 0
    check(od, dx.numpy())
    np.testing.assert_array_equal(wd.numpy(), dw.numpy())
    np.testing.assert_array_equal(bd.numpy(), db.numpy())


# --------------------------------------------------------------------- refusals

def test_refusals(ctx, pcu_pkg):
    from fusion_pcu_amd import _abi
    E = pcu_pkg.PcuExecutionError
    f32 = lambda *s: ctx.empty(s, np.float32)
    i32 = lambda *s: ctx.empty(s, np.int32)
    table, x = f32(10, 8), f32(4, 8)
    for call in (lambda: ctx.native_embedding(table, f32(4)), lambda: ctx.native_embedding(f32(10), i32(4)),
                 lambda: ctx.native_embedding(table, i32(4), out=f32(4, 7)), lambda: ctx.native_embedding(table, i32(4, 1)),
                 lambda: ctx.native_embedding(table, i32(4), scale=np.inf), lambda: ctx.native_embedding(table, i32(4), scale=1e60),
                 lambda: ctx.native_embedding(ctx.empty((10, 8), np.int32), i32(4)),
                 lambda: ctx.native_embedding_backward(x, i32(5), 10), lambda: ctx.native_embedding_backward(x, i32(4), -1),
                 lambda: ctx.native_embedding_backward(x, i32(4), (1 << 22) + 1), lambda: ctx.native_embedding_backward(x, i32(4), 4, out=x),
                 lambda: ctx.native_embedding_backward(x, i32(4), 10, base=f32(9, 8)),
                 lambda: ctx.native_layer_norm(x, weight=f32(7)), lambda: ctx.native_layer_norm(x, eps=-1.0),
                 lambda: ctx.native_layer_norm(x, eps=np.nan), lambda: ctx.native_layer_norm(x, weight=ctx.empty((8,), np.float64)),
                 lambda: ctx.native_layer_norm(x, weight=f32(8), bias=ctx.empty((8,), np.float16)),
                 lambda: ctx.native_layer_norm(x, stats=f32(4, 3)),
                 lambda: ctx.native_layer_norm_backward(x, f32(4, 1), x), lambda: ctx.native_layer_norm_backward(x, f32(4, 2), f32(4, 9))):
        with pytest.raises(E):
            call()
    # Through the C ABI: alignment, overlaps, strides, nulls.
    lib, h, rows = ctx._lib, ctx.handle, lambda p, s=8, d=0, r=4, c=8: ctypes.byref(_abi.Rows(p, d, 0, r, c, s))
    big, t = f32(64, 64), i32(64)
    f = ctypes.byref(_abi.Fault())
    A, S = _abi.PCU_ERR_ARGUMENT, _abi.PCU_ERR_SHAPE
    assert lib.pcu_native_embedding(h, rows(big.ptr + 2), t.ptr, 4, 1.0, x.ptr, 8, f) == A
    assert lib.pcu_native_embedding(h, rows(big.ptr), t.ptr + 1, 4, 1.0, x.ptr, 8, f) == A
    assert lib.pcu_native_embedding(h, rows(big.ptr), t.ptr, 4, 1.0, big.ptr + 64, 8, f) == A
    assert lib.pcu_native_embedding(h, rows(big.ptr), None, 4, 1.0, x.ptr, 8, f) == A
    assert lib.pcu_native_embedding(h, rows(None), t.ptr, 4, 1.0, x.ptr, 8, f) == A
    assert lib.pcu_native_embedding(h, rows(big.ptr, d=4), t.ptr, 4, 1.0, x.ptr, 8, f) == A
    assert lib.pcu_native_embedding(h, None, t.ptr, 4, 1.0, x.ptr, 8, f) == A
    assert lib.pcu_native_embedding(h, rows(big.ptr, s=7), t.ptr, 4, 1.0, x.ptr, 8, f) == S
    assert lib.pcu_native_embedding(h, rows(big.ptr), t.ptr, 4, 1.0, x.ptr, 7, f) == S
    assert lib.pcu_native_embedding(h, rows(big.ptr, s=1 << 31, r=1), t.ptr, 4, 1.0, x.ptr, 8, f) == S
    assert lib.pcu_native_embedding(h, rows(big.ptr, r=(1 << 22) + 1), t.ptr, 4, 1.0, x.ptr, 8, f) == S
    assert lib.pcu_native_embedding_backward(h, rows(big.ptr), t.ptr, 4, 1.0, x.ptr, 9, x.ptr, 8, f) == A
    assert lib.pcu_native_embedding_backward(h, rows(big.ptr), t.ptr, 4, 1.0, big.ptr + 4096, 8, big.ptr + 4100, 8, f) == A
    assert lib.pcu_native_embedding_backward(h, rows(big.ptr), t.ptr, 4, 1.0, None, 0, None, 8, f) == A
    assert lib.pcu_native_embedding_backward(h, rows(big.ptr, r=1 << 29), t.ptr, 4, 1.0, None, 0, x.ptr, 8, f) == S
    assert lib.pcu_native_embedding_backward(h, rows(big.ptr, r=1 << 20, c=1 << 18, s=1 << 18), t.ptr, 4, 1.0, None, 0, x.ptr, 1 << 18, f) == S
    assert lib.pcu_native_layer_norm(h, rows(big.ptr), None, None, 1, 1e-5, x.ptr, 8, None) == A
    assert lib.pcu_native_layer_norm(h, rows(big.ptr), None, None, 0, 1e-5, big.ptr + 4, 8, None) == A
    assert lib.pcu_native_layer_norm(h, rows(big.ptr), x.ptr, None, 0, 1e-5, big.ptr, 8, x.ptr) == A
    assert lib.pcu_native_layer_norm(h, rows(big.ptr), None, None, 0, 1e-5, None, 8, None) == A
    assert lib.pcu_native_layer_norm_backward(h, rows(big.ptr), None, x.ptr, 8, None, 0, x.ptr, 8, None, None) == A
    assert lib.pcu_native_layer_norm_backward(h, rows(big.ptr), t.ptr, x.ptr, 8, None, 0, x.ptr + 4, 8, None, None) == A
    assert lib.pcu_native_layer_norm_backward(h, rows(big.ptr), t.ptr, x.ptr, 8, None, 0, None, 8, x.ptr, None) == A
    # Nothing is in flight after a refusal, and the context works on.
    y, _ = ctx.native_layer_norm(ctx.upload(np.ones((4, 8), np.float32)))
    assert not np.any(y.numpy())
