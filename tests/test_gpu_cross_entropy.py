"""The cross entropy of an output layer whose logits are not kept, and its gradients, on the GPU against
the definition in 64 bits.

Tolerances. u = 2^-24. Products of 16-bit values are exact in binary32; binary32 operands enter as 3
parts whose 6 largest products are kept, which leaves out 3 products of at most 2^-24 of the whole. A
sum of n products is rounded at most once for every 4 of them on the way of any term, by 2 u at most (the
matrix cores' adds), and at most 32 more times where parts of it are joined: with A the sum of the
magnitudes and `pairs` 6 or 1, E(n, A) = u (pairs n / 2 + 64 + 3) A. A logit is off by e = E(width, sum
|x w|). An exponential of l - m carries 4 u |l - m| + 2 u, and a sum over the vocabulary at most
(vocab / 16 + 128) u more, so a log-sum-exp is off by L = e + u (16 B + vocab / 16 + 128), B the
largest |l|; the loss by L + e. A probability's relative error is then P = e + L + u (8 B + 8).
G = p - [label] is rounded to the operands' type, a relative error of U, or in binary16, where it is held
2^14 times as large, of 2^-39 of the largest scale if that is more; its scale carries 2 roundings. The
gradients' sums add E over the vocabulary or the rows, and are rounded to their type.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "bf16", "f16"]
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}  # parts of a binary32 below 2^-126 are dropped
u = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def _stored(pkg, x, dtype):
    x = np.asarray(x, dtype=np.float64)
    if dtype == "bf16":
        a = pkg.to_bfloat16(x.astype(np.float32))
        return a, pkg.from_bfloat16(a).astype(np.float64)
    a = x.astype({"f32": np.float32, "f16": np.float16}[dtype])
    return a, a.astype(np.float64)


def _values(pkg, a):
    return (pkg.from_bfloat16(a) if a.dtype == pkg.bfloat16 else a).astype(np.float64)


def _bits(a):
    return np.ascontiguousarray(a).view({2: np.uint16, 4: np.uint32}[a.dtype.itemsize])


def _sum_error(dtype, n, magnitude):
    return u * ((6 if dtype == "f32" else 1) * n / 2 + 67) * magnitude


class Exact:
    """The definition, and the bounds of the module's docstring."""

    def __init__(self, x, w, labels, dtype, scale=None):
        rows, vocab = x.shape[0], w.shape[0]
        has = labels >= 0
        y = np.maximum(labels, 0)
        x = np.where(has[:, None] | np.all(np.isfinite(x), axis=1, keepdims=True), x, 0.0)
        l = x @ w.T
        e = _sum_error(dtype, x.shape[1], np.abs(x) @ np.abs(w).T)
        m = l.max(axis=1, keepdims=True)
        self.log_sum = (m + np.log(np.exp(l - m).sum(axis=1, keepdims=True)))[:, 0]
        self.d_log_sum = e.max(axis=1) + u * (16 * np.abs(l).max(axis=1) + vocab / 16 + 128)
        at = np.arange(rows)
        self.loss = np.where(has, self.log_sum - l[at, y], 0.0)
        self.d_loss = np.where(has, self.d_log_sum + e[at, y] + u * np.abs(self.loss), 0.0)
        s = np.where(has, np.ones(rows) if scale is None else scale.astype(np.float64), 0.0)[:, None]
        p = np.exp(l - self.log_sum[:, None])
        g = p.copy()
        g[at, y] -= 1.0
        rel = e + self.d_log_sum[:, None] + u * (8 * np.abs(l) + 8)
        d = p * np.expm1(rel)
        least = np.abs(s).max(initial=0.0) * (2.0 ** -39 if dtype == "f16" else 0.0)
        d = np.abs(s) * (d + (U[dtype] + 2 * u) * (np.abs(g) + d)) + least
        d = np.where(has[:, None], d, 0.0)
        g = s * g
        size = np.abs(g) + d
        self.dx, self.dw = g @ w, g.T @ x
        self.d_dx = d @ np.abs(w) + _sum_error(dtype, vocab, size @ np.abs(w))
        self.d_dw = d.T @ np.abs(x) + _sum_error(dtype, rows, size.T @ np.abs(x))


def _near(got, want, bound, dtype, what):
    off, limit = np.abs(got - want), bound + U[dtype] * (np.abs(want) + bound) + LEAST[dtype]
    assert np.all(off <= limit), (what, float(np.max(off / limit)))


def _inputs(pkg, rng, rows, vocab, width, dtype, sharp=2.0):
    w = rng.normal(0, sharp / np.sqrt(width), (vocab, width))
    labels = rng.integers(-1, vocab, rows).astype(np.int32)
    x = rng.normal(0, 1, (rows, width)) + 2 * rng.random((rows, 1)) * w[np.maximum(labels, 0)]
    if rows:
        labels[-1] = vocab - 1
    (xa, xv), (wa, wv) = _stored(pkg, x, dtype), _stored(pkg, w, dtype)
    return xa, xv, wa, wv, labels


# Every tile: few rows (32 across), 128 x 128, and 256 x 256 in each product; odd sizes of all three.
SHAPES = [(1, 1, 1), (1, 1000, 64), (5, 7, 3), (31, 255, 63), (32, 257, 128), (33, 256, 64), (64, 1000, 64), (65, 129, 65),
          (130, 2049, 200), (300, 50000, 64), (1, 40000, 72), (257, 300, 1000), (20, 3000, 320), (2, 12289, 1024)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_loss_and_gradients(ctx, pcu_pkg, rows, vocab, width, dtype):
    rng = np.random.default_rng(rows + 3 * vocab + 7 * width)
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, rows, vocab, width, dtype)
    scale = np.full(rows, 1.0 / rows, np.float32)
    want = Exact(xv, wv, labels, dtype, scale)
    x, w, y, s = (ctx.upload(a) for a in (xa, wa, labels, scale))
    loss, log_sum = ctx.native_cross_entropy_loss(x, w, y)
    assert np.all(np.abs(log_sum.numpy() - want.log_sum) <= want.d_log_sum)
    assert np.all(np.abs(loss.numpy() - want.loss) <= want.d_loss)
    dx, dw = ctx.native_cross_entropy_backward(x, w, y, log_sum, row_scale=s)
    _near(_values(pcu_pkg, dx.numpy()), want.dx, want.d_dx, dtype, "dx")
    _near(_values(pcu_pkg, dw.numpy()), want.dw, want.d_dw, dtype, "dw")
    # One call gives the same bits, and so does another.
    for _ in range(2):
        loss2, dx2, dw2 = ctx.native_cross_entropy_step(x, w, y, row_scale=s)
        for one, two in ((loss, loss2), (dx, dx2), (dw, dw2)):
            np.testing.assert_array_equal(_bits(one.numpy()), _bits(two.numpy()))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", [(3200, 300, 4096), (70, 12300, 1100)])
def test_large_tiles_of_the_gradients(ctx, pcu_pkg, rows, vocab, width, dtype):
    rng = np.random.default_rng(rows)
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, rows, vocab, width, dtype)
    want = Exact(xv, wv, labels, dtype)
    loss, dx, dw = ctx.native_cross_entropy_step(ctx.upload(xa), ctx.upload(wa), ctx.upload(labels))
    assert np.all(np.abs(loss.numpy() - want.loss) <= want.d_loss)
    _near(_values(pcu_pkg, dx.numpy()), want.dx, want.d_dx, dtype, "dx")
    _near(_values(pcu_pkg, dw.numpy()), want.dw, want.d_dw, dtype, "dw")


@pytest.mark.parametrize("dtype", DTYPES)
def test_several_pieces_of_the_vocabulary(ctx, pcu_pkg, dtype):
    """So many rows that a piece of the vocabulary is a few hundred tokens."""
    rng = np.random.default_rng(3)
    rows, vocab, width = 100001, 801, 16
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, rows, vocab, width, dtype)
    want = Exact(xv, wv, labels, dtype)
    loss, dx, dw = ctx.native_cross_entropy_step(ctx.upload(xa), ctx.upload(wa), ctx.upload(labels))
    assert np.all(np.abs(loss.numpy() - want.loss) <= want.d_loss)
    _near(_values(pcu_pkg, dx.numpy()), want.dx, want.d_dx, dtype, "dx")
    _near(_values(pcu_pkg, dw.numpy()), want.dw, want.d_dw, dtype, "dw")


def test_weights_too_many_to_keep_packed(ctx, pcu_pkg):
    """Binary32 weights whose parts would take more than 512 MiB, for few rows and in two pieces of the vocabulary."""
    rng = np.random.default_rng(4)
    rows, vocab, width = 9, 262144, 384
    w = rng.standard_normal((vocab, width), np.float32) * np.float32(0.1)
    x = rng.standard_normal((rows, width), np.float32)
    labels = rng.integers(0, vocab, rows).astype(np.int32)
    labels[0] = -1
    want = Exact(x.astype(np.float64), w.astype(np.float64), labels, "f32")
    loss, dx, dw = ctx.native_cross_entropy_step(ctx.upload(x), ctx.upload(w), ctx.upload(labels))
    assert np.all(np.abs(loss.numpy() - want.loss) <= want.d_loss)
    _near(dx.numpy().astype(np.float64), want.dx, want.d_dx, "f32", "dx")
    _near(dw.numpy().astype(np.float64), want.dw, want.d_dw, "f32", "dw")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows", [7, 40, 200])
def test_rows_without_a_label_reach_nothing(ctx, pcu_pkg, rows, dtype):
    """Whatever their features hold; and all rows without one."""
    rng = np.random.default_rng(rows)
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, rows, 500, 96, dtype)
    labels[::3] = -7
    bad = xv.copy()
    bad[::3] = np.array([np.nan, np.inf, -np.inf, 1e4])[np.arange(96) % 4]
    ba, bv = _stored(pcu_pkg, bad, dtype)
    want = Exact(bv, wv, labels, dtype)
    w, y = ctx.upload(wa), ctx.upload(labels)
    first = ctx.native_cross_entropy_step(ctx.upload(xa), w, y)
    second = ctx.native_cross_entropy_step(ctx.upload(ba), w, y)
    for one, two in zip(first, second):
        np.testing.assert_array_equal(_bits(one.numpy()), _bits(two.numpy()))
    _near(_values(pcu_pkg, second[1].numpy()), want.dx, want.d_dx, dtype, "dx")
    _near(_values(pcu_pkg, second[2].numpy()), want.dw, want.d_dw, dtype, "dw")
    assert not np.any(second[0].numpy()[::3]) and not np.any(_values(pcu_pkg, second[1].numpy())[::3])
    loss, log_sum = ctx.native_cross_entropy_loss(ctx.upload(ba), w, y)
    np.testing.assert_array_equal(loss.numpy(), first[0].numpy())
    dx, dw = ctx.native_cross_entropy_backward(ctx.upload(ba), w, y, log_sum)
    np.testing.assert_array_equal(_bits(dx.numpy()), _bits(first[1].numpy()))
    np.testing.assert_array_equal(_bits(dw.numpy()), _bits(first[2].numpy()))
    none = ctx.upload(np.full(rows, -1, np.int32))
    for a in ctx.native_cross_entropy_step(ctx.upload(ba), w, none):
        assert not np.any(_values(pcu_pkg, a.numpy()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_padded_vocabulary(ctx, pcu_pkg, dtype):
    """Rows of weights past the vocabulary are not read, and their gradient is 0."""
    rng = np.random.default_rng(8)
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, 70, 331, 64, dtype)
    padded = np.concatenate([wv, np.full((5, 64), np.nan)])
    pa, _ = _stored(pcu_pkg, padded, dtype)
    x, y = ctx.upload(xa), ctx.upload(labels)
    whole = ctx.native_cross_entropy_step(x, ctx.upload(wa), y)
    part = ctx.native_cross_entropy_step(x, ctx.upload(pa), y, vocab=331)
    np.testing.assert_array_equal(whole[0].numpy(), part[0].numpy())
    np.testing.assert_array_equal(_bits(whole[1].numpy()), _bits(part[1].numpy()))
    np.testing.assert_array_equal(_bits(whole[2].numpy()), _bits(part[2].numpy())[:331])
    assert not np.any(_bits(part[2].numpy())[331:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kind", ["mixed", "zeros", "large", "small", "negative"])
def test_row_scales(ctx, pcu_pkg, kind, dtype):
    rng = np.random.default_rng(9)
    rows = 90
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, rows, 400, 64, dtype)
    scale = {"mixed": rng.choice([0.0, 1e-3, 0.5, 1.0], rows), "zeros": np.zeros(rows), "large": rng.random(rows) * 100,
             "small": rng.random(rows) * 1e-3, "negative": rng.normal(0, 1, rows)}[kind].astype(np.float32)
    want = Exact(xv, wv, labels, dtype, scale)
    _, dx, dw = ctx.native_cross_entropy_step(ctx.upload(xa), ctx.upload(wa), ctx.upload(labels), row_scale=ctx.upload(scale))
    _near(_values(pcu_pkg, dx.numpy()), want.dx, want.d_dx, dtype, "dx")
    _near(_values(pcu_pkg, dw.numpy()), want.dw, want.d_dw, dtype, "dw")


def test_special_scales_stay_in_their_rows(ctx):
    """An infinite or NaN scale spoils its row's gradient, and not another row's."""
    rng = np.random.default_rng(10)
    x, w = rng.normal(0, 1, (40, 64)).astype(np.float32), rng.normal(0, 0.2, (300, 64)).astype(np.float32)
    labels = rng.integers(0, 300, 40).astype(np.int32)
    scale = rng.random(40).astype(np.float32)
    args = [ctx.upload(a) for a in (x, w, labels)]
    _, plain, _ = ctx.native_cross_entropy_step(*args, row_scale=ctx.upload(scale))
    scale[3], scale[5] = np.inf, np.nan
    _, dx, dw = ctx.native_cross_entropy_step(*args, row_scale=ctx.upload(scale))
    dx, keep = dx.numpy(), np.setdiff1d(np.arange(40), [3, 5])
    assert not np.any(np.isfinite(dx[[3, 5]])) and np.all(np.isnan(dw.numpy()))
    # The scales' common factor may be another one: two roundings more, of G's sums' magnitudes.
    want = Exact(x.astype(np.float64), w.astype(np.float64), labels, "f32", np.where(np.isfinite(scale), scale, 0).astype(np.float32))
    _near(dx[keep].astype(np.float64), want.dx[keep], want.d_dx[keep], "f32", "dx")


def test_special_logits(ctx):
    """Logits that overflow, all equal ones, and NaN: as the definition has them, row by row."""
    w = np.zeros((300, 64), np.float32)
    w[:, 0] = np.linspace(-1, 1, 300)
    w[7, 1] = 1.0
    x = np.zeros((5, 64), np.float32)
    x[1, 0] = 3e4
    x[2, 0] = -50.0
    x[3, 0] = np.nan
    x[4, 1] = np.inf
    labels = np.array([0, 299, 299, 1, 7], np.int32)
    loss, log_sum = ctx.native_cross_entropy_loss(*(ctx.upload(a) for a in (x, w, labels)))
    got_l, got = log_sum.numpy().astype(np.float64), loss.numpy().astype(np.float64)
    want = Exact(x[:3].astype(np.float64), w.astype(np.float64), labels[:3], "f32")
    assert np.all(np.abs(got_l[:3] - want.log_sum) <= want.d_log_sum) and np.all(np.abs(got[:3] - want.loss) <= want.d_loss)
    assert np.all(np.isnan(got[3:]))
    # Row 2's logits fall from 50 to -50 in steps of 100 / 299: log_sum = 50 + log(sum of e^(-100 i / 299)),
    # and that sum is 1 / (1 - e^(-100 / 299)) = 3.52 less e^-100.
    assert abs(got[0] - np.log(300.0)) < 1e-5 and got[1] < 1e-3
    assert abs(got[2] - 100 + np.log1p(-np.exp(-100 / 299))) < 1e-3


def test_gradient_is_the_differences(ctx):
    """Central differences of sum(s loss) along random directions. The loss's bound E gives 2 E / (2 h);
    a third derivative of a row's log-sum-exp is at most the cube of its logits' range of slopes."""
    rng = np.random.default_rng(11)
    rows, vocab, width, h = 20, 150, 24, 2.0 ** -6
    x, w = rng.normal(0, 1, (rows, width)), rng.normal(0, 0.3, (vocab, width))
    labels = rng.integers(0, vocab, rows).astype(np.int32)
    s = rng.random(rows).astype(np.float32)
    y = ctx.upload(labels)

    def loss(x, w):
        """At the points that binary32 holds, and its bound."""
        a, b = x.astype(np.float32), w.astype(np.float32)
        got, _ = ctx.native_cross_entropy_loss(ctx.upload(a), ctx.upload(b), y)
        return float(s.astype(np.float64) @ got.numpy()), Exact(a.astype(np.float64), b.astype(np.float64), labels, "f32")

    x, w = x.astype(np.float32).astype(np.float64), w.astype(np.float32).astype(np.float64)
    _, dx, dw = ctx.native_cross_entropy_step(ctx.upload(x.astype(np.float32)), ctx.upload(w.astype(np.float32)), y, row_scale=ctx.upload(s))
    for k, grad in enumerate((dx, dw)):
        d = np.sign(rng.normal(0, 1, grad.shape)) * 2.0 ** -3
        # Steps of 2^-9 keep the points within a few of binary32's last bits of the exact ones.
        up, down = [x, w], [x, w]
        up[k], down[k] = up[k] + h * d, down[k] - h * d
        (one, e1), (two, e2) = loss(*up), loss(*down)
        slopes = d @ w.T if k == 0 else x @ d.T
        third = float(s @ (slopes.max(1) - slopes.min(1)) ** 3)
        moved = 2.0 ** -24 * 4 * float(np.abs(grad.numpy()).sum())  # the points' rounding
        bound = (float(s @ e1.d_loss) + float(s @ e2.d_loss) + moved) / (2 * h) + third * h * h / 6
        slope = (one - two) / (2 * h)
        assert abs(slope - float(np.sum(grad.numpy().astype(np.float64) * d))) <= bound
        assert bound < 0.2 * abs(slope) + 0.05


@pytest.mark.parametrize("dtype,code", [("f32", 0), ("f16", 3), ("bf16", 2)])
@pytest.mark.parametrize("lead,more", [(0, 8), (1, 0), (3, 5), (8, 64)])
@pytest.mark.parametrize("width", [64, 100])
def test_strided_rows(ctx, pcu_pkg, dtype, code, lead, more, width):
    """Rows at every stride and alignment give the bits of dense ones; what lies between keeps its values."""
    from fusion_pcu_amd import _abi
    rng = np.random.default_rng(width + more)
    rows, vocab = 50, 700
    xa, _, wa, _, labels = _inputs(pcu_pkg, rng, rows, vocab, width, dtype)
    y = ctx.upload(labels)
    want = [a.numpy() for a in ctx.native_cross_entropy_step(ctx.upload(xa), ctx.upload(wa), y)]
    stride = width + more

    def spread(v):
        host = np.zeros(lead + v.shape[0] * stride, v.dtype)
        _bits(host)[:] = 0x3C00
        host[lead:].reshape(v.shape[0], stride)[:, :width] = v
        dev = ctx.upload(host)
        return dev, dev.ptr + lead * host.itemsize

    (xd, xp), (wd, wp), (dxd, dxp), (dwd, dwp) = (spread(v) for v in (xa, wa, np.zeros_like(xa), np.zeros_like(wa)))
    loss = ctx.empty((rows,), np.float32)
    xr, wr = _abi.Rows(xp, code, 0, rows, width, stride), _abi.Rows(wp, code, 0, vocab, width, stride)
    assert ctx._lib.pcu_native_cross_entropy_step(ctx.handle, ctypes.byref(xr), ctypes.byref(wr), y.ptr, None, loss.ptr, dxp, stride,
                                                  dwp, vocab, stride, None) == 0
    np.testing.assert_array_equal(loss.numpy(), want[0])
    for dev, v in ((dxd, want[1]), (dwd, want[2])):
        host = _bits(dev.numpy())
        assert not np.any(host[:lead] != 0x3C00)
        host = host[lead:].reshape(v.shape[0], stride)
        np.testing.assert_array_equal(host[:, :width], _bits(v))
        assert np.all(host[:, width:] == 0x3C00)
    # Either gradient alone.
    log_sum = ctx.empty((rows,), np.float32)
    assert ctx._lib.pcu_native_cross_entropy_loss(ctx.handle, ctypes.byref(xr), ctypes.byref(wr), y.ptr, loss.ptr, log_sum.ptr, None) == 0
    a, b = ctx.empty(want[1].shape, want[1].dtype), ctx.empty(want[2].shape, want[2].dtype)
    assert ctx._lib.pcu_native_cross_entropy_backward(ctx.handle, ctypes.byref(xr), ctypes.byref(wr), y.ptr, log_sum.ptr, None, a.ptr,
                                                      width, None, 0, 0, None) == 0
    assert ctx._lib.pcu_native_cross_entropy_backward(ctx.handle, ctypes.byref(xr), ctypes.byref(wr), y.ptr, log_sum.ptr, None, None,
                                                      0, b.ptr, vocab, width, None) == 0
    np.testing.assert_array_equal(_bits(a.numpy()), _bits(want[1]))
    np.testing.assert_array_equal(_bits(b.numpy()), _bits(want[2]))


def test_no_rows_and_no_vocabulary(ctx):
    w = ctx.upload(np.ones((30, 8), np.float32))
    loss, dx, dw = ctx.native_cross_entropy_step(ctx.empty((0, 8), np.float32), w, ctx.empty((0,), np.int32))
    assert loss.numpy().shape == (0,) and not np.any(dw.numpy())
    x, y = ctx.upload(np.ones((3, 8), np.float32)), ctx.upload(np.full(3, -1, np.int32))
    loss, dx, dw = ctx.native_cross_entropy_step(x, w, y, vocab=0)
    assert not np.any(loss.numpy()) and not np.any(dx.numpy()) and not np.any(dw.numpy())
    loss, log_sum = ctx.native_cross_entropy_loss(x, w, y, vocab=0)
    assert not np.any(loss.numpy()) and np.all(np.isneginf(log_sum.numpy()))


@pytest.mark.parametrize("rows", [3, 300, 3000])
def test_labels_out_of_range_are_faults(ctx, pcu_pkg, rows):
    x, w = ctx.upload(np.ones((rows, 16), np.float32)), ctx.upload(np.ones((30, 16), np.float32))
    labels = np.zeros(rows, np.int32)
    labels[[1, rows - 1]] = [29, 30]
    for call in (lambda: ctx.native_cross_entropy_loss(x, w, ctx.upload(labels)),
                 lambda: ctx.native_cross_entropy_step(x, w, ctx.upload(labels)),
                 lambda: ctx.native_cross_entropy_backward(x, w, ctx.upload(labels), ctx.upload(np.zeros(rows, np.float32)))):
        with pytest.raises(pcu_pkg.PcuExecutionError) as e:
            call()
        assert e.value.tensor_fault.element_index == rows - 1
    labels[1] = 2 ** 31 - 1
    with pytest.raises(pcu_pkg.PcuExecutionError) as e:
        ctx.native_cross_entropy_loss(x, w, ctx.upload(labels))
    assert e.value.tensor_fault.element_index == 1


def test_refusals(ctx, pcu_pkg):
    from fusion_pcu_amd import _abi
    f32 = lambda *s: ctx.empty(s, np.float32)
    x, w, y = f32(4, 8), f32(30, 8), ctx.upload(np.zeros(4, np.int32))
    half = lambda *s: ctx.empty(s, np.float16)
    for call in (lambda: ctx.native_cross_entropy_loss(x, f32(30, 9), y), lambda: ctx.native_cross_entropy_loss(x, half(30, 8), y),
                 lambda: ctx.native_cross_entropy_loss(x, w, f32(4)), lambda: ctx.native_cross_entropy_loss(x, w, y, vocab=31),
                 lambda: ctx.native_cross_entropy_loss(x, w, y, loss=f32(3)),
                 lambda: ctx.native_cross_entropy_loss(f32(4, 0), f32(30, 0), y),
                 lambda: ctx.native_cross_entropy_step(x, w, y, weight_gradient=f32(29, 8)),
                 lambda: ctx.native_cross_entropy_step(x, w, y, feature_gradient=x),
                 lambda: ctx.native_cross_entropy_step(x, w, y, weight_gradient=w),
                 lambda: ctx.native_cross_entropy_backward(x, w, y, f32(5)),
                 lambda: ctx.native_cross_entropy_step(x, w, y, row_scale=half(4))):
        with pytest.raises(pcu_pkg.PcuExecutionError):
            call()
    d64 = lambda *s: ctx.empty(s, np.float64)
    with pytest.raises(pcu_pkg.PcuExecutionError) as e:
        ctx.native_cross_entropy_loss(d64(4, 8), d64(30, 8), y)
    assert e.value.status == _abi.PCU_ERR_UNSUPPORTED
    lib, h = ctx._lib, ctx.handle
    big, out = f32(64, 64), f32(64, 64)
    R = lambda p, r=4, c=8, s=8, d=0: ctypes.byref(_abi.Rows(p, d, 0, r, c, s))
    A, S = _abi.PCU_ERR_ARGUMENT, _abi.PCU_ERR_SHAPE
    loss = lib.pcu_native_cross_entropy_loss
    assert loss(h, R(big.ptr), R(w.ptr, 30), None, out.ptr, None, None) == A
    assert loss(h, R(big.ptr), R(w.ptr, 30), y.ptr, None, None, None) == A
    assert loss(h, R(big.ptr), R(w.ptr, 30), y.ptr, out.ptr + 2, None, None) == A
    assert loss(h, R(big.ptr), R(w.ptr, 30), y.ptr, out.ptr, out.ptr + 8, None) == A
    assert loss(h, R(big.ptr + 1), R(w.ptr, 30), y.ptr, out.ptr, None, None) == A
    assert loss(h, None, R(w.ptr, 30), y.ptr, out.ptr, None, None) == A
    assert loss(h, R(big.ptr), R(None, 30), y.ptr, out.ptr, None, None) == A
    assert loss(h, R(big.ptr, r=(1 << 22) + 1), R(w.ptr, 30), y.ptr, out.ptr, None, None) == S
    assert loss(h, R(big.ptr), R(w.ptr, (1 << 22) + 1), y.ptr, out.ptr, None, None) == S
    assert loss(h, R(big.ptr, c=(1 << 16) + 1, s=1 << 17), R(w.ptr, 30, (1 << 16) + 1, 1 << 17), y.ptr, out.ptr, None, None) == S
    assert loss(h, R(big.ptr, r=1 << 22), R(w.ptr, 1 << 16), y.ptr, out.ptr, None, None) == S
    assert loss(h, R(big.ptr, c=1 << 16, s=1 << 16), R(w.ptr, 1 << 22, 1 << 16, 1 << 16), y.ptr, out.ptr, None, None) == S
    step = lib.pcu_native_cross_entropy_step
    assert step(h, R(x.ptr), R(w.ptr, 30), y.ptr, None, out.ptr, None, 0, out.ptr + 64, 29, 8, None) == S
    assert step(h, R(x.ptr), R(w.ptr, 30), y.ptr, None, out.ptr, out.ptr + 64, 7, None, 0, 0, None) == S
    assert step(h, R(x.ptr), R(w.ptr, 30), y.ptr, None, out.ptr, out.ptr + 64, 8, out.ptr + 128, 30, 8, None) == A
    back = lib.pcu_native_cross_entropy_backward
    assert back(h, R(x.ptr), R(w.ptr, 30), y.ptr, None, None, out.ptr, 8, None, 0, 0, None) == A
    assert not np.any(np.isnan(ctx.native_cross_entropy_loss(ctx.upload(np.ones((4, 8), np.float32)), ctx.upload(np.ones((30, 8), np.float32)), y)[0].numpy()))


# Binary32 weights above 8 MiB, split on the way to the tiles for at most 128 rows: every tile, odd widths, one slab and
# many, several pieces of the vocabulary, rows that start at any binary32 value.
@pytest.mark.parametrize("rows", [1, 32, 33, 64, 65, 128, 129])
@pytest.mark.parametrize("vocab,width", [(30001, 131), (2111, 1023), (70001, 33)])
@pytest.mark.parametrize("lead,more", [(0, 0), (1, 2)])
def test_large_binary32_weights(ctx, pcu_pkg, rows, vocab, width, lead, more):
    from fusion_pcu_amd import _abi
    rng = np.random.default_rng(rows + vocab)
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, rows, vocab, width, "f32")
    want = Exact(xv, wv, labels, "f32")
    x, y = ctx.upload(xa), ctx.upload(labels)
    loss, log_sum = ctx.empty((rows,), np.float32), ctx.empty((rows,), np.float32)
    dx, dw = ctx.empty((rows, width), np.float32), ctx.empty((vocab, width), np.float32)
    stride = width + more
    host = np.full(lead + vocab * stride, np.nan, np.float32)
    host[lead:].reshape(vocab, stride)[:, :width] = wa
    w = ctx.upload(host)
    xr, wr = _abi.Rows(x.ptr, 0, 0, rows, width, width), _abi.Rows(w.ptr + 4 * lead, 0, 0, vocab, width, stride)
    assert ctx._lib.pcu_native_cross_entropy_step(ctx.handle, ctypes.byref(xr), ctypes.byref(wr), y.ptr, None, loss.ptr, dx.ptr, width,
                                                  dw.ptr, vocab, width, None) == 0
    assert np.all(np.abs(loss.numpy() - want.loss) <= want.d_loss)
    _near(dx.numpy().astype(np.float64), want.dx, want.d_dx, "f32", "dx")
    _near(dw.numpy().astype(np.float64), want.dw, want.d_dw, "f32", "dw")
    assert ctx._lib.pcu_native_cross_entropy_loss(ctx.handle, ctypes.byref(xr), ctypes.byref(wr), y.ptr, loss.ptr, log_sum.ptr, None) == 0
    assert np.all(np.abs(loss.numpy() - want.loss) <= want.d_loss) and np.all(np.abs(log_sum.numpy() - want.log_sum) <= want.d_log_sum)


def test_few_rows_and_several_pieces(ctx, pcu_pkg):
    rng = np.random.default_rng(8)
    xa, xv, wa, wv, labels = _inputs(pcu_pkg, rng, 5, 140001, 17, "f32")
    want = Exact(xv, wv, labels, "f32")
    loss, dx, dw = ctx.native_cross_entropy_step(ctx.upload(xa), ctx.upload(wa), ctx.upload(labels))
    assert np.all(np.abs(loss.numpy() - want.loss) <= want.d_loss)
    _near(dx.numpy().astype(np.float64), want.dx, want.d_dx, "f32", "dx")
    _near(dw.numpy().astype(np.float64), want.dw, want.d_dw, "f32", "dw")


def test_binary32_parts_beyond_what_is_kept(ctx):
    """Weights whose parts take more than 2 GiB are split for every piece of the vocabulary. All but some of the
    vocabulary's rows are zeros, so that the definition needs those alone and the zeros' number."""
    rng = np.random.default_rng(6)
    rows, vocab, width = 130, 1000003, 384
    at = np.unique(np.concatenate([[0, 255, 256, 131071, 131072, 931839, 931840, vocab - 1], rng.integers(0, vocab, 500)]))
    some = (0.1 * rng.standard_normal((len(at), width))).astype(np.float32)
    weights = np.zeros((vocab, width), np.float32)
    weights[at] = some
    x = rng.standard_normal((rows, width)).astype(np.float32)
    which = rng.integers(0, len(at), rows)
    labels = at[which].astype(np.int32)
    labels[3] = -1
    has = labels >= 0
    xw, sw = x.astype(np.float64), some.astype(np.float64)
    l = xw @ sw.T
    log_sum = np.log(np.exp(l).sum(axis=1) + (vocab - len(at)))
    e = _sum_error("f32", width, np.abs(xw) @ np.abs(sw).T)
    d_log_sum = e.max(axis=1) + u * (16 * np.abs(l).max(axis=1) + vocab / 16 + 128)
    r = np.arange(rows)
    loss = np.where(has, log_sum - l[r, which], 0)
    d_loss = np.where(has, d_log_sum + e[r, which] + u * np.abs(loss), 0)
    g = np.exp(l - log_sum[:, None])
    d = g * np.expm1(e + d_log_sum[:, None] + u * (8 * np.abs(l) + 8))
    g[r, which] -= 1
    d = np.where(has[:, None], d + 3 * u * (np.abs(g) + d), 0)
    g = np.where(has[:, None], g, 0)
    zero = np.where(has, np.exp(-log_sum), 0)[:, None]
    d_zero = zero * (np.expm1(d_log_sum[:, None] + 8 * u) + 4 * u)
    xd, wd, yd = (ctx.upload(a) for a in (x, weights, labels))
    got_loss, dx, dw = ctx.native_cross_entropy_step(xd, wd, yd)
    size = np.abs(g) + d
    assert np.all(np.abs(got_loss.numpy() - loss) <= d_loss)
    _near(dx.numpy().astype(np.float64), g @ sw, d @ np.abs(sw) + _sum_error("f32", vocab, size @ np.abs(sw)), "f32", "dx")
    dw = dw.numpy()
    _near(dw[at].astype(np.float64), g.T @ xw, d.T @ np.abs(xw) + _sum_error("f32", rows, size.T @ np.abs(xw)), "f32", "dw")
    others = np.setdiff1d(np.concatenate([np.arange(0, vocab, 997), at + 1, at - 1]), np.concatenate([at, [-1, vocab]]))
    bound = d_zero.T @ np.abs(xw) + _sum_error("f32", rows, (zero + d_zero).T @ np.abs(xw))
    _near(dw[others].astype(np.float64), (zero.T @ xw).repeat(len(others), axis=0), bound, "f32", "dw of zeros")
    loss2, sums = ctx.native_cross_entropy_loss(xd, wd, yd)
    np.testing.assert_array_equal(_bits(loss2.numpy()), _bits(got_loss.numpy()))
    assert np.all(np.abs(sums.numpy() - log_sum) <= d_log_sum)
