"""The cross entropy of an output layer whose logits are not kept, where operands or logits are infinite or NaN, on
the GPU against the definition in 64 bits: sums of products of which one is infinite, and what they leave of the rest.

Tolerances are those of test_gpu_cross_entropy.py: u = 2^-24, E(n, A) = u (pairs n / 2 + 67) A with A the sum of the
finite terms' magnitudes and `pairs` 6 for binary32 or 1; a log-sum-exp is off by L = E + u (16 B + vocab / 16 + 128), B the
largest finite |l| that counts, a loss by L + E. G is rounded by U relative to it (2^-39 of the largest scale in
binary16), its probabilities off by E + L + u (8 B + 8) relative to them. What is infinite or NaN has to be so.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

DTYPES = ["f32", "bf16", "f16"]
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}
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


def _sum_error(dtype, n, magnitude):
    return u * ((6 if dtype == "f32" else 1) * n / 2 + 67) * magnitude


def _near(got, want, bound, what):
    """Where `want` is finite within the bound, else the same infinity or NaN."""
    real = np.isfinite(want)
    np.testing.assert_array_equal(got[~real], want[~real], err_msg=what)
    off, limit = np.abs(got[real] - want[real]), np.broadcast_to(bound, want.shape)[real]
    assert np.all(off <= limit), (what, float(np.max(off / limit)))


# Few rows and small weights (packed); large ones that few rows read (split on the way to the tiles in binary32);
# many rows; one row and one word.
SHAPES = [(1, 1, 1), (7, 300, 64), (40, 300, 100), (5, 30001, 131), (100, 2111, 1023), (129, 1000, 200), (300, 5000, 64)]


def _masked(pkg, rows, vocab, width, dtype):
    """Features whose first value is a power of two (or another number of few bits), weights whose first is -inf at some
    tokens, as a bias that masks them: in every tile of the vocabulary, its first and last token among them."""
    rng = np.random.default_rng(rows + 3 * vocab + 7 * width)
    x, w = rng.normal(0, 1, (rows, width)), rng.normal(0, 2 / np.sqrt(width), (vocab, width))
    x[:, 0] = rng.choice([1.0, 0.5, 2.0, 1.5, 0.3], rows)
    masked = np.unique(np.concatenate([rng.integers(0, vocab, vocab // 50), np.arange(0, vocab, 100), [vocab - 1]]))
    masked = masked[:vocab - 1]
    labels = np.setdiff1d(np.arange(vocab), masked)[rng.integers(0, vocab - len(masked), rows)].astype(np.int32)
    (xa, xv), (wa, wv) = _stored(pkg, x, dtype), _stored(pkg, w, dtype)
    (whole, _), finite = _stored(pkg, np.where(np.isin(np.arange(vocab), masked)[:, None] & (np.arange(width) == 0), -np.inf, wv), dtype), wv
    return xa, xv, whole, finite, masked, labels


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", SHAPES)
def test_tokens_masked_by_infinite_weights(ctx, pcu_pkg, rows, vocab, width, dtype):
    """A -inf weight against a positive feature is a logit of -inf: probability 0, finite losses and gradients. The
    features' gradient of the infinite column alone is 0 * inf = NaN."""
    xa, xv, wa, wv, masked, labels = _masked(pcu_pkg, rows, vocab, width, dtype)
    kept = np.setdiff1d(np.arange(vocab), masked)
    x, w, y = ctx.upload(xa), ctx.upload(wa), ctx.upload(labels)
    l = xv @ wv[kept].T
    e = _sum_error(dtype, width, np.abs(xv) @ np.abs(wv[kept]).T)
    place = np.searchsorted(kept, labels)
    at = np.arange(rows)
    top = l.max(axis=1, keepdims=True)
    log_sum = (top + np.log(np.exp(l - top).sum(axis=1, keepdims=True)))[:, 0]
    d_log_sum = e.max(axis=1) + u * (16 * np.abs(l).max(axis=1) + vocab / 16 + 128)
    want, d_want = log_sum - l[at, place], d_log_sum + e[at, place] + u * np.abs(log_sum - l[at, place])
    loss, sums = ctx.native_cross_entropy_loss(x, w, y)
    _near(sums.numpy().astype(np.float64), log_sum, d_log_sum, "log_sum")
    _near(loss.numpy().astype(np.float64), want, d_want, "loss")
    p = np.exp(l - log_sum[:, None])
    g = p.copy()
    g[at, place] -= 1.0
    d = p * np.expm1(e + d_log_sum[:, None] + u * (8 * np.abs(l) + 8))
    d = d + (U[dtype] + 2 * u) * (np.abs(g) + d) + (2.0 ** -39 if dtype == "f16" else 0.0)
    size = np.abs(g) + d
    dw, d_dw = g.T @ xv, d.T @ np.abs(xv) + _sum_error(dtype, rows, size.T @ np.abs(xv))
    dx, d_dx = g @ wv[kept], d @ np.abs(wv[kept]) + _sum_error(dtype, vocab, size @ np.abs(wv[kept]))
    if len(masked):
        dx[:, 0] = np.nan
    for got_loss, got_dx, got_dw in (ctx.native_cross_entropy_step(x, w, y),
                                     (loss,) + ctx.native_cross_entropy_backward(x, w, y, sums)):
        _near(got_loss.numpy().astype(np.float64), want, d_want, "loss")
        _near(_values(pcu_pkg, got_dx.numpy()), dx, d_dx + U[dtype] * (np.abs(dx) + d_dx) + LEAST[dtype], "dx")
        got_dw = _values(pcu_pkg, got_dw.numpy())
        _near(got_dw[kept], dw, d_dw + U[dtype] * (np.abs(dw) + d_dw) + LEAST[dtype], "dw")
        assert not np.any(got_dw[masked])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("feature,weight", [(f, w) for f in (1.0, -0.25, np.inf, -np.inf)
                                            for w in (1.0, 0.5, 1.375, -2.0, 1.0 + 2.0 ** -7, np.inf, -np.inf, 0.0, np.nan)
                                            if not (np.isinf([f, w]).any() and f * w > 0)])
def test_one_product_with_an_infinity(ctx, pcu_pkg, feature, weight, dtype):
    """A vocabulary of one token: the log-sum-exp is the logit (here no +inf)."""
    want = feature * weight
    x, _ = _stored(pcu_pkg, np.full((3, 5), 0.0) + np.array([feature, 0, 0, 1, 0]), dtype)
    w, _ = _stored(pcu_pkg, np.array([[weight, 0, 0, 0.5, 0]]), dtype)
    _, sums = ctx.native_cross_entropy_loss(ctx.upload(x), ctx.upload(w), ctx.upload(np.zeros(3, np.int32)))
    np.testing.assert_array_equal(sums.numpy(), np.full(3, want + 0.5, np.float32))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 64, 130])
def test_an_infinite_scale_of_one_row(ctx, pcu_pkg, width, dtype):
    """G is then +inf but for the label's -inf, and the weights' gradient the infinity of the feature's sign."""
    rng = np.random.default_rng(width)
    x, xv = _stored(pcu_pkg, rng.choice([1.0, -1.0, 0.5, 1.3, -0.7], (1, width)), dtype)
    w, _ = _stored(pcu_pkg, rng.normal(0, 1 / np.sqrt(width), (20, width)), dtype)
    label = np.array([4], np.int32)
    _, dw = ctx.native_cross_entropy_step(ctx.upload(x), ctx.upload(w), ctx.upload(label),
                                          row_scale=ctx.upload(np.array([np.inf], np.float32)))[1:]
    want = np.where(np.arange(20)[:, None] == 4, -np.inf, np.inf) * xv
    np.testing.assert_array_equal(_values(pcu_pkg, dw.numpy()), want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,width", [(2, 8, 2), (40, 300, 100), (5, 40001, 70), (129, 1000, 200), (300, 5000, 64)])
def test_an_infinite_logit(ctx, pcu_pkg, rows, vocab, width, dtype):
    """An infinite weight: a logit of +inf in rows whose feature is positive, -inf in the others. The first have an
    infinite log-sum-exp, an infinite loss (NaN if it is the label's), and reach the other tokens' weights through
    their label alone."""
    rng = np.random.default_rng(rows + vocab)
    x, w = rng.normal(0, 1, (rows, width)), rng.normal(0, 1 / np.sqrt(width), (vocab, width))
    x[:, 1] = rng.choice([1.0, -1.0, 0.3, -0.7], rows)
    x[0, 1], x[-1, 1] = 1.0, -0.5
    labels = rng.integers(0, vocab, rows).astype(np.int32)
    labels[labels == 7] = 6
    labels[rows // 2] = 7
    (xa, xv), (_, wv) = _stored(pcu_pkg, x, dtype), _stored(pcu_pkg, w, dtype)
    wv[7, 1] = np.inf
    wa, _ = _stored(pcu_pkg, wv, dtype)
    kept, at = np.arange(vocab) != 7, np.arange(rows)
    up = xv[:, 1] > 0
    inner = np.where(np.isinf(wv), 0, wv)
    l = xv @ inner.T
    e = _sum_error(dtype, width, np.abs(xv) @ np.abs(inner).T)
    log_sum = np.where(up, np.inf, np.log(np.exp(l[:, kept]).sum(axis=1)))
    l[:, 7] = np.where(up, np.inf, -np.inf)
    d_log_sum = e.max(axis=1) + u * (16 * np.abs(l[:, kept]).max(axis=1) + vocab / 16 + 128)
    with np.errstate(invalid="ignore"):
        want = log_sum - l[at, labels]
        d_want = d_log_sum + e[at, labels] + u * np.abs(want)
        p = np.exp(l - log_sum[:, None])[:, kept]
    x, w, y = ctx.upload(xa), ctx.upload(wa), ctx.upload(labels)
    loss, sums = ctx.native_cross_entropy_loss(x, w, y)
    _near(sums.numpy().astype(np.float64), log_sum, d_log_sum, "log_sum")
    _near(loss.numpy().astype(np.float64), want, d_want, "loss")
    g = p - (np.arange(vocab) == labels[:, None])[:, kept]
    d = p * np.expm1((e + d_log_sum[:, None])[:, kept] + u * (8 * np.abs(l[:, kept]) + 8))
    d = d + (U[dtype] + 2 * u) * (np.abs(g) + d) + (2.0 ** -39 if dtype == "f16" else 0.0)
    dw, d_dw = g.T @ xv, d.T @ np.abs(xv) + _sum_error(dtype, rows, (np.abs(g) + d).T @ np.abs(xv))
    for got_loss, _, got in (ctx.native_cross_entropy_step(x, w, y), (loss,) + ctx.native_cross_entropy_backward(x, w, y, sums)):
        _near(got_loss.numpy().astype(np.float64), want, d_want, "loss")
        got = _values(pcu_pkg, got.numpy())
        _near(got[kept], dw, d_dw + U[dtype] * (np.abs(dw) + d_dw) + LEAST[dtype], "dw")
        assert np.all(np.isnan(got[7]))
