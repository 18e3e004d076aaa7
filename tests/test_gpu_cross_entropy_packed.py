"""The cross entropy's 16-bit weights of odd width, whose copy for the gradients would take more than the 2 GiB that a call
keeps, on the GPU: they are copied for every piece of the vocabulary. Tolerances as in test_gpu_cross_entropy.py."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

u, U = 2.0 ** -24, 2.0 ** -11


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def _sum_error(n, magnitude):
    return u * (n / 2 + 67) * magnitude


def _near(got, want, bound, what):
    off, limit = np.abs(got - want), bound + U * (np.abs(want) + bound) + 2.0 ** -25
    assert np.all(off <= limit), (what, float(np.max(off / limit)))


@pytest.mark.parametrize("rows", [40, 300])
def test_weights_beyond_what_is_kept(ctx, rows):
    """1000003 rows of 1027 values, copied as 1088 each. All but some of the vocabulary's rows are zeros, so that the
    definition needs those alone and the zeros' number."""
    rng = np.random.default_rng(rows)
    vocab, width = 1000003, 1027
    at = np.unique(np.concatenate([[0, 255, 256, 196607, 196608, 393215, 393216, 786431, 786432, vocab - 1], rng.integers(0, vocab, 300)]))
    some = (0.1 * rng.standard_normal((len(at), width))).astype(np.float16)
    weights = np.zeros((vocab, width), np.float16)
    weights[at] = some
    x = rng.standard_normal((rows, width)).astype(np.float16)
    which = rng.integers(0, len(at), rows)
    labels = at[which].astype(np.int32)
    labels[3] = -1
    has, r = labels >= 0, np.arange(rows)
    scale = np.full(rows, 64.0, np.float32)
    xw, sw = x.astype(np.float64), some.astype(np.float64)
    l = xw @ sw.T
    log_sum = np.log(np.exp(l).sum(axis=1) + (vocab - len(at)))
    e = _sum_error(width, np.abs(xw) @ np.abs(sw).T)
    d_log_sum = e.max(axis=1) + u * (16 * np.abs(l).max(axis=1) + vocab / 16 + 128)
    loss = np.where(has, log_sum - l[r, which], 0)
    d_loss = np.where(has, d_log_sum + e[r, which] + u * np.abs(loss), 0)
    p = np.exp(l - log_sum[:, None])
    d = p * np.expm1(e + d_log_sum[:, None] + u * (8 * np.abs(l) + 8))
    g = p.copy()
    g[r, which] -= 1
    s = np.where(has, 64.0, 0)[:, None]
    d = s * (d + (U + 2 * u) * (np.abs(g) + d) + 2.0 ** -39)
    g = s * g
    zero = s * np.where(has, np.exp(-log_sum), 0)[:, None]
    d_zero = zero * (np.expm1(d_log_sum[:, None] + 8 * u) * 2 + U + 2 * u) + s * 2.0 ** -39
    xd, wd, yd, sd = (ctx.upload(a) for a in (x, weights, labels, scale))
    got_loss, dx, dw = ctx.native_cross_entropy_step(xd, wd, yd, row_scale=sd)
    size = np.abs(g) + d
    assert np.all(np.abs(got_loss.numpy() - loss) <= d_loss)
    _near(dx.numpy().astype(np.float64), g @ sw, d @ np.abs(sw) + _sum_error(vocab, size @ np.abs(sw)), "dx")
    dw = dw.numpy()
    _near(dw[at].astype(np.float64), g.T @ xw, d.T @ np.abs(xw) + _sum_error(rows, size.T @ np.abs(xw)), "dw")
    others = np.setdiff1d(np.concatenate([np.arange(0, vocab, 997), at + 1, at - 1]), np.concatenate([at, [-1, vocab]]))
    bound = d_zero.T @ np.abs(xw) + _sum_error(rows, (zero + d_zero).T @ np.abs(xw))
    _near(dw[others].astype(np.float64), (zero.T @ xw).repeat(len(others), axis=0), bound, "dw of zeros")
    loss2, sums = ctx.native_cross_entropy_loss(xd, wd, yd)
    assert np.all(np.abs(loss2.numpy() - loss) <= d_loss) and np.all(np.abs(sums.numpy() - log_sum) <= d_log_sum)
    # The gradients from those sums.
    dx2, dw2 = ctx.native_cross_entropy_backward(xd, wd, yd, sums, row_scale=sd)
    _near(dx2.numpy().astype(np.float64), g @ sw, d @ np.abs(sw) + _sum_error(vocab, size @ np.abs(sw)), "dx")
    _near(dw2.numpy()[at].astype(np.float64), g.T @ xw, d.T @ np.abs(xw) + _sum_error(rows, size.T @ np.abs(xw)), "dw")
