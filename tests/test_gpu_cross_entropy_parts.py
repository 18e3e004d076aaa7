"""What binary32 operands lose as three parts of 8 bits, product by product, on the GPU.

u = 2^-24. The second part of a value is at most 2^-8 of it and the third 2^-17, so the three products that are left
out are at most (1 + 2^-10) u of the whole. The six others are summed in binary32, the largest last: that addition is
off by at most 2 u of the whole, the one before it by 2 u of 2^-6 of it, and so on: 2.04 u. In all 3.1 u, and a result is
rounded once more where it is stored (u). Each bound below is 4 u, or 5 u for what is stored as a product with a factor.
Values: any mantissa, and those whose parts are largest (1 + 2^-7 - 2^-23 cut off after 8 bits leaves 7.8 u out).
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

u = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def _values(rng, n):
    """Binary32 values in [1, 2): of any mantissa, near the borders of 8 and 16 bits, and the largest rests."""
    v = rng.integers(0, 1 << 23, n)
    near = rng.choice([0, 1 << 16, 1 << 15, (1 << 16) - 1, (1 << 15) + 1, (1 << 15) + (1 << 7), (1 << 15) - (1 << 7) - 1], n)
    v = np.where(rng.random(n) < 0.5, (v & ~0xFFFF) + near & 0x7FFFFF, v)
    v[:2] = (1 << 16) - 1
    return (v.astype(np.uint32) | np.uint32(0x3F800000)).view(np.float32)


@pytest.mark.parametrize("weight", range(6))
@pytest.mark.parametrize("sign", [1, -1])
def test_a_logit_of_one_product(ctx, weight, sign):
    """A vocabulary of one token and a width of 1: the log-sum-exp is the product."""
    rng = np.random.default_rng(weight)
    x, w = _values(rng, 3000), sign * _values(rng, 8)[weight:weight + 1]
    _, sums = ctx.native_cross_entropy_loss(ctx.upload(x[:, None]), ctx.upload(w[:, None]), ctx.upload(np.zeros(3000, np.int32)))
    want = x.astype(np.float64) * w.astype(np.float64)
    assert np.max(np.abs(sums.numpy() - want) / np.abs(want)) <= 4 * u


@pytest.mark.parametrize("rows", [3, 100])
def test_a_logit_of_large_weights(ctx, rows):
    """Weights above 8 MiB, which few rows have split on their way to the tiles: all tokens but one have no probability."""
    rng = np.random.default_rng(rows)
    x, w = _values(rng, rows), np.full(2200001, -np.inf, np.float32)
    w[1500000] = _values(rng, 1)[0]
    _, sums = ctx.native_cross_entropy_loss(ctx.upload(x[:, None]), ctx.upload(w[:, None]), ctx.upload(np.full(rows, 1500000, np.int32)))
    want = x.astype(np.float64) * np.float64(w[1500000])
    assert np.max(np.abs(sums.numpy() - want) / want) <= 4 * u


@pytest.mark.parametrize("rows", [3, 40, 100, 500])
def test_gradients_of_one_product(ctx, rows):
    """Labels without probability, one a row: G is there -scale. Token 0 has all of it: its weight is 0 and its own
    gradient is left out, so both gradients are products of two values."""
    rng = np.random.default_rng(rows)
    x, w = _values(rng, rows), np.concatenate([[0.0], -1e4 * _values(rng, rows)]).astype(np.float32)
    scale = (_values(rng, rows) / 2).astype(np.float32)
    scale[0] = 1.0  # the others are kept relative to it
    labels = np.arange(1, rows + 1, dtype=np.int32)
    _, dx, dw = ctx.native_cross_entropy_step(ctx.upload(x[:, None]), ctx.upload(w[:, None]), ctx.upload(labels),
                                              row_scale=ctx.upload(scale))
    s, xv, wv = scale.astype(np.float64), x.astype(np.float64), w[1:].astype(np.float64)
    assert np.max(np.abs(dx.numpy()[:, 0] + s * wv) / np.abs(s * wv)) <= 5 * u
    assert np.max(np.abs(dw.numpy()[1:, 0] + s * xv) / (s * xv)) <= 5 * u


def test_the_largest_values(ctx):
    """Values that 8 bits would round to infinity."""
    x = np.array([[np.finfo(np.float32).max], [-3.3961e38], [3.3895314e38], [2.0 ** 127]], np.float32)
    w = np.array([[2.0 ** -100]], np.float32)
    for a, b in ((x, w), (w, x[:1])):
        _, sums = ctx.native_cross_entropy_loss(ctx.upload(a), ctx.upload(b), ctx.upload(np.zeros(len(a), np.int32)))
        want = a.astype(np.float64)[:, 0] * b.astype(np.float64)[0, 0]
        assert np.max(np.abs(sums.numpy() - want) / np.abs(want)) <= 4 * u
