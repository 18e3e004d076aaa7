"""The embedding and its gradient at sizes of nothing, at long batches and long runs of one token, on the GPU. Results have
to be equal, bit for bit: values are whole numbers whose sums the type holds exactly, or two calls' sums are of the same terms."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def _fault(pkg, call):
    with pytest.raises(pkg.PcuExecutionError) as e:
        call()
    return e.value.tensor_fault.element_index


@pytest.mark.parametrize("dtype", [np.float32, np.float64, np.float16])
@pytest.mark.parametrize("rows", [1, 70, 1500, 100000])
def test_faults_where_there_is_nothing_to_compute(ctx, pcu_pkg, rows, dtype):
    """A token at or past the table's rows is a fault where the table has no rows or no columns, too."""
    tokens = np.full(rows, -1, np.int32)
    good = ctx.upload(tokens)
    tokens[[rows // 2, rows - 1]] = 3
    bad = ctx.upload(tokens)
    table, none, flat = ctx.empty((3, 0), dtype), ctx.empty((0, 5), dtype), ctx.empty((rows, 0), dtype)
    gradient = ctx.upload(np.ones((rows, 5), dtype))
    # No columns: forward and backward.
    assert ctx.native_embedding(table, good).shape == (rows, 0)
    assert _fault(pcu_pkg, lambda: ctx.native_embedding(table, bad)) == rows // 2
    assert ctx.native_embedding_backward(flat, good, 3).shape == (3, 0)
    assert _fault(pcu_pkg, lambda: ctx.native_embedding_backward(flat, bad, 3)) == rows // 2
    # No rows, in the table or of its gradient.
    assert not np.any(ctx.native_embedding(none, good).numpy())
    assert _fault(pcu_pkg, lambda: ctx.native_embedding(none, bad)) == rows // 2
    assert ctx.native_embedding_backward(gradient, good, 0).shape == (0, 5)
    assert _fault(pcu_pkg, lambda: ctx.native_embedding_backward(gradient, bad, 0)) == rows // 2
    assert ctx.native_embedding_backward(flat, good, 0).shape == (0, 0)
    # In a program, whose later calls are then left out; and the next call is right.
    mark = ctx.upload(np.full((3, 5), 7, dtype))
    with pytest.raises(pcu_pkg.PcuExecutionError):
        with ctx.program():
            ctx.native_embedding_backward(flat, bad, 3)
            ctx.native_embedding_backward(gradient, good, 3, out=mark)
    assert np.all(mark.numpy() == 7)
    assert not np.any(ctx.native_embedding_backward(gradient, good, 3, out=mark).numpy())


@pytest.mark.parametrize("dtype", [np.float32, np.float64, np.float16])
@pytest.mark.parametrize("width", [1, 5, 64, 300])
@pytest.mark.parametrize("times", [3, 48, 49, 95, 96, 97, 145, 1000])
def test_a_tokens_sum_does_not_depend_on_the_other_tokens(ctx, times, width, dtype):
    """Its terms in their order, wherever other tokens push them in the sorted order, and whatever these are."""
    rng = np.random.default_rng(times + width)
    rows, vocab, token = 2500, 400, 200
    terms = rng.normal(0, 1, (times, width)).astype(dtype)
    first = None
    for less in (0, 1, 7, 47, 48, 50, 333, 1499):
        others = np.concatenate([rng.choice([3, token - 1], less), rng.integers(token + 1, vocab, rows - times - less)]).astype(np.int32)
        tokens, gradient = np.empty(rows, np.int32), rng.normal(0, 1, (rows, width)).astype(dtype)
        place = np.sort(rng.permutation(rows)[:times])
        rest = np.setdiff1d(np.arange(rows), place)
        tokens[place], tokens[rest], gradient[place] = token, rng.permutation(others), terms
        got = ctx.native_embedding_backward(ctx.upload(gradient), ctx.upload(tokens), vocab).numpy()[token]
        first = got if first is None else first
        np.testing.assert_array_equal(got, first)
    u, size = {2: 2.0 ** -11, 4: 2.0 ** -24, 8: 2.0 ** -53}[first.itemsize], np.abs(terms.astype(np.float64)).sum(axis=0)
    acc = 2.0 ** -53 if dtype == np.float64 else 2.0 ** -24
    exact = terms.astype(np.longdouble).sum(axis=0)
    assert np.all(np.abs(first - exact) <= acc * times * size + u * (np.abs(exact) + acc * times * size))


@pytest.mark.parametrize("vocab", [5, 3000, 1 << 17, 1 << 22])
@pytest.mark.parametrize("rows", [65536, 65537, 70001, 512 * 2048, 512 * 2048 + 1, 1100003])
@pytest.mark.parametrize("width,base", [(1, False), (3, True)])
def test_long_batches(ctx, rows, vocab, width, base):
    """More than 32 tiles of 2048 tokens, whose counts are summed by launches of their own, and more than 512 tiles, which
    one workgroup's pass over them does not reach."""
    rng = np.random.default_rng(rows + vocab + width)
    tokens = (vocab * rng.random(rows) ** 3).astype(np.int32)  # some far more often than others
    tokens[rng.random(rows) < 0.1] = -1
    tokens[[0, rows - 1]] = vocab - 1
    gradient = rng.integers(-3, 4, (rows, width)).astype(np.float32)
    start = rng.integers(-9, 9, (vocab, width)).astype(np.float32)
    want = start.astype(np.float64) if base else np.zeros((vocab, width))
    for c in range(width):
        real = tokens >= 0
        want[:, c] += np.bincount(tokens[real], weights=gradient[real, c], minlength=vocab)
    got = ctx.native_embedding_backward(ctx.upload(gradient), ctx.upload(tokens), vocab, base=ctx.upload(start) if base else None)
    np.testing.assert_array_equal(got.numpy(), want)
