"""The operators on logits (top logits, distillation, sampling) on the GPU against plain
implementations in 64 bits, at the sizes, ties, masks and settings where they can go wrong.

Tolerances. u is half the statistics' unit roundoff spacing (2^-24 binary32, 2^-53 binary64).
A row's exponentials are taken of (s - m) * c with c = log2(e) / T, which carries 3 roundings,
so an exponent x in natural units is off by at most 4 u |x| and the exponential by 2 u more (the
hardware's 2^x and the product); a sum of n positive terms over at least 64 lanes adds at most
(n / 64 + 16) u. With B the largest |s / T| (and |v / T|) of finite values this bounds the relative
error of a probability by R = u (8 B + n / 64 + 64) and the absolute error of a log-sum-exp by R as
well (its own rounding is within u |lse| <= u (B + log n)). Outputs are rounded once more to
their type.
"""
import ctypes

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

ONE = 1 << 40
DTYPES = ["f32", "f64", "bf16", "f16"]
OUT_U = {"f32": 2.0 ** -24, "f64": 2.0 ** -53, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # 24, 53, 8 and 11 bits
LEAST = {"f32": 2.0 ** -149, "f64": 2.0 ** -1074, "bf16": 2.0 ** -133, "f16": 2.0 ** -25}


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def _stored(pkg, x, dtype):
    """binary64 values as an array of the type, and the values that it then holds."""
    x = np.asarray(x, dtype=np.float64)
    with np.errstate(over="ignore"):
        if dtype == "bf16":
            a = pkg.to_bfloat16(x.astype(np.float32))
            return a, pkg.from_bfloat16(a).astype(np.float64)
        a = x.astype({"f32": np.float32, "f64": np.float64, "f16": np.float16}[dtype])
    return a, a.astype(np.float64)


def _values(pkg, a, dtype):
    return (pkg.from_bfloat16(a) if dtype == "bf16" else a).astype(np.float64)


def _u(dtype):
    return 2.0 ** -53 if dtype == "f64" else 2.0 ** -24


def _relative(dtype, n, *magnitudes):
    """R of the module's docstring."""
    b = max([0.0] + [float(np.max(np.abs(m[np.isfinite(m)]), initial=0.0)) for m in magnitudes])
    return _u(dtype) * (8 * b + n / 64 + 64)


def _lse(z):
    m = np.max(z, axis=1, keepdims=True)
    m = np.where(np.isfinite(m), m, 0.0)
    with np.errstate(divide="ignore", invalid="ignore"):
        return (m + np.log(np.sum(np.exp(z - m), axis=1, keepdims=True)))[:, 0]


def _order(x):
    """Value descending, index ascending, NaN after minus infinity."""
    nan = np.isnan(x)
    key = np.where(nan, -np.inf, x) + 0.0
    return np.lexsort((np.arange(x.size), -key, nan))


# ------------------------------------------------------------------------- top logits

TOP_SHAPES = [(1, 1, 1), (3, 7, 7), (2, 5, 9), (64, 33, 1), (5, 1000, 8), (130, 257, 31), (3, 8193, 100),
              (2, 8192, 1024), (2, 50257, 1024), (3, 40001, 500), (1, 131075, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k", TOP_SHAPES)
def test_top_logits_are_the_first_of_the_order(ctx, pcu_pkg, rows, vocab, k, dtype):
    rng = np.random.default_rng(rows + 3 * vocab + 7 * k)
    a, x = _stored(pcu_pkg, rng.normal(0, 3, (rows, vocab)), dtype)
    values, indices, log_sum = ctx.native_top_logits(ctx.upload(a), k, temperature=1.5)
    got_v, got_i = _values(pcu_pkg, values.numpy(), dtype), indices.numpy()
    for r in range(rows):
        want = _order(x[r])[:k]
        np.testing.assert_array_equal(got_i[r, : len(want)], want)
        np.testing.assert_array_equal(got_v[r, : len(want)], x[r][want])
        assert np.all(got_i[r, vocab:] == -1) and np.all(np.isneginf(got_v[r, vocab:]))
    tol = _relative(dtype, vocab, x / 1.5)
    assert np.max(np.abs(log_sum.numpy() - _lse(x / 1.5))) <= tol


def _hard_rows(n, rng):
    """Rows at which a selection can go wrong."""
    low = float(np.finfo(np.float16).min)
    few = rng.integers(-3, 4, n) / 2.0
    masked = np.where(rng.random(n) < 0.99, -np.inf, rng.normal(0, 1, n))
    zeros = np.where(rng.random(n) < 0.5, -0.0, 0.0)
    nans = np.where(rng.random(n) < 0.3, np.nan, rng.normal(0, 1, n))
    lowest = np.full(n, low)
    lowest[n // 2] = 1.0
    outlier = rng.normal(0, 1, n)
    outlier[n // 3] = 60000.0
    one_sided = -np.abs(rng.normal(0, 1, n)) - 1
    block = rng.normal(0, 1, n)
    block[: min(n, 3000)] += 20.0  # the largest values lie side by side
    return {
        "equal": np.full(n, 1.25), "few": few, "ascending": np.linspace(-8, 8, n), "descending": np.linspace(8, -8, n),
        "masked": masked, "all_masked": np.full(n, -np.inf), "zeros": zeros, "nans": nans,
        "all_nan": np.full(n, np.nan), "lowest": np.full(n, low), "lowest_but_one": lowest, "outlier": outlier,
        "negative": one_sided, "block": block, "infinite": np.where(np.arange(n) % 97 == 5, np.inf, few),
        "mostly_equal": np.where(rng.random(n) < 0.02, 3.0 + rng.random(n), 1.0),
    }


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab,k", [(700, 50), (9001, 300), (33000, 1024), (70000, 17)])
def test_top_logits_of_hard_rows(ctx, pcu_pkg, vocab, k, dtype):
    rows = _hard_rows(vocab, np.random.default_rng(vocab))
    a, x = _stored(pcu_pkg, np.stack(list(rows.values())), dtype)
    values, indices, log_sum = ctx.native_top_logits(ctx.upload(a), k)
    got_v, got_i, got_l = _values(pcu_pkg, values.numpy(), dtype), indices.numpy(), log_sum.numpy()
    for r, name in enumerate(rows):
        want = _order(x[r])[:k]
        np.testing.assert_array_equal(got_i[r], want, err_msg=name)
        np.testing.assert_array_equal(got_v[r], x[r][want], err_msg=name)
        np.testing.assert_array_equal(np.signbit(got_v[r]), np.signbit(x[r][want]), err_msg=name)
        if np.any(np.isnan(x[r])) or np.any(np.isposinf(x[r])):
            assert np.isnan(got_l[r]), name
        else:
            want_l = _lse(x[r: r + 1])[0]
            assert got_l[r] == want_l or abs(got_l[r] - want_l) <= _relative(dtype, vocab, x[r]), name


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride,vocab", [(1001, 1000), (1024, 997), (9000, 8999), (40003, 40000)])
def test_top_logits_of_padded_rows(ctx, pcu_pkg, stride, vocab, dtype):
    """Rows that start at every alignment, with larger values in the padding."""
    rng = np.random.default_rng(stride)
    full = rng.normal(0, 3, (9, stride))
    full[:, vocab:] = 100.0
    a, x = _stored(pcu_pkg, full, dtype)
    values, indices, log_sum = ctx.native_top_logits(ctx.upload(a), 20, vocab=vocab)
    for r in range(9):
        np.testing.assert_array_equal(indices.numpy()[r], _order(x[r, :vocab])[:20])
    tol = _relative(dtype, vocab, x[:, :vocab])
    assert np.max(np.abs(log_sum.numpy() - _lse(x[:, :vocab]))) <= tol


def test_top_logits_of_no_rows_and_no_entries(ctx):
    empty = ctx.empty((0, 5), np.float32)
    values, indices, log_sum = ctx.native_top_logits(empty, 3)
    assert values.shape == (0, 3) and indices.shape == (0, 3) and log_sum.shape == (0,)
    x = np.array([[1.0, 2.0]], dtype=np.float32)
    _, _, log_sum = ctx.native_top_logits(ctx.upload(x), 0)
    assert abs(log_sum.numpy()[0] - np.log(np.exp(1) + np.exp(2))) <= _relative("f32", 2, x)
    values, indices, log_sum = ctx.native_top_logits(ctx.upload(x), 2, vocab=0)
    assert np.all(indices.numpy() == -1) and np.isneginf(values.numpy()).all() and np.isneginf(log_sum.numpy()).all()


# ----------------------------------------------------------------------- distillation


def _plain_distill(s, tv, ti, tl, labels, t, a, b, scale):
    """Loss, both log-sum-exps and gradient in binary64, row by row."""
    rows, vocab = s.shape
    loss, sums, grad = np.zeros(rows), np.zeros((rows, 2)), np.zeros(s.shape)
    for r in range(rows):
        with np.errstate(all="ignore"):
            sums[r] = _lse(s[r: r + 1] / t)[0], _lse(s[r: r + 1])[0]
            there = (ti[r] >= 0) & ~np.isneginf(tv[r])
            at, z = ti[r][there], tv[r][there] / t
            base = tl[r] if tl is not None else (_lse(z[None])[0] if z.size else 0.0)
            q = np.exp(z - base)
            p = np.zeros(vocab) if np.isneginf(sums[r, 0]) else np.exp(s[r] / t - sums[r, 0])
            p1 = np.zeros(vocab) if np.isneginf(sums[r, 1]) else np.exp(s[r] - sums[r, 1])
            if a and q.sum() > 0:
                sat = s[r][at]
                log_p = np.where(np.isneginf(sat), -np.inf, sat / t - sums[r, 0])
                loss[r] += a * t * t * np.sum(np.where(q > 0, q * (z - base - log_p), 0.0))
                grad[r] += a * t * q.sum() * p
                np.add.at(grad[r], at, -a * t * q)
            if b and labels is not None and labels[r] >= 0:
                y = labels[r]
                loss[r] += b * (np.inf if np.isneginf(s[r][y]) else sums[r, 1] - s[r][y])
                grad[r] += b * p1
                grad[r][y] -= b
        grad[r] *= scale[r]
    return loss, sums, grad


def _distill_inputs(pkg, rng, rows, vocab, k, dtype, teacher_dtype, full, labelled, t):
    a, s = _stored(pkg, rng.normal(0, 3, (rows, vocab)), dtype)
    teacher = 0.5 * s + rng.normal(0, 2, (rows, vocab))
    ti = np.stack([np.argsort(-x, kind="stable")[:k] for x in teacher]).astype(np.int32).reshape(rows, k)
    tv_a, tv = _stored(pkg, np.take_along_axis(teacher, ti.astype(np.int64), 1), teacher_dtype)
    drop = rng.random((rows, k)) < 0.1
    drop[rows // 2] = True  # a row without entries
    ti = np.where(drop, rng.integers(-5, 0, (rows, k)), ti).astype(np.int32)
    tl = None
    if full:
        tl = _lse(teacher / t)
        tl = tl if teacher_dtype == "f64" else tl.astype(np.float32)
    labels = None
    if labelled:
        labels = np.where(rng.random(rows) < 0.3, -1, rng.integers(0, vocab, rows)).astype(np.int32)
        labels[rows // 2] = -1  # nor a label
        if k:
            labels[0] = max(ti[0, 0], 0)  # a label among the entries
    return a, s, tv_a, tv, ti, tl, labels


def _check_distill(ctx, pkg, dtype, teacher_dtype, a, s, tv_a, tv, ti, tl, labels, t, wa, wb, scale, vocab=None,
                   in_place=False):
    """All three calls against the plain form; `a` may have padding columns."""
    stat = np.float64 if dtype == "f64" else np.float32
    cols, n = a.shape[1], s.shape[1]
    scale = scale.astype(stat)
    kw = dict(teacher_log_sum=None if tl is None else ctx.upload(tl), labels=None if labels is None else ctx.upload(labels),
              temperature=t, distill_weight=wa, label_weight=wb, vocab=vocab)
    tv_d, ti_d, sc = ctx.upload(tv_a), ctx.upload(ti), ctx.upload(scale)
    student = ctx.upload(a)
    loss, sums = ctx.native_distill_loss(student, tv_d, ti_d, **kw)
    grad = ctx.native_distill_backward(student, tv_d, ti_d, sums, row_scale=sc, **kw)
    student2 = ctx.upload(a) if in_place else student
    loss2, grad2 = ctx.native_distill_step(student2, tv_d, ti_d, row_scale=sc, gradient=student2 if in_place else None, **kw)
    if in_place:
        student3 = ctx.upload(a)
        again = ctx.native_distill_backward(student3, tv_d, ti_d, sums, row_scale=sc, gradient=student3, **kw)
        np.testing.assert_array_equal(_values(pkg, again.numpy(), dtype), _values(pkg, grad.numpy(), dtype))
    want_loss, want_sums, want_grad = _plain_distill(s, tv, ti, None if tl is None else tl.astype(np.float64), labels, t,
                                                     wa, wb, scale.astype(np.float64))
    rel = _relative(dtype, n, s / t, s, tv / t, np.zeros(1) if tl is None else tl)
    fine = np.isfinite(want_sums)
    got = sums.numpy()
    np.testing.assert_array_equal(got[~fine], want_sums[~fine])
    assert np.all(np.abs(got[fine] - want_sums[fine]) <= rel)
    # A loss is a sum of q (log q - log p) with both logarithms off by at most rel and q by rel
    # relatively, and the label's term likewise: at most 4 rel times the sum of absolute terms.
    with np.errstate(all="ignore"):
        mass = 1.0 + (0 if tl is None else 1)
        size = abs(wa) * t * t * mass * (2 + np.abs(want_loss) / max(t * t * abs(wa), 1e-9) + np.log(n + 1)) + abs(wb) * (2 + np.abs(want_loss))
    for x in (loss.numpy(), loss2.numpy()):
        ok = np.isfinite(want_loss)
        np.testing.assert_array_equal(x[~ok], want_loss[~ok])
        assert np.all(np.abs(x[ok] - want_loss[ok]) <= (4 * rel * size)[ok] + _u(dtype) * np.abs(want_loss[ok]))
    # Absolute terms of a gradient: probabilities off by 2 rel (from the given log-sums), q by 2 rel.
    p_size = np.abs(scale[:, None]) * (abs(wa) * t * 2 * mass + abs(wb) * 2)
    for x in (grad.numpy(), grad2.numpy()):
        x = _values(pkg, x, dtype)
        assert x.shape == (s.shape[0], cols)
        assert np.all(x[:, n:] == 0)
        # Each term is at most 2 |gradient| + its own cancellation, so bound by the parts.
        err = np.abs(x[:, :n] - want_grad)
        parts = np.abs(want_grad) + np.minimum(p_size, 2 * p_size * _parts(s, t, want_sums, ti))
        assert np.all(err <= 4 * rel * parts + OUT_U[dtype] * np.abs(want_grad) * 1.01 + LEAST[dtype])
    return loss, grad


def _parts(s, t, sums, ti):
    """p, p1 and 1 at the entries and everywhere a label may be: the size of the terms that cancel."""
    with np.errstate(all="ignore"):
        p = np.exp(s / t - sums[:, :1]) + np.exp(s - sums[:, 1:])
    p = np.where(np.isfinite(p), p, 0.0)
    for r in range(s.shape[0]):
        p[r, ti[r][ti[r] >= 0]] += 1.0
    return p


DISTILL_SHAPES = [(1, 1, 1), (3, 5, 2), (7, 100, 0), (64, 1000, 16), (5, 1023, 100), (3, 4097, 7), (70, 5000, 33),
                  (66, 20001, 65), (2, 33000, 1024), (64, 36007, 20), (65, 70001, 12), (2, 140001, 50)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab,k", DISTILL_SHAPES)
def test_distillation_against_the_formulas(ctx, pcu_pkg, rows, vocab, k, dtype):
    rng = np.random.default_rng(rows + 11 * vocab + k)
    if vocab > 60000 and rows > 8:  # one type is enough at the largest size
        if dtype in ("f64", "f16"):
            pytest.skip("covered by the other types")
    for full, labelled, t, wa, wb in [(False, False, 2.0, 1.0, 0.0), (True, True, 1.0, 0.7, 0.3), (False, True, 3.0, 0.5, 0.5)]:
        teacher_dtype = dtype if labelled else {"f32": "bf16", "f64": "f32", "bf16": "f32", "f16": "f64"}[dtype]
        a, s, tv_a, tv, ti, tl, labels = _distill_inputs(pcu_pkg, rng, rows, vocab, k, dtype, teacher_dtype, full, labelled, t)
        scale = rng.normal(0, 1, rows)
        _check_distill(ctx, pcu_pkg, dtype, teacher_dtype, a, s, tv_a, tv, ti, tl, labels, t, wa, wb, scale,
                       in_place=labelled)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride,vocab", [(129, 128), (1056, 1001), (8196, 8193), (40100, 40007)])
@pytest.mark.parametrize("rows", [3, 80])
def test_distillation_of_padded_rows(ctx, pcu_pkg, stride, vocab, rows, dtype):
    rng = np.random.default_rng(stride + rows)
    if rows > 3 and vocab > 10000 and dtype != "bf16":
        pytest.skip("covered by bf16")
    a, s, tv_a, tv, ti, tl, labels = _distill_inputs(pcu_pkg, rng, rows, vocab, 9, dtype, dtype, True, True, 2.0)
    padded, _ = _stored(pcu_pkg, np.concatenate([s, np.full((rows, stride - vocab), 50.0)], 1), dtype)
    _check_distill(ctx, pcu_pkg, dtype, dtype, padded, s, tv_a, tv, ti, tl, labels, 2.0, 0.6, 0.4, np.ones(rows),
                   vocab=vocab, in_place=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [600, 9000, 150000])
def test_distillation_of_masked_rows(ctx, pcu_pkg, vocab, dtype):
    """Students with masked tokens (minus infinity and the type's lowest value), rows that are
    masked altogether, teachers whose entries are all minus infinity, the same index twice."""
    rng = np.random.default_rng(vocab)
    a, s, tv_a, tv, ti, tl, labels = _distill_inputs(pcu_pkg, rng, 8, vocab, 12, dtype, dtype, False, True, 2.0)
    low = {"f32": np.finfo(np.float32).min, "f64": np.finfo(np.float64).min, "bf16": -3.3895313892515355e38, "f16": -65504.0}[dtype]
    keep = np.zeros(s.shape, dtype=bool)
    for r in range(8):
        keep[r, ti[r][ti[r] >= 0]] = True
        keep[r, max(labels[r], 0)] = True
    hide = ~keep & (rng.random(s.shape) < 0.5)
    s[hide] = np.where(rng.random(s.shape) < 0.5, -np.inf, low)[hide]
    s[1] = -np.inf  # nothing left: p = 0, the loss is infinite where the teacher has entries
    tv[2] = -np.inf  # a teacher without a finite entry counts as none
    ti[3, 5:9] = ti[3, 4] if ti[3, 4] >= 0 else 17
    labels[4] = 3
    s[4, 3] = -np.inf  # the label itself is masked
    s[5] = np.nan
    ti[5], labels[5] = -1, -1  # nothing asks for this row: 0 whatever it holds
    a, s = _stored(pcu_pkg, s, dtype)
    tv_a, tv = _stored(pcu_pkg, tv, dtype)
    want = _plain_distill(np.where(np.isnan(s), 0.0, s), tv, ti, None, labels, 2.0, 0.5, 0.5, np.ones(8))
    kw = dict(labels=ctx.upload(labels), temperature=2.0, distill_weight=0.5, label_weight=0.5)
    loss, grad = ctx.native_distill_step(ctx.upload(a), ctx.upload(tv_a), ctx.upload(ti), **kw)
    got = _values(pcu_pkg, grad.numpy(), dtype)
    assert not np.isnan(loss.numpy()).any() and not np.isnan(got).any()
    assert loss.numpy()[5] == 0 and np.all(got[5] == 0)
    assert np.isposinf(loss.numpy()[1]) and np.isposinf(loss.numpy()[4])
    # Masked logits' own magnitude must not enter the error: |s| <= 20 where the mass is.
    rel = _relative(dtype, vocab, np.array([20.0]), tv / 2.0)
    ok = np.isfinite(want[0])
    assert np.all(np.abs(loss.numpy()[ok] - want[0][ok]) <= 64 * rel)
    assert np.all(np.abs(got - want[2]) <= 16 * rel + OUT_U[dtype] * np.abs(want[2]) * 1.01 + LEAST[dtype])


def test_distillation_passes_nan_and_infinity_on(ctx):
    s = np.random.default_rng(1).normal(0, 1, (3, 500)).astype(np.float32)
    s[0, 7], s[1, 9] = np.nan, np.inf
    tv, ti = np.ones((3, 2), np.float32), np.tile(np.array([[1, 2]], np.int32), (3, 1))
    loss, grad = ctx.native_distill_step(ctx.upload(s), ctx.upload(tv), ctx.upload(ti))
    assert np.isnan(loss.numpy()[:2]).all() and np.isfinite(loss.numpy()[2])
    assert np.isnan(grad.numpy()[:2]).all() and np.isfinite(grad.numpy()[2]).all()


def test_distillation_gradient_against_differences(ctx):
    """Central differences of the binary64 loss, step h: the truncation is h^2 / 6 times the third
    derivative (below T^2 in the units of the weights), the rounding |loss| 2^-52 / h."""
    rng = np.random.default_rng(3)
    rows, vocab, k, t, h = 3, 40, 6, 2.0, 1e-4
    s = rng.normal(0, 2, (rows, vocab))
    ti = np.stack([rng.permutation(vocab)[:k] for _ in range(rows)]).astype(np.int32)
    ti[1, 2] = ti[1, 4]  # twice the same
    tv, labels = rng.normal(0, 2, (rows, k)), np.array([5, -1, 7], np.int32)
    dev = [ctx.upload(x) for x in (tv, ti)]
    for tl in (None, ctx.upload(rng.normal(4, 0.1, rows))):
        kw = dict(teacher_log_sum=tl, labels=ctx.upload(labels), temperature=t, distill_weight=0.6, label_weight=0.4)
        _, grad = ctx.native_distill_step(ctx.upload(s), *dev, **kw)
        grad = grad.numpy()
        tol = h * h * t * t + 64 * 2.0 ** -52 / h
        for v in range(vocab):
            d = np.zeros(vocab)
            d[v] = h
            up = ctx.native_distill_loss(ctx.upload(s + d), *dev, **kw)[0].numpy()
            down = ctx.native_distill_loss(ctx.upload(s - d), *dev, **kw)[0].numpy()
            assert np.max(np.abs((up - down) / (2 * h) - grad[:, v])) <= tol


def test_distillation_is_the_same_on_every_run(ctx, pcu_pkg):
    rng = np.random.default_rng(9)
    for rows, vocab in ((66, 20001), (3, 140001)):
        a, s, tv_a, tv, ti, tl, labels = _distill_inputs(pcu_pkg, rng, rows, vocab, 40, "f32", "f32", False, True, 2.0)
        ti[:, 7] = ti[:, 3]
        args = [ctx.upload(x) for x in (a, tv_a, ti)]
        kw = dict(labels=ctx.upload(labels), temperature=2.0, distill_weight=0.5, label_weight=0.5)
        first = [x.numpy() for x in ctx.native_distill_step(*args, **kw)]
        for _ in range(3):
            again = [x.numpy() for x in ctx.native_distill_step(*args, **kw)]
            assert all(np.array_equal(p.view(np.uint32), q.view(np.uint32)) for p, q in zip(first, again))


# ---------------------------------------------------------------------------- sampling


def _weights(x, temperature, dtype):
    """The definition's integers, with the exponential in binary64 of the binary32 argument."""
    peak = np.max(np.where(np.isnan(x), -np.inf, x))
    with np.errstate(all="ignore"):
        inv = np.float32(1) / np.float32(temperature) if temperature else np.float32(np.inf)
        greedy = np.isinf(inv)
        inv = np.float32(1) if greedy else inv
        near = x - peak if dtype == "f64" else x.astype(np.float32) - np.float32(peak)
        z = (near.astype(np.float32) * inv).astype(np.float64)
        w = np.floor(np.where(x < peak, np.exp(z), 0.0) * 2.0 ** 40).astype(np.int64)
    w[x == peak] = ONE
    return w, greedy


def _plain_sample(x, u, temperature, top_k, top_p, min_p, dtype):
    """[(token, log_prob)] with u and top_p as they are and moved by 2^-20 of themselves: the device's
    binary32 exponential is within 2^-23 of the one here, so a running mass is within 2^-22 and its
    share of a total within 2^-21. The first is the definition's own."""
    n = x.size
    if n == 0 or np.all(np.isneginf(x) | np.isnan(x)):
        return [(-1, -np.inf)]
    w, greedy = _weights(x, temperature, dtype)
    by = _order(x)
    by = by[:1] if greedy else (by[:top_k] if 0 < top_k < n else by)
    mass, ws = int(w[by].sum()), w[by]
    before = np.cumsum(ws) - ws
    least = int(np.ceil(float(np.float32(min_p)) * 2 ** 40))
    top_p, out = float(np.float32(top_p)), []
    for p in (top_p, top_p * (1 - 2.0 ** -20), top_p * (1 + 2.0 ** -20)):
        part = int(p * 2 ** 31)
        kept = by if part >= 2 ** 31 else by[: max(1, int(np.sum(before < mass * part // 2 ** 31)))]
        kept = np.sort(kept[w[kept] >= least])
        upto = np.cumsum(w[kept])
        total = int(upto[-1])
        for v in (float(u), float(u) * (1 - 2.0 ** -20), min(float(u) * (1 + 2.0 ** -20), 1 - 2.0 ** -31)):
            token = kept[np.searchsorted(upto, total * int(v * 2 ** 31) // 2 ** 31, side="right")]
            out.append((int(token), float(np.log(float(w[token])) - np.log(float(total)))))
    return out


SETTINGS = [  # temperature, top_k, top_p, min_p
    (1.0, 0, 1.0, 0.0), (0.7, 50, 0.9, 0.0), (1.3, 0, 0.95, 0.0), (0.9, 0, 0.3, 0.02), (1.0, 1, 1.0, 0.0),
    (1.0, 0, 0.0, 0.0), (2.0, 7, 1.0, 0.2), (0.0, 5, 0.5, 0.1), (1e-39, 0, 1.0, 0.0), (1.0, 0, 1.0, 1.0),
    (0.5, 3000, 0.999, 0.0), (5.0, 0, 0.99, 0.0), (1e-3, 0, 0.9, 0.0), (1e4, 0, 0.8, 0.0), (1.0, 10 ** 9, 1.0, 1e-6),
    (1.0, 0, 1e-12, 0.0), (1.0, 1500, 1.0, 0.0),
]
UNIFORM = [0.0, 1 - 2.0 ** -24, 0.5, 0.999, 1e-9]


def _check_sample(ctx, pkg, x64, dtype, settings, uniforms, vocab=None, names=None):
    """Each row of x64 with each setting and uniform, in one call with arrays of settings."""
    a, x = _stored(pkg, x64, dtype)
    rows = [(r, s, u) for r in range(x.shape[0]) for s in settings for u in uniforms]
    big = a[[r for r, _, _ in rows]]
    arrays = dict(temperature=np.array([s[0] for _, s, _ in rows], np.float32),
                  top_k=np.array([s[1] for _, s, _ in rows], np.int32),
                  top_p=np.array([s[2] for _, s, _ in rows], np.float32),
                  min_p=np.array([s[3] for _, s, _ in rows], np.float32))
    u = np.array([u for _, _, u in rows], np.float32)
    tokens, log_prob = ctx.native_sample(ctx.upload(big), ctx.upload(u), vocab=vocab,
                                         **{n: ctx.upload(v) for n, v in arrays.items()})
    tokens, log_prob, exact = tokens.numpy(), log_prob.numpy(), 0
    for i, (r, s, _) in enumerate(rows):
        want = _plain_sample(x[r, :vocab] if vocab is not None else x[r], u[i], float(arrays["temperature"][i]), s[1], s[2], s[3], dtype)
        where = (names[r] if names else r, s, float(u[i]))
        drawn = [t for t, _ in want]
        assert min(drawn) <= tokens[i] <= max(drawn), where
        exact += tokens[i] == drawn[0]
        # Within the mass's 2^-21, and a unit of the weight (a small one has few bits).
        near = [lp for t, lp in want if t == tokens[i]]
        if near:
            tol = 2.0 ** -20 * (1 + abs(near[0])) + 2.0 ** -40 * np.exp(-near[0])
            assert np.isneginf(near[0]) and np.isneginf(log_prob[i]) or \
                min(near) - tol <= log_prob[i] <= max(near) + tol, where
    # A random number within 2^-20 of a boundary is rare, and half of those fall to one side.
    assert exact >= 0.98 * len(rows)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [1, 2, 63, 64, 65, 1000, 4099, 8193, 40001])
def test_samples_are_the_definitions(ctx, pcu_pkg, vocab, dtype):
    rng = np.random.default_rng(vocab)
    x = np.stack([rng.normal(0, 1, vocab), rng.normal(0, 4, vocab), -2 * np.log1p(rng.random(vocab) * vocab)])
    _check_sample(ctx, pcu_pkg, x, dtype, SETTINGS, UNIFORM + list(rng.random(3)))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [700, 9001, 70000])
def test_samples_of_hard_rows(ctx, pcu_pkg, vocab, dtype):
    rng = np.random.default_rng(vocab)
    rows = _hard_rows(vocab, rng)
    settings = SETTINGS if vocab < 20000 else SETTINGS[:4] + SETTINGS[10:12]
    _check_sample(ctx, pcu_pkg, np.stack(list(rows.values())), dtype, settings, [0.0, 0.37, 1 - 2.0 ** -24], names=list(rows))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("stride,vocab", [(101, 100), (1024, 999), (9007, 9000), (40003, 40000)])
def test_samples_of_padded_rows(ctx, pcu_pkg, stride, vocab, dtype):
    rng = np.random.default_rng(stride)
    x = rng.normal(0, 2, (3, stride))
    x[:, vocab:] = 30.0
    _check_sample(ctx, pcu_pkg, x, dtype, SETTINGS[:6], [0.0, 0.6, 1 - 2.0 ** -24], vocab=vocab)


def test_samples_follow_the_probabilities(ctx):
    """With n evenly spread random numbers each token is drawn n p times, to within one at each
    end of its interval, where p = exp(l / T) / sum in binary64 (its error of 1e-5 n is far
    below one)."""
    rng = np.random.default_rng(2)
    n, vocab, t = 2048, 300, 0.8
    row = rng.normal(0, 2, vocab).astype(np.float32)
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    tokens, _ = ctx.native_sample(ctx.upload(np.tile(row, (n, 1))), ctx.upload(u), temperature=t)
    p = np.exp(row.astype(np.float64) / t)
    p /= p.sum()
    drawn = np.bincount(tokens.numpy(), minlength=vocab)
    assert np.max(np.abs(drawn - n * p)) <= 1.01
    assert np.all(np.diff(tokens.numpy()) >= 0)  # by index


def test_a_rows_token_does_not_depend_on_its_batch(ctx):
    rng = np.random.default_rng(4)
    x = rng.normal(0, 2, (40, 30001)).astype(np.float32)
    u = rng.random(40).astype(np.float32)
    for kw in (dict(temperature=0.8, top_p=0.9), dict(top_k=40), dict()):
        whole, _ = ctx.native_sample(ctx.upload(x), ctx.upload(u), **kw)
        for r in (0, 17, 39):
            one, _ = ctx.native_sample(ctx.upload(x[r: r + 1]), ctx.upload(u[r: r + 1]), **kw)
            assert one.numpy()[0] == whole.numpy()[r]


def test_samples_of_no_rows_and_no_vocabulary(ctx):
    tokens, log_prob = ctx.native_sample(ctx.empty((0, 9), np.float32), ctx.empty((0,), np.float32))
    assert tokens.shape == (0,) and log_prob.shape == (0,)
    tokens, log_prob = ctx.native_sample(ctx.upload(np.ones((2, 4), np.float32)), ctx.upload(np.zeros(2, np.float32)), vocab=0)
    assert list(tokens.numpy()) == [-1, -1] and np.isneginf(log_prob.numpy()).all()


# ---------------------------------------------------------------------------- refusals


def _fault(pkg, call):
    with pytest.raises(pkg.PcuExecutionError) as e:
        call()
    assert e.value.status == 1
    return e.value.tensor_fault


def test_indices_and_labels_out_of_range_are_faults(ctx, pcu_pkg):
    s = ctx.upload(np.zeros((5, 50), np.float32))
    tv = ctx.upload(np.zeros((5, 3), np.float32))
    ti = np.zeros((5, 3), np.int32)
    ti[2, 1], ti[4, 0] = 50, 2 ** 31 - 1
    f = _fault(pcu_pkg, lambda: ctx.native_distill_step(s, tv, ctx.upload(ti)))
    assert f.kind == pcu_pkg.PcuExecutionFaultKind.InvalidFloatingOperand and f.element_index == 2 * 4 + 1
    f = _fault(pcu_pkg, lambda: ctx.native_distill_loss(s, tv, ctx.upload(ti)))
    assert f.element_index == 2 * 4 + 1
    ti[:] = 0
    labels = np.array([0, 49, -1, 50, 51], np.int32)
    f = _fault(pcu_pkg, lambda: ctx.native_distill_loss(s, tv, ctx.upload(ti), labels=ctx.upload(labels), label_weight=1.0))
    assert f.element_index == 3 * 4 + 3
    assert ctx.last_fault().element_index == 15
    ctx.native_distill_loss(s, tv, ctx.upload(ti))  # the next call is clean
    assert ctx.last_fault() is None


@pytest.mark.parametrize("name,bad", [("temperature", -1.0), ("temperature", np.nan), ("temperature", np.inf), ("top_p", 1.5),
                                      ("top_p", np.nan), ("min_p", -0.1), ("min_p", 2.0), ("uniform", 1.0),
                                      ("uniform", -1e-9), ("uniform", np.nan)])
def test_settings_out_of_range_are_faults(ctx, pcu_pkg, name, bad):
    x = ctx.upload(np.zeros((6, 20), np.float32))
    v = np.full(6, 0.5, np.float32)
    v[[3, 5]] = bad
    kw = {} if name == "uniform" else {name: ctx.upload(v)}
    u = ctx.upload(v if name == "uniform" else np.zeros(6, np.float32))
    assert _fault(pcu_pkg, lambda: ctx.native_sample(x, u, **kw)).element_index == 3
    if name != "uniform":
        with pytest.raises(pcu_pkg.PcuExecutionError) as e:
            ctx.native_sample(x, u, **{name: bad})
        assert e.value.status == 2


def test_arguments_are_refused(ctx, pcu_pkg):
    def refused(status, call):
        with pytest.raises(pcu_pkg.PcuExecutionError) as e:
            call()
        assert e.value.status == status, e.value

    f = lambda *shape: ctx.upload(np.zeros(shape, np.float32))
    i = lambda *shape: ctx.upload(np.zeros(shape, np.int32))
    s, tv, ti, u = f(4, 50), f(4, 3), i(4, 3), f(4)
    refused(4, lambda: ctx.native_top_logits(i(4, 50), 3))
    refused(3, lambda: ctx.native_top_logits(f(50), 3))
    refused(3, lambda: ctx.native_top_logits(s, 1025))
    refused(3, lambda: ctx.native_top_logits(s, -1))
    refused(3, lambda: ctx.native_top_logits(s, 3, vocab=51))
    refused(3, lambda: ctx.native_top_logits(s, 3, values=f(4, 4)))
    refused(3, lambda: ctx.native_top_logits(s, 3, indices=f(4, 3)))
    for t in (0.0, -1.0, np.nan, np.inf):
        refused(2, lambda: ctx.native_top_logits(s, 3, temperature=t))
        refused(2, lambda: ctx.native_distill_loss(s, tv, ti, temperature=t))
    refused(2, lambda: ctx.native_distill_loss(s, tv, ti, distill_weight=np.inf))
    refused(2, lambda: ctx.native_distill_loss(s, tv, ti, label_weight=np.nan))
    refused(3, lambda: ctx.native_distill_loss(s, f(3, 3), ti))
    refused(3, lambda: ctx.native_distill_loss(s, tv, i(4, 2)))
    refused(3, lambda: ctx.native_distill_loss(s, tv, tv))
    refused(3, lambda: ctx.native_distill_loss(s, f(4, 1025), i(4, 1025)))
    refused(3, lambda: ctx.native_distill_loss(s, tv, ti, labels=i(3)))
    refused(3, lambda: ctx.native_distill_loss(s, tv, ti, teacher_log_sum=f(4, 1)))
    refused(4, lambda: ctx.native_distill_loss(i(4, 50), tv, ti))
    refused(3, lambda: ctx.native_distill_backward(s, tv, ti, f(4)))
    refused(3, lambda: ctx.native_distill_backward(s, tv, ti, f(4, 2), row_scale=f(5)))
    refused(3, lambda: ctx.native_distill_step(s, tv, ti, gradient=f(4, 51)))
    refused(3, lambda: ctx.native_sample(s, f(5)))
    refused(3, lambda: ctx.native_sample(s, u, top_k=f(4)))
    refused(3, lambda: ctx.native_sample(s, u, temperature=i(4)))
    refused(3, lambda: ctx.native_sample(s, u, tokens=f(4)))
    # Outputs on other tensors.
    refused(2, lambda: ctx.native_sample(s, u, log_prob=u))
    refused(2, lambda: ctx.native_distill_loss(s, f(4, 1), i(4, 1), teacher_log_sum=u, loss=u))
    shifted = pcu_pkg.DeviceArray(ctx, s.ptr + 4, (3, 50), np.float32)
    part = pcu_pkg.DeviceArray(ctx, s.ptr, (3, 50), np.float32)
    refused(2, lambda: ctx.native_distill_step(part, f(3, 3), i(3, 3), gradient=shifted))
    # Inside the C ABI: null pointers, strides, sizes.
    from fusion_pcu_amd import _abi
    lib, out = pcu_pkg.lib(), u.ptr
    top = lambda lg, k=1: lib.pcu_native_top_logits(ctx.handle, lg and ctypes.byref(lg), k, 1.0, tv.ptr, ti.ptr, None)
    assert top(None) == 2
    assert top(_abi.Logits(s.ptr, 7, 0, 4, 50, 50)) == 2
    assert top(_abi.Logits(None, 0, 0, 4, 50, 50)) == 2
    assert top(_abi.Logits(s.ptr + 2, 0, 0, 3, 50, 50)) == 2
    assert top(_abi.Logits(s.ptr, 0, 0, 4, 50, 49)) == 3
    assert top(_abi.Logits(s.ptr, 0, 0, 4, 1 << 23, 1 << 23)) == 3
    assert top(_abi.Logits(s.ptr, 0, 0, 1 << 31, 50, 50)) == 3
    assert top(_abi.Logits(s.ptr, 0, 0, 4, 50, 50), 1025) == 3
    lg = _abi.Logits(s.ptr, 0, 0, 4, 50, 50)
    assert lib.pcu_native_sample(ctx.handle, ctypes.byref(lg), None, out, None, None) == 2
    assert lib.pcu_native_sample(None, ctypes.byref(lg), None, out, None, None) == 2
    assert lib.pcu_native_distill_loss(ctx.handle, ctypes.byref(lg), None, out, None, None) == 2


# ------------------------------------------------------------------- inside programs


def test_a_program_runs_them_together_and_stops_at_the_first_fault(ctx, pcu_pkg):
    rng = np.random.default_rng(6)
    rows, vocab, k = 37, 3001, 12
    x = ctx.upload(rng.normal(0, 1, (rows, 64)).astype(np.float32))
    w = ctx.upload(rng.normal(0, 1, (64, vocab)).astype(np.float32))
    u = ctx.upload(rng.random(rows).astype(np.float32))
    alone = ctx.native_matmul(x, w)
    tv, ti, tl = ctx.native_top_logits(alone, k, temperature=2.0)
    loss, grad = ctx.native_distill_step(alone, tv, ti, teacher_log_sum=tl, temperature=2.0)
    tokens, _ = ctx.native_sample(alone, u, top_p=0.9)
    with ctx.program():
        logits = ctx.native_matmul(x, w)
        tv2, ti2, tl2 = ctx.native_top_logits(logits, k, temperature=2.0)
        loss2, grad2 = ctx.native_distill_step(logits, tv2, ti2, teacher_log_sum=tl2, temperature=2.0)
        tokens2, _ = ctx.native_sample(logits, u, top_p=0.9)
        assert ctx.next_node() == 4
    for p, q in ((tv, tv2), (ti, ti2), (tl, tl2), (loss, loss2), (grad, grad2), (tokens, tokens2)):
        np.testing.assert_array_equal(p.numpy(), q.numpy())
    # A fault of node 1 is the one reported; the sample after it is skipped.
    bad = ti.numpy()
    bad[3, 4] = vocab
    bad_d, bad_u = ctx.upload(bad), ctx.upload(np.full(rows, 2.0, np.float32))
    marked = ctx.upload(np.full(rows, -7, np.int32))
    with pytest.raises(pcu_pkg.PcuExecutionError) as e:
        with ctx.program():
            ctx.native_top_logits(logits, k)
            ctx.native_distill_loss(logits, tv, bad_d)
            ctx.native_sample(logits, bad_u, tokens=marked)
    assert e.value.tensor_fault.node == 1 and e.value.tensor_fault.element_index == 3 * (k + 1) + 4
    assert np.all(marked.numpy() == -7)


def test_rows_past_two_to_the_thirty_one_elements(ctx, pcu_pkg):
    """Offsets into a long tensor: a few rows whose stride puts the last ones past 2^31 elements."""
    from fusion_pcu_amd import _abi
    rng = np.random.default_rng(8)
    rows, stride, vocab = 6, 1 << 29, 700
    buf = ctx.empty((rows * stride,), np.float16)
    a, x = _stored(pcu_pkg, rng.normal(0, 2, (rows, vocab + 64)), "f16")
    part = [pcu_pkg.DeviceArray(ctx, buf.ptr + 2 * r * stride, (vocab + 64,), np.float16) for r in range(rows)]
    for r in range(rows):
        ctx.upload_into(part[r], a[r])
    x = x[:, :vocab]
    lg = _abi.Logits(buf.ptr, _abi.PCU_F16, 0, rows, vocab, stride)
    values, indices, log_sum = ctx.empty((rows, 4), np.float16), ctx.empty((rows, 4), np.int32), ctx.empty((rows,), np.float32)
    ctx.check(ctx._lib.pcu_native_top_logits(ctx.handle, ctypes.byref(lg), 4, 1.0, values.ptr, indices.ptr, log_sum.ptr))
    for r in range(rows):
        np.testing.assert_array_equal(indices.numpy()[r], _order(x[r])[:4])
    u = ctx.upload(np.full(rows, 0.3, np.float32))
    p = _abi.Sampling(u.ptr, None, None, None, None, 1.0, 0, 1.0, 0.0)
    tokens = ctx.empty((rows,), np.int32)
    ctx.check(ctx._lib.pcu_native_sample(ctx.handle, ctypes.byref(lg), ctypes.byref(p), tokens.ptr, None, None))
    for r in range(rows):
        assert tokens.numpy()[r] in [t for t, _ in _plain_sample(x[r], np.float32(0.3), 1.0, 0, 1.0, 0.0, "f16")]
    d = _abi.Distill(values.ptr, indices.ptr, None, None, _abi.PCU_F16, 4, 1.0, 1.0, 0.0)
    loss = ctx.empty((rows,), np.float32)
    ctx.check(ctx._lib.pcu_native_distill_step(ctx.handle, ctypes.byref(lg), ctypes.byref(d), None, loss.ptr, buf.ptr,
                                               vocab, stride, None))
    want = _plain_distill(x, np.take_along_axis(x, indices.numpy().astype(np.int64), 1), indices.numpy(), None, None,
                          1.0, 1.0, 0.0, np.ones(rows))
    got = np.stack([q.numpy() for q in part])
    rel = _relative("f16", vocab, x)
    err = np.abs(got[:, :vocab].astype(np.float64) - want[2])
    assert np.all(err <= 16 * rel + OUT_U["f16"] * np.abs(want[2]) * 1.01 + LEAST["f16"])
    np.testing.assert_array_equal(got[:, vocab:], a[:, vocab:])  # the columns between are the caller's
    buf.free()


# ----------------------------------------------------------- the range of a temperature


@pytest.mark.parametrize("dtype", DTYPES)
def test_temperatures_without_a_number_for_them_are_refused(ctx, pcu_pkg, dtype):
    """Beyond the range in which the temperature, log2(e) / T and a loss's T^2 are numbers of the
    statistics' type."""
    a, _ = _stored(pcu_pkg, np.array([[0.0, -1.0, -np.inf, -2.0]]), dtype)
    s = ctx.upload(a)
    tv, ti = ctx.upload(np.zeros((1, 2), np.float32)), ctx.upload(np.array([[0, 1]], np.int32))
    sums = ctx.upload(np.zeros((1, 2), np.float64 if dtype == "f64" else np.float32))
    step = lambda **kw: ctx.native_distill_step(s, tv, ti, **kw)
    loss = lambda **kw: ctx.native_distill_loss(s, tv, ti, **kw)
    backward = lambda **kw: ctx.native_distill_backward(s, tv, ti, sums, **kw)
    top = lambda **kw: ctx.native_top_logits(s, 2, **kw)

    def refused(call, **kw):
        with pytest.raises(pcu_pkg.PcuExecutionError) as e:
            call(**kw)
        assert e.value.status == 2

    for t in ((1e-310, 5e-324) if dtype == "f64" else (4e-39, 1e-40, 1e-60, 3.5e38, 1e200)):
        for call in (step, loss, backward, top):
            refused(call, temperature=t)
    if dtype == "f64":
        for t in (1e-200, 1e200):  # the square
            refused(step, temperature=t)
            refused(loss, temperature=t)
            backward(temperature=t)
            top(temperature=t)
    else:
        for name in ("distill_weight", "label_weight"):
            for call in (step, loss, backward):
                refused(call, **{name: 1e39})


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(3, 700), (70, 9001), (3, 140001)])
def test_temperatures_at_the_ends_of_the_range(ctx, pcu_pkg, rows, vocab, dtype):
    """Logits of 0, -1 and masked ones, and powers of two as temperatures: everything below is exact but
    for the large temperature's log-sum-exps and probabilities, which carry the tolerance of any other."""
    rng = np.random.default_rng(vocab)
    stat = np.float64 if dtype == "f64" else np.float32
    x = np.where(rng.random((rows, vocab)) < 0.3, -np.inf, -1.0)
    best = rng.integers(0, vocab - 2, rows)
    x[np.arange(rows), best] = 0.0
    x[:, vocab - 2:] = -1.0
    a, x = _stored(pcu_pkg, x, dtype)
    s = ctx.upload(a)
    # The teacher's choice is the last logit, 1 below the student's.
    ti = np.tile(np.array([[vocab - 2, vocab - 1]], np.int32), (rows, 1))
    tv = np.tile(np.array([[-1.0, 0.0]], stat), (rows, 1))
    tv_d, ti_d = ctx.upload(tv), ctx.upload(ti)
    for t in ((2.0 ** -500, 2.0 ** -40) if dtype == "f64" else (2.0 ** -127, 2.0 ** -100, 2.0 ** -40)):
        # All mass lies on the largest: q and p are 0 or 1, loss T^2 / T, gradient -T and T.
        values, indices, log_sum = ctx.native_top_logits(s, 1, temperature=t)
        assert np.array_equal(indices.numpy()[:, 0], best) and np.all(log_sum.numpy() == 0)
        loss, grad = ctx.native_distill_step(s, tv_d, ti_d, temperature=t)
        loss2, sums = ctx.native_distill_loss(s, tv_d, ti_d, temperature=t)
        back = ctx.native_distill_backward(s, tv_d, ti_d, sums, temperature=t)
        want = np.zeros((rows, vocab))
        want[np.arange(rows), best] = t
        want[:, vocab - 1] = -t
        want = _stored(pcu_pkg, want, dtype)[1]
        assert np.all(sums.numpy()[:, 0] == 0)
        assert np.all(loss.numpy() == t) and np.all(loss2.numpy() == t)
        for g in (grad, back):
            np.testing.assert_array_equal(_values(pcu_pkg, g.numpy(), dtype), want)
    t = 2.0 ** 127
    n = np.sum(~np.isneginf(x), axis=1)
    rel = _relative(dtype, vocab, np.array([1.0]))
    assert np.max(np.abs(ctx.native_top_logits(s, 1, temperature=t)[2].numpy() - np.log(n))) <= rel
    loss, sums = ctx.native_distill_loss(s, tv_d, ti_d, temperature=t)
    assert np.max(np.abs(sums.numpy()[:, 0] - np.log(n))) <= rel
    # T^2 (log(n / 2)) is past binary32, and a number in binary64.
    want = t * t * np.log(n / 2)
    if dtype == "f64":
        assert np.all(np.abs(loss.numpy() - want) <= 4 * rel * t * t * (2 + np.log(n)))
    else:
        assert np.all(np.isposinf(loss.numpy()))
    # Small enough a weight brings the loss, and 2^-127 the gradient's factor, back.
    weight = 2.0 ** -140 if dtype != "f64" else 2.0 ** -127
    loss, grad = ctx.native_distill_step(s, tv_d, ti_d, temperature=t, distill_weight=weight)
    assert np.all(np.abs(loss.numpy() - weight * want) <= (4 * rel + _u(dtype)) * weight * t * t * (2 + np.log(n)))
    loss, sums = ctx.native_distill_loss(s, tv_d, ti_d, temperature=t)
    back = ctx.native_distill_backward(s, tv_d, ti_d, sums, temperature=t, distill_weight=2.0 ** -126)
    _, grad = ctx.native_distill_step(s, tv_d, ti_d, temperature=t, distill_weight=2.0 ** -126)
    want = np.where(np.isneginf(x), 0.0, 1.0 / n[:, None])
    want[:, vocab - 2:] -= 0.5
    for g in (grad, back):
        got = _values(pcu_pkg, g.numpy(), dtype) / 2
        assert np.all(np.abs(got - want) <= 4 * rel * (np.abs(want) + 1.0 / n[:, None]) + OUT_U[dtype] * np.abs(want) * 1.01
                      + LEAST[dtype])


def test_pointers_that_are_not_aligned_to_their_type_are_refused(ctx, pcu_pkg):
    """Before any launch; each pointer of the C ABI in turn, off by half a value. Aligned ones pass."""
    from fusion_pcu_amd import _abi
    lib = pcu_pkg.lib()
    f = lambda *shape: ctx.upload(np.zeros(shape, np.float64)).ptr
    lg = lambda dtype: _abi.Logits(f(4, 50), dtype, 0, 2, 20, 20)

    def each(call, pointers, off):
        assert call(*pointers) == 0
        for i in range(len(pointers)):
            moved = list(pointers)
            moved[i] += off[i]
            assert call(*moved) == 2, i

    for dtype, size, stat in ((_abi.PCU_F32, 4, 4), (_abi.PCU_F64, 8, 8), (_abi.PCU_BF16, 2, 4), (_abi.PCU_F16, 2, 4)):
        x = lg(dtype)
        each(lambda v, i, s: lib.pcu_native_top_logits(ctx.handle, ctypes.byref(x), 3, 1.0, v, i, s),
             [f(8), f(8), f(8)], [size // 2, 2, stat // 2])

        def distill(mode):
            def call(tv, ti, tl, labels, scale, sums, loss, out):
                d = _abi.Distill(tv, ti, tl, labels, dtype, 3, 1.0, 0.5, 0.5)
                args = (ctx.handle, ctypes.byref(x), ctypes.byref(d))
                if mode == "loss":
                    return lib.pcu_native_distill_loss(*args, loss, out, None)
                if mode == "backward":
                    return lib.pcu_native_distill_backward(*args, sums, scale, f(8, 8), 20, 20, None)
                return lib.pcu_native_distill_step(*args, scale, loss, f(8, 8), 20, 20, None)
            return call

        teacher, steps = [f(8), f(8), f(8), f(8)], [size // 2, 2, stat // 2, 2]
        a, b, c = f(8), f(8), f(8)
        one = stat // 2
        each(lambda tv, ti, tl, y, loss, out: distill("loss")(tv, ti, tl, y, None, None, loss, out), teacher + [a, b],
             steps + [one, one])
        each(lambda tv, ti, tl, y, scale, sums: distill("backward")(tv, ti, tl, y, scale, sums, None, None), teacher + [a, b],
             steps + [one, one])
        each(lambda tv, ti, tl, y, scale, loss: distill("step")(tv, ti, tl, y, scale, None, loss, None), teacher + [a, c],
             steps + [one, one])

        def sample(u, t, tk, tp, mp, tokens, log_prob):
            p = _abi.Sampling(u, t, tk, tp, mp, 1.0, 0, 1.0, 0.0)
            return lib.pcu_native_sample(ctx.handle, ctypes.byref(x), ctypes.byref(p), tokens, log_prob, None)

        each(sample, [f(8) for _ in range(7)], [2] * 7)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [50, 9000, 150000])
def test_a_masked_entry_of_a_row_with_nan_has_no_probability_either(ctx, pcu_pkg, vocab, dtype):
    """log p of a row that holds a NaN or plus infinity is NaN everywhere, at a masked entry or label as
    at any other; in a row of masked logits alone it is minus infinity."""
    s = np.zeros((6, vocab))
    s[:, [3, 4]] = -np.inf
    s[[0, 3], 7] = np.nan
    s[[1, 4], 9] = np.inf
    s[[2, 5]] = -np.inf
    s = ctx.upload(_stored(pcu_pkg, s, dtype)[0])
    tv = ctx.upload(np.zeros((6, 1), np.float32))
    ti = np.full((6, 1), -1, np.int32)
    labels = np.full(6, -1, np.int32)
    ti[:3], labels[3:] = 3, 4  # rows of an entry alone, rows of a label alone
    args = (s, tv, ctx.upload(ti))
    kw = dict(labels=ctx.upload(labels), distill_weight=0.5, label_weight=0.5, temperature=2.0)
    loss, grad = ctx.native_distill_step(*args, **kw)
    for x in (loss, ctx.native_distill_loss(*args, **kw)[0]):
        x = x.numpy()
        assert np.all(np.isnan(x[[0, 1, 3, 4]])) and np.all(np.isposinf(x[[2, 5]]))
    got = _values(pcu_pkg, grad.numpy(), dtype)
    assert np.all(np.isnan(got[[0, 1, 3, 4]])) and not np.any(np.isnan(got[[2, 5]]))


# --------------------------------------------- settings that hold for every row of a call


def _check_sample_of_all(ctx, pkg, x64, dtype, setting, u, names=None):
    """Rows of x64 with one setting, given as numbers, against the definition."""
    a, x = _stored(pkg, x64, dtype)
    temperature, top_k, top_p, min_p = setting
    u = np.asarray(u, np.float32)
    tokens, log_prob = ctx.native_sample(ctx.upload(a), ctx.upload(u), temperature=temperature, top_k=top_k, top_p=top_p,
                                         min_p=min_p)
    tokens, log_prob = tokens.numpy(), log_prob.numpy()
    for r in range(x.shape[0]):
        want = _plain_sample(x[r], u[r], float(np.float32(temperature)), top_k, top_p, min_p, dtype)
        where = (names[r] if names else r, setting, float(u[r]))
        drawn = [t for t, _ in want]
        assert min(drawn) <= tokens[r] <= max(drawn), where
        near = [lp for t, lp in want if t == tokens[r]]
        if near:
            tol = 2.0 ** -20 * (1 + abs(near[0])) + 2.0 ** -40 * np.exp(-near[0])
            assert np.isneginf(near[0]) and np.isneginf(log_prob[r]) or \
                min(near) - tol <= log_prob[r] <= max(near) + tol, where


# temperature, top_k, top_p, min_p. Long rows are done by the first launch where the chunks' lists of
# top_k make the row's, by the second without a nucleus or with a longer list, by the third with one.
ALL_ROWS = [(0.8, 50, 0.9, 0.0), (1.0, 5, 1.0, 0.0), (1.0, 1, 1.0, 0.0), (1.0, 0, 1.0, 0.05), (1.2, 0, 1.0, 0.0), (0.9, 0, 0.95, 0.0),
            (1.0, 0, 0.9, 0.02), (1.0, 400, 1.0, 0.0), (0.7, 400, 0.8, 0.1), (1.0, 3000, 1.0, 0.0), (1.0, 3000, 0.9, 0.0),
            (0.0, 0, 1.0, 0.0), (0.0, 0, 0.9, 0.0), (0.0, 50, 0.9, 0.1)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("vocab", [9001, 70000])
@pytest.mark.parametrize("copies", [1, 5])  # 16 rows end their program in the last launch, 80 do not
def test_samples_with_one_setting_are_the_definitions(ctx, pcu_pkg, vocab, copies, dtype):
    if copies > 1 and (vocab > 10000 or dtype in ("f64", "f16")):
        pytest.skip("covered by the shorter rows of the other types")
    rng = np.random.default_rng(vocab + copies)
    rows = _hard_rows(vocab, rng)
    names = list(rows) * copies
    x = np.tile(np.stack(list(rows.values())), (copies, 1))
    for setting in ALL_ROWS:
        _check_sample_of_all(ctx, pcu_pkg, x, dtype, setting, rng.random(len(names)), names)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,vocab", [(1, 50257), (3, 128000), (64, 9001)])
def test_samples_of_ordinary_rows_with_one_setting(ctx, pcu_pkg, rows, vocab, dtype):
    rng = np.random.default_rng(rows + vocab)
    x = rng.normal(0, 2, (rows, vocab)) - 2 * np.log1p(rng.random((rows, vocab)) * vocab)
    for setting in ALL_ROWS:
        _check_sample_of_all(ctx, pcu_pkg, x, dtype, setting, rng.random(rows))


@pytest.mark.parametrize("rows,vocab", [(4, 9001), (64, 9001), (4, 40001), (70, 9001)])
def test_one_invalid_random_number_of_a_call(ctx, pcu_pkg, rows, vocab):
    """The row is reported, however the call ends its program, and the next call is a clean one."""
    rng = np.random.default_rng(rows)
    x = ctx.upload(rng.normal(0, 2, (rows, vocab)).astype(np.float32))
    u = rng.random(rows).astype(np.float32)
    good = ctx.upload(u)
    u[rows - 2] = 1.0
    bad = ctx.upload(u)
    for temperature, top_k, top_p, min_p in ALL_ROWS:
        kw = dict(temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        want = [a.numpy() for a in ctx.native_sample(x, good, **kw)]
        assert _fault(pcu_pkg, lambda: ctx.native_sample(x, bad, **kw)).element_index == rows - 2
        for a, b in zip(ctx.native_sample(x, good, **kw), want):
            np.testing.assert_array_equal(a.numpy(), b)
