"""The operators on logits as they are used together, and where the way a call is carried out
changes with its sizes: every way gives a row the same results, bit for bit."""
import importlib.util
import os

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def test_the_example_learns_and_writes(ctx, pcu_pkg):
    spec = importlib.util.spec_from_file_location("distill_and_sample", os.path.join(ROOT, "examples", "distill_and_sample.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses, text = example.run(ctx)
    # Plain 64-bit training on inputs drawn alike ends at 0.23 of its first loss.
    assert np.all(np.isfinite(losses)) and losses[-1] < 0.5 * losses[0]
    assert text.shape == (4, 13) and np.all((text >= 0) & (text < 1000))
    again, same = example.run(ctx)
    assert losses == again and np.array_equal(text, same)


def _distill_args(ctx, rng, rows, vocab, k, dtype=np.float32):
    s = rng.normal(0, 2, (rows, vocab)).astype(dtype)
    ti = rng.integers(0, vocab, (rows, k)).astype(np.int32)
    ti[0, : k // 2] = ti[0, 0]  # duplicates
    ti[rows // 2, 1] = -1
    tv = rng.normal(0, 2, (rows, k)).astype(np.float32)
    labels = rng.integers(-1, vocab, rows).astype(np.int32)
    return s, tv, ti, labels


def _some(a, rows):
    return np.ascontiguousarray(a[rows])


# 64 rows end their program in the kernel, 65 do not.
@pytest.mark.parametrize("vocab", [250, 1000])
@pytest.mark.parametrize("dtype", [np.float32, np.float64, np.float16])
@pytest.mark.parametrize("pad", [0, 3])
def test_small_calls_give_a_row_what_larger_ones_do(ctx, vocab, dtype, pad):
    rng = np.random.default_rng(vocab + pad)
    rows = 130
    s, tv, ti, labels = _distill_args(ctx, rng, rows, vocab + pad, 9, dtype)
    ti, labels = np.minimum(ti, vocab - 1), np.minimum(labels, vocab - 1)

    def call(part):
        x = ctx.upload(_some(s, part))
        loss, grad = ctx.native_distill_step(x, ctx.upload(_some(tv, part)), ctx.upload(_some(ti, part)), vocab=vocab,
                                             labels=ctx.upload(_some(labels, part)), temperature=1.7, label_weight=0.4)
        loss2, sums = ctx.native_distill_loss(x, ctx.upload(_some(tv, part)), ctx.upload(_some(ti, part)), vocab=vocab,
                                              labels=ctx.upload(_some(labels, part)), temperature=1.7, label_weight=0.4)
        values, indices, log_sum = ctx.native_top_logits(x, 9, vocab=vocab)
        tokens, log_prob = ctx.native_sample(x, ctx.upload(np.linspace(0, 0.99, rows, dtype=np.float32)[part]), top_p=0.9,
                                             vocab=vocab)
        return [a.numpy() for a in (loss, grad, loss2, sums, values, indices, log_sum, tokens, log_prob)]

    whole = call(np.arange(rows))
    for part in (np.arange(64), np.arange(64, 65), np.arange(65, 130)):
        for a, b in zip(call(part), whole):
            np.testing.assert_array_equal(a, b[part])


# Rows split over workgroups (few of them) and rows that one workgroup holds; the sums' order differs,
# so the bound is that of two sums of n positive terms and the exponentials of each.
def test_few_long_rows_agree_with_many(ctx):
    rng = np.random.default_rng(3)
    rows, vocab, k = 64, 40007, 20
    s, tv, ti, labels = _distill_args(ctx, rng, rows, vocab, k)
    kw = dict(temperature=1.3, label_weight=0.6)
    many = ctx.native_distill_step(ctx.upload(s), ctx.upload(tv), ctx.upload(ti), labels=ctx.upload(labels), **kw)
    few = ctx.native_distill_step(ctx.upload(s[:5]), ctx.upload(tv[:5]), ctx.upload(ti[:5]), labels=ctx.upload(labels[:5]), **kw)
    rel = 2 * 2.0 ** -24 * (8 * np.abs(s).max() + vocab / 64 + 64)
    scale = 1.3 * 1.3 + 0.6
    for a, b in zip(few, many):
        a, b = a.numpy().astype(np.float64), b.numpy()[:5].astype(np.float64)
        assert np.max(np.abs(a - b)) <= rel * scale * 16


@pytest.mark.parametrize("rows,vocab", [(3, 70001), (5, 150000), (70, 9001)])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
def test_a_gradient_in_the_logits_place(ctx, rows, vocab, temperature):
    rng = np.random.default_rng(rows)
    s, tv, ti, labels = _distill_args(ctx, rng, rows, vocab, 30)
    args = [ctx.upload(a) for a in (tv, ti)]
    kw = dict(labels=ctx.upload(labels), temperature=temperature, label_weight=0.5)
    x = ctx.upload(s)
    loss, grad = ctx.native_distill_step(x, *args, **kw)
    loss2, grad2 = ctx.native_distill_step(x, *args, gradient=x, **kw)
    assert grad2 is x
    np.testing.assert_array_equal(loss.numpy(), loss2.numpy())
    np.testing.assert_array_equal(grad.numpy(), x.numpy())
    x = ctx.upload(s)
    _, sums = ctx.native_distill_loss(x, *args, **kw)
    apart = ctx.native_distill_backward(x, *args, sums, **kw).numpy()
    ctx.native_distill_backward(x, *args, sums, gradient=x, **kw)
    np.testing.assert_array_equal(apart, x.numpy())


def test_a_large_gradient_is_a_small_ones(ctx):
    """Gradients above the size that is stored past the caches against those of the rows' halves."""
    rng = np.random.default_rng(4)
    rows, vocab = 300, 60001  # 72 MB
    s, tv, ti, labels = _distill_args(ctx, rng, rows, vocab, 40)

    def call(part):
        x = ctx.upload(_some(s, part))
        args = [ctx.upload(_some(a, part)) for a in (tv, ti)]
        kw = dict(labels=ctx.upload(_some(labels, part)), temperature=2.0, label_weight=0.2)
        loss, grad = ctx.native_distill_step(x, *args, **kw)
        _, sums = ctx.native_distill_loss(x, *args, **kw)
        back = ctx.native_distill_backward(x, *args, sums, **kw)
        return [a.numpy() for a in (loss, grad, sums, back)]

    whole = call(np.arange(rows))
    for part in (np.arange(150), np.arange(150, 300)):
        for a, b in zip(call(part), whole):
            np.testing.assert_array_equal(a, b[part])


def _mixed(ctx, rng, rows):
    return {"temperature": ctx.upload((0.5 + rng.random(rows)).astype(np.float32)),
            "top_k": ctx.upload(np.where(rng.random(rows) < 0.5, rng.integers(1, 1500, rows), 0).astype(np.int32)),
            "top_p": ctx.upload(np.where(rng.random(rows) < 0.5, rng.random(rows), 1.0).astype(np.float32)),
            "min_p": ctx.upload(np.where(rng.random(rows) < 0.3, 0.1, 0.0).astype(np.float32))}


@pytest.mark.parametrize("dtype,vocab", [(np.float64, 2101), (np.float32, 4111)])
def test_samples_of_more_rows_than_share_a_scratch(ctx, dtype, vocab):
    rng = np.random.default_rng(vocab)
    rows = 2100
    x = rng.normal(0, 2, (rows, vocab)).astype(dtype)
    u = rng.random(rows).astype(np.float32)
    settings = _mixed(ctx, rng, rows)
    tokens, log_prob = ctx.native_sample(ctx.upload(x), ctx.upload(u), **settings)
    tokens, log_prob = tokens.numpy(), log_prob.numpy()
    assert np.all((tokens >= 0) & (tokens < vocab))
    host = {n: a.numpy() for n, a in settings.items()}
    for part in (np.arange(7), np.arange(1000, 1070), np.arange(2040, 2100)):
        t, lp = ctx.native_sample(ctx.upload(_some(x, part)), ctx.upload(u[part]),
                                  **{n: ctx.upload(_some(a, part)) for n, a in host.items()})
        np.testing.assert_array_equal(t.numpy(), tokens[part])
        np.testing.assert_array_equal(lp.numpy(), log_prob[part])


def test_samples_after_a_fault_are_what_they_were(ctx, pcu_pkg):
    """What the launches of long rows leave for the next call is in order again after a fault, in a
    call of its own and in a program whose later nodes are skipped."""
    rng = np.random.default_rng(12)
    rows, vocab = 40, 30001
    x = ctx.upload(rng.normal(0, 2, (rows, vocab)).astype(np.float32))
    u = rng.random(rows).astype(np.float32)
    good, settings = ctx.upload(u), _mixed(ctx, rng, rows)
    bad = u.copy()
    bad[17] = 1.5
    bad = ctx.upload(bad)
    want = ctx.native_sample(x, good, **settings)[0].numpy()
    with pytest.raises(pcu_pkg.PcuExecutionError) as e:
        ctx.native_sample(x, bad, **settings)
    assert e.value.tensor_fault.element_index == 17
    np.testing.assert_array_equal(ctx.native_sample(x, good, **settings)[0].numpy(), want)
    with pytest.raises(pcu_pkg.PcuExecutionError):
        with ctx.program():
            ctx.native_sample(x, bad, **settings)
            ctx.native_sample(x, good, **settings)
    for _ in range(2):
        np.testing.assert_array_equal(ctx.native_sample(x, good, **settings)[0].numpy(), want)
    with ctx.program():
        tokens = [ctx.native_sample(x, good, **settings)[0] for _ in range(3)]
    for t in tokens:
        np.testing.assert_array_equal(t.numpy(), want)


def test_more_rows_than_one_axis_of_a_grid(ctx, pcu_pkg):
    """17 million rows of three logits: more threads than a launch takes along one axis."""
    rows, vocab = (1 << 24) + 259, 3
    rng = np.random.default_rng(9)
    x = rng.integers(-8, 9, (rows, vocab), dtype=np.int8).astype(np.float16)
    xd = ctx.upload(x)
    values, indices, _ = ctx.native_top_logits(xd, 1)
    first = np.argmax(x, axis=1)  # the lowest index of the largest
    assert np.array_equal(indices.numpy()[:, 0], first)
    assert np.array_equal(values.numpy()[:, 0], x[np.arange(rows), first])
    tokens, _ = ctx.native_sample(xd, ctx.upload(np.zeros(rows, np.float32)), top_k=1)
    assert np.array_equal(tokens.numpy(), first)
    # One entry a row, the largest logit: q = 1 and T = 1, so the gradient is p less one there.
    loss, grad = ctx.native_distill_step(xd, values, indices)
    back = ctx.native_distill_backward(xd, values, indices, ctx.native_distill_loss(xd, values, indices)[1])
    e = np.exp(x.astype(np.float32) - x.max(axis=1, keepdims=True))
    total = e.sum(axis=1)
    # Exponents of at most 16: each side within 200 units of binary32; the gradient's own rounding 2^-11.
    tol = 400 * 2.0 ** -24
    want = e / total[:, None]
    want[np.arange(rows), first] -= 1
    assert np.max(np.abs(loss.numpy() - np.log(total))) <= tol
    for g in (grad, back):
        assert np.max(np.abs(g.numpy() - want)) <= tol + 2.0 ** -11
    labels = np.full(rows, -1, np.int32)
    labels[-1] = vocab
    with pytest.raises(pcu_pkg.PcuExecutionError) as e:
        ctx.native_distill_loss(xd, values, indices, labels=ctx.upload(labels), label_weight=1.0)
    assert e.value.tensor_fault.element_index == (rows - 1) * 2 + 1


def test_rows_without_logits(ctx):
    """Rows of padding alone: every output as a row without probabilities has it."""
    x = ctx.upload(np.ones((5, 3), np.float32))
    tv, ti = ctx.upload(np.zeros((5, 2), np.float32)), ctx.upload(np.full((5, 2), -1, np.int32))
    loss, grad = ctx.native_distill_step(x, tv, ti, vocab=0)
    assert np.all(loss.numpy() == 0) and np.all(grad.numpy() == 0)
    loss, sums = ctx.native_distill_loss(x, tv, ti, vocab=0)
    assert np.all(loss.numpy() == 0) and np.all(np.isneginf(sums.numpy()))
    grad = ctx.native_distill_backward(x, tv, ti, sums, vocab=0)
    assert np.all(grad.numpy() == 0)
    values, indices, log_sum = ctx.native_top_logits(x, 2, vocab=0)
    assert np.all(np.isneginf(values.numpy())) and np.all(indices.numpy() == -1) and np.all(np.isneginf(log_sum.numpy()))
    tokens, log_prob = ctx.native_sample(x, ctx.upload(np.zeros(5, np.float32)), vocab=0)
    assert np.all(tokens.numpy() == -1) and np.all(np.isneginf(log_prob.numpy()))


def test_settings_may_change_as_soon_as_a_call_is_back(ctx, pcu_pkg):
    """Small calls end their program in their last launch. The caller then writes the next settings
    from another stream, while a third keeps the chip's units busy, so that workgroups start late: the
    calls' tokens are those of calls that nothing disturbs. Settings change every row's way through the
    launches: the largest logit alone, top-k in one launch and in two, beyond any list, no truncation, a
    nucleus, rows without a logit."""
    rng = np.random.default_rng(21)
    rows, vocab = 64, 20001
    x = rng.normal(0, 2, (rows, vocab)).astype(np.float32)
    x[5] = -np.inf
    x, u = ctx.upload(x), ctx.upload(rng.random(rows).astype(np.float32))
    ones, none = np.ones(rows, np.float32), np.zeros(rows, np.int32)
    mixed = {n: a.numpy() for n, a in _mixed(ctx, rng, rows).items()}
    nucleus = dict(temperature=ones, top_k=none, top_p=0.9 * ones, min_p=0 * ones)
    ways = [dict(nucleus, top_p=ones), nucleus, mixed, dict(nucleus, temperature=0 * ones), nucleus,
            dict(nucleus, top_k=none + 20, top_p=ones), nucleus, dict(nucleus, top_k=none + 900), mixed,
            dict(nucleus, top_k=none + 3000, top_p=ones), nucleus]
    want = [[a.numpy() for a in ctx.native_sample(x, u, **{n: ctx.upload(a) for n, a in w.items()})] for w in ways]
    with pcu_pkg.Context(0) as writer, pcu_pkg.Context(0) as busy:
        settings = {n: ctx.upload(a) for n, a in ways[0].items()}
        theirs = {n: pcu_pkg.DeviceArray(writer, a.ptr, a.shape, a.dtype) for n, a in settings.items()}
        tokens, log_prob = ctx.empty((rows,), np.int32), ctx.empty((rows,), np.float32)
        a = busy.upload(rng.normal(0, 1, (2048, 2048)).astype(np.float32))
        out = busy.empty((2048, 2048), np.float32)
        for _ in range(4):
            with busy.program():
                for _ in range(40):
                    busy.native_matmul(a, a, out=out)
                for w, way in enumerate(ways):
                    for n in theirs:
                        writer.upload_into(theirs[n], way[n])
                    ctx.native_sample(x, u, **settings, tokens=tokens, log_prob=log_prob)
                    for n in theirs:
                        writer.upload_into(theirs[n], ways[(w + 1) % len(ways)][n])
                    np.testing.assert_array_equal(tokens.numpy(), want[w][0])
                    np.testing.assert_array_equal(log_prob.numpy(), want[w][1])


def test_small_calls_results_are_there_for_any_stream(ctx, pcu_pkg):
    """What a call that ends its own program returns is complete for a copy on another stream that
    starts as soon as the call is back: each call's inputs and results differ from the last one's."""
    rng = np.random.default_rng(31)
    rows, vocab, k, calls = 48, 1000, 9, 30
    inputs, want = [], []
    for c in range(calls):
        s, tv, ti, labels = _distill_args(ctx, rng, rows, vocab, k)
        long = rng.normal(0, 2, (rows, 12 * vocab)).astype(np.float32)
        inputs.append([ctx.upload(a) for a in (s, tv, ti, labels, rng.random(rows).astype(np.float32), long)])
    out = {"loss": ctx.empty((rows,), np.float32), "gradient": ctx.empty((rows, vocab), np.float32),
           "values": ctx.empty((rows, k), np.float32), "indices": ctx.empty((rows, k), np.int32),
           "log_sum": ctx.empty((rows,), np.float32), "tokens": ctx.empty((rows,), np.int32),
           "log_prob": ctx.empty((rows,), np.float32)}

    def call(i, read):
        s, tv, ti, labels, u, long = inputs[i]
        got = []
        ctx.native_distill_step(s, tv, ti, labels=labels, temperature=1.7, label_weight=0.4, loss=out["loss"],
                                gradient=out["gradient"])
        got += [read("gradient"), read("loss")]
        ctx.native_top_logits(s, k, values=out["values"], indices=out["indices"], log_sum=out["log_sum"])
        got += [read("values"), read("indices"), read("log_sum")]
        for x in (s, long):
            for kw in (dict(top_k=20), dict(top_p=0.9), dict(min_p=0.1), dict(temperature=0.0)):
                ctx.native_sample(x, u, tokens=out["tokens"], log_prob=out["log_prob"], **kw)
                got += [read("tokens"), read("log_prob")]
        return got

    for i in range(calls):
        want.append(call(i, lambda name: out[name].numpy()))
    with pcu_pkg.Context(0) as reader:
        theirs = {n: pcu_pkg.DeviceArray(reader, a.ptr, a.shape, a.dtype) for n, a in out.items()}
        for i in range(calls):
            for a, b in zip(call(i, lambda name: theirs[name].numpy()), want[i]):
                np.testing.assert_array_equal(a, b)


def test_two_contexts_sample_at_the_same_time(ctx, pcu_pkg):
    """Each context has its own counters and lists: programs of both, open at once, and calls from two
    threads."""
    import threading
    rng = np.random.default_rng(33)
    rows, vocab = 40, 30001
    with pcu_pkg.Context(0) as other:
        both = []
        for c in (ctx, other):
            x = c.upload(rng.normal(0, 2, (rows, vocab)).astype(np.float32))
            u = c.upload(rng.random(rows).astype(np.float32))
            settings = _mixed(c, rng, rows)
            both.append((c, x, u, settings, c.native_sample(x, u, **settings)[0].numpy(),
                         c.native_sample(x, u, top_k=30, top_p=0.9)[0].numpy()))
        with ctx.program(), other.program():
            drawn = [[c.native_sample(x, u, **settings)[0] for c, x, u, settings, _, _ in both] for _ in range(10)]
        for pair in drawn:
            for tokens, (_, _, _, _, want, _) in zip(pair, both):
                np.testing.assert_array_equal(tokens.numpy(), want)
        wrong = []

        def work(c, x, u, settings, want, want_k):
            for _ in range(50):
                if not np.array_equal(c.native_sample(x, u, **settings)[0].numpy(), want) or \
                   not np.array_equal(c.native_sample(x, u, top_k=30, top_p=0.9)[0].numpy(), want_k):
                    wrong.append(c)

        threads = [threading.Thread(target=work, args=a) for a in both]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong
