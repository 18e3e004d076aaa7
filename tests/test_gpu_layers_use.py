"""Embedding, layer norm and cross entropy as they are used together: a language model whose table is its
output layer too, in one program and call by call, after faults, from other streams and contexts.

The bounds of the whole chain follow the operators' own (u = 2^-24, U half a step of the rows' type): each
stage takes the error of what it reads through its formula, adds its own roundings and sums, and
rounds what it stores.
"""
import importlib.util
import os
import threading

import numpy as np
import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
u = 2.0 ** -24
U = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
LEAST = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -25}
EPS = 1e-5


@pytest.fixture(scope="module")
def ctx(pcu_pkg):
    c = pcu_pkg.Context(0)
    yield c
    c.close()


def _example(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(ROOT, "examples", name + ".py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _stored(pkg, x, dtype):
    if dtype == "bf16":
        a = pkg.to_bfloat16(x.astype(np.float32))
        return a, pkg.from_bfloat16(a).astype(np.float64)
    a = x.astype({"f32": np.float32, "f16": np.float16}[dtype])
    return a, a.astype(np.float64)


def _values(pkg, a):
    return (pkg.from_bfloat16(a) if a.dtype == pkg.bfloat16 else a).astype(np.float64)


def _mean(x):
    return np.mean(x, axis=1, keepdims=True)


class Chain:
    """The model in 64 bits: each row's loss, the gradients of its sum by `scale`, and what the
    operators' results may be off by (`off`)."""

    def __init__(self, table, weight, bias, tokens, labels, scale, dtype="f32"):
        rows, width, vocab = len(tokens), table.shape[1], table.shape[0]
        has = labels >= 0
        label = np.maximum(labels, 0)
        at = np.arange(rows)

        def store(value, d):  # rounded to the type
            return d + U[dtype] * (np.abs(value) + d) + LEAST[dtype]

        def product(n, magnitude):  # of the matrix cores
            return u * ((6 if dtype == "f32" else 1) * n / 2 + 67) * magnitude

        x = np.where(tokens[:, None] >= 0, table[np.maximum(tokens, 0)], 0.0)
        m = _mean(x)
        square = _mean((x - m) ** 2)
        r = 1 / np.sqrt(square + np.float64(np.float32(EPS)))
        near = (x - m) * r
        y = near * weight + bias
        sums = u * (width / 16 + 64)
        d_m = (sums + 2 * u) * _mean(np.abs(x))
        d_diff = d_m + u * (np.abs(x) + np.abs(m))
        d_square = _mean(2 * np.abs(x - m) * d_diff + d_diff ** 2)
        d_square = d_square + (sums + 3 * u) * (square + d_square)
        d_r = r * (d_square * r ** 2 / 2 * 1.1 + 4 * u)
        d_near = d_diff * (r + d_r) + np.abs(x - m) * d_r + 3 * u * r * (np.abs(x) + np.abs(m))
        d_y = store(y, d_near * np.abs(weight) + 3 * u * (np.abs(near * weight) + np.abs(bias)))

        l = y @ table.T
        d_l = d_y @ np.abs(table).T
        d_l = d_l + product(width, (np.abs(y) + d_y) @ np.abs(table).T)
        top = l.max(axis=1, keepdims=True)
        log_sum = top + np.log(np.exp(l - top).sum(axis=1, keepdims=True))
        d_log_sum = d_l.max(axis=1, keepdims=True) + u * (16 * np.abs(l).max(axis=1, keepdims=True) + vocab / 16 + 128)
        self.loss = np.where(has, log_sum[:, 0] - l[at, label], 0.0)
        off_loss = np.where(has, d_log_sum[:, 0] + d_l[at, label] + u * np.abs(self.loss), 0.0)

        s = np.where(has, scale, 0.0)[:, None]
        p = np.exp(l - log_sum)
        g = p.copy()
        g[at, label] -= 1.0
        d_g = p * np.expm1(d_l + d_log_sum + u * (8 * np.abs(l) + 8))
        least = np.abs(s).max() * (2.0 ** -39 if dtype == "f16" else 0.0)
        d_g = np.where(has[:, None], np.abs(s) * (d_g + (U[dtype] + 2 * u) * (np.abs(g) + d_g)) + least, 0.0)
        g = s * g
        size = np.abs(g) + d_g
        dy = g @ table
        d_dy = store(dy, d_g @ np.abs(table) + product(vocab, size @ np.abs(table)))
        of_table = g.T @ y
        d_table = store(of_table, d_g.T @ np.abs(y) + size.T @ d_y + product(rows, size.T @ (np.abs(y) + d_y)))

        h = dy * weight
        d_h = d_dy * np.abs(weight) + u * np.abs(h)
        c0, c1 = _mean(h), _mean(h * near)
        d_c0 = _mean(d_h) + (sums + 3 * u) * _mean(np.abs(h) + d_h)
        d_c1 = _mean(d_h * (np.abs(near) + d_near) + np.abs(h) * d_near)
        d_c1 = d_c1 + (sums + 4 * u) * _mean((np.abs(h) + d_h) * (np.abs(near) + d_near))
        dx = r * (h - c0 - near * c1)
        inner = d_h + d_c0 + d_near * (np.abs(c1) + d_c1) + np.abs(near) * d_c1
        whole = np.abs(h) + np.abs(c0) + np.abs(near * c1) + inner
        d_dx = store(dx, d_r * whole + (r + d_r) * (inner + 5 * u * whole))
        down = u * (rows + 64) + 3 * u
        of_weight, of_bias = np.sum(dy * near, 0), np.sum(dy, 0)
        d_weight = np.sum(d_dy * (np.abs(near) + d_near) + np.abs(dy) * d_near, 0)
        d_weight = store(of_weight, d_weight + down * np.sum((np.abs(dy) + d_dy) * (np.abs(near) + d_near), 0))
        d_bias = store(of_bias, np.sum(d_dy, 0) + down * np.sum(np.abs(dy) + d_dy, 0))

        of_table = of_table.copy()
        magnitude = np.abs(of_table) + d_table
        read = tokens >= 0
        np.add.at(of_table, tokens[read], dx[read])
        np.add.at(d_table, tokens[read], d_dx[read])
        np.add.at(magnitude, tokens[read], np.abs(dx[read]) + d_dx[read])
        d_table = store(of_table, d_table + u * (rows + 4) * magnitude)
        self.gradients = {"table": of_table, "weight": of_weight, "bias": of_bias}
        self.off = {"loss": off_loss, "table": d_table, "weight": d_weight, "bias": d_bias}

    def check(self, loss, gradients):
        for name, got, want in [("loss", loss, self.loss)] + [(n, gradients[n], self.gradients[n]) for n in self.gradients]:
            off = np.abs(got - want)
            assert np.all(off <= self.off[name]), (name, float(np.max(off / np.maximum(self.off[name], 1e-300))))


def _inputs(rng, vocab, width, rows):
    """A token that most rows read, tokens that none does, padding at the ends of sequences of 20."""
    table, weight, bias = rng.normal(0, width ** -0.5, (vocab, width)), rng.normal(1, 0.2, width), rng.normal(0, 0.2, width)
    tokens = np.where(rng.random(rows) < 0.3, 7 % vocab, rng.integers(0, max(vocab * 2 // 3, 1), rows)).astype(np.int32)
    labels = rng.integers(0, vocab, rows).astype(np.int32)
    padding = np.arange(rows) % 20 >= 17
    tokens[padding] = labels[padding] = -1
    return table, weight, bias, tokens, labels


def test_the_chain_is_its_differences():
    """The 64-bit model against central differences of its loss: off by h^2 / 6 of the third derivative and 2^-52 / h
    of the loss, both below 1e-8 of the sums here."""
    rng = np.random.default_rng(1)
    table, weight, bias, tokens, labels = _inputs(rng, 13, 9, 40)
    scale = rng.random(40)
    exact = Chain(table, weight, bias, tokens, labels, scale)
    values = {"table": table, "weight": weight, "bias": bias}
    for name in values:
        for _ in range(5):
            way = rng.normal(0, 1, values[name].shape)
            h, loss = 1e-5, []
            for sign in (1, -1):
                moved = dict(values, **{name: values[name] + sign * h * way})
                loss.append(np.sum(scale * Chain(moved["table"], moved["weight"], moved["bias"], tokens, labels, scale).loss))
            want = np.sum(exact.gradients[name] * way)
            assert abs((loss[0] - loss[1]) / (2 * h) - want) <= 1e-6 * np.sum(np.abs(exact.gradients[name] * way))


# One row; few rows, whose calls end their own programs; many, through the sorted gradient and the larger tiles.
SIZES = [(1, 1, 1), (1, 500, 96), (3, 40, 7), (60, 1000, 64), (700, 333, 100), (1500, 4100, 129)]


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,vocab,width", SIZES)
@pytest.mark.parametrize("program", [False, True])
def test_a_training_steps_gradients(ctx, pcu_pkg, rows, vocab, width, dtype, program):
    example = _example("train_language_model")
    rng = np.random.default_rng(rows + width)
    table, weight, bias, tokens, labels = _inputs(rng, vocab, width, rows)
    held = {n: _stored(pcu_pkg, v, dtype) for n, v in (("table", table), ("weight", weight), ("bias", bias))}
    scale = np.full(rows, 2.0 ** -6, np.float32)
    exact = Chain(*(held[n][1] for n in ("table", "weight", "bias")), tokens, labels, scale.astype(np.float64), dtype)
    model = {n: ctx.upload(a) for n, (a, _) in held.items()}
    args = [ctx.upload(a) for a in (tokens, labels, scale)]
    if program:
        with ctx.program():
            loss, grads = example.gradients(ctx, model, *args)
    else:
        loss, grads = example.gradients(ctx, model, *args)
    exact.check(loss.numpy().astype(np.float64), {n: _values(pcu_pkg, a.numpy()) for n, a in grads.items()})


def test_the_example_trains_and_writes(ctx):
    example = _example("train_language_model")
    losses, text = example.run(ctx, steps=40)
    assert len(losses) == 40 and np.all(np.isfinite(losses))
    assert text.shape == (4, 13) and np.all((text >= 0) & (text < 500))
    again, same = example.run(ctx, steps=40)
    assert losses == again and np.array_equal(text, same)


def test_the_example_changes_its_model_by_the_gradients(ctx):
    """A step: the values less the learning rate's multiple of the gradients, rounded at each operation."""
    example = _example("train_language_model")
    rng = np.random.default_rng(5)
    model = example.start(ctx, rng, 200, 48)
    before = {n: a.numpy() for n, a in model.items()}
    tokens, labels = example.batch(rng, rng.permutation(200), 8, 20)
    assert np.any(labels < 0) and np.array_equal(tokens < 0, labels < 0)
    real = int((labels >= 0).sum())
    scale = np.full(len(labels), 1.0 / real, np.float32)
    exact = Chain(*(before[n].astype(np.float64) for n in ("table", "weight", "bias")), tokens, labels, scale.astype(np.float64))
    means = example.train(ctx, model, [(tokens, labels)], 0.25)
    assert abs(means[0] - exact.loss.sum() / real) <= exact.off["loss"].sum() / real + 2.0 ** -50 * exact.loss.sum()
    for n, a in model.items():
        change = 0.25 * exact.gradients[n]
        bound = 0.25 * exact.off[n] + u * (2 * np.abs(change) + np.abs(before[n]) + exact.off[n])
        assert np.all(np.abs(a.numpy() - (before[n] - change)) <= bound + u * np.abs(before[n])), n


@pytest.mark.parametrize("rows,vocab,width", [(40, 300, 32), (900, 2000, 100)])
def test_a_fault_leaves_later_stages_out(ctx, pcu_pkg, rows, vocab, width):
    """A token out of range in the first node: what later nodes write keeps its bits, and the next step is
    right again."""
    example = _example("train_language_model")
    rng = np.random.default_rng(rows)
    table, weight, bias, tokens, labels = _inputs(rng, vocab, width, rows)
    model = {n: ctx.upload(v.astype(np.float32)) for n, v in (("table", table), ("weight", weight), ("bias", bias))}
    scale, good, wanted = ctx.upload(np.full(rows, 0.5, np.float32)), ctx.upload(tokens), ctx.upload(labels)
    loss, grads = example.gradients(ctx, model, good, wanted, scale)
    want = [loss.numpy()] + [grads[n].numpy() for n in model]
    wrong = tokens.copy()
    wrong[23], wrong[31] = vocab, vocab + 5
    wrong = ctx.upload(wrong)
    kept = np.full(rows, 7.0, np.float32)
    out = {"loss": ctx.upload(kept), "log_sum": ctx.upload(kept)}
    mark = ctx.upload(np.full((rows, width), 3.0, np.float32))
    marks = {n: ctx.upload(np.full(a.shape, 5.0, np.float32)) for n, a in model.items()}
    with pytest.raises(pcu_pkg.PcuExecutionError) as e:
        with ctx.program():
            x = ctx.native_embedding(model["table"], wrong)
            y, stats = ctx.native_layer_norm(x, model["weight"], model["bias"], out=mark)
            ctx.native_cross_entropy_loss(y, model["table"], wanted, **out)
            dx, _, _ = ctx.native_layer_norm_backward(x, stats, x, model["weight"], weight_gradient=marks["weight"],
                                                      bias_gradient=marks["bias"])
            ctx.native_embedding_backward(dx, good, vocab, out=marks["table"])
    assert e.value.tensor_fault.element_index == 23
    assert np.all(out["loss"].numpy() == 7) and np.all(out["log_sum"].numpy() == 7) and np.all(mark.numpy() == 3)
    assert all(np.all(a.numpy() == 5) for a in marks.values())
    for _ in range(2):
        loss, grads = example.gradients(ctx, model, good, wanted, scale)
        for a, b in zip([loss] + [grads[n] for n in model], want):
            np.testing.assert_array_equal(a.numpy(), b)


def _calls(ctx, rng, rows, vocab, width):
    """Arrays of a small model on `ctx` and a function that runs every operator into the same
    outputs, handing each call's to `read`."""
    table, weight, bias, tokens, labels = _inputs(rng, vocab, width, rows)
    t, w, b = (ctx.upload(v.astype(np.float32)) for v in (table, weight, bias))
    tokens, labels = ctx.upload(tokens), ctx.upload(labels)
    up = ctx.upload(rng.normal(0, 1, (rows, width)).astype(np.float32))
    return t, w, b, tokens, labels, up


def _outputs(ctx, rows, vocab, width):
    shapes = {"x": (rows, width), "y": (rows, width), "stats": (rows, 2), "dx": (rows, width), "dw": (width,), "db": (width,),
              "loss": (rows,), "log_sum": (rows,), "dy": (rows, width), "dt": (vocab, width), "de": (vocab, width)}
    return {n: ctx.empty(s, np.float32) for n, s in shapes.items()}


def _run(ctx, inputs, o, read):
    t, w, b, tokens, labels, up = inputs
    got = []
    ctx.native_embedding(t, tokens, out=o["x"])
    got += [read("x")]
    ctx.native_layer_norm(o["x"], w, b, out=o["y"], stats=o["stats"])
    got += [read("y"), read("stats")]
    ctx.native_cross_entropy_loss(o["y"], t, labels, loss=o["loss"], log_sum=o["log_sum"])
    got += [read("loss"), read("log_sum")]
    ctx.native_cross_entropy_backward(o["y"], t, labels, o["log_sum"], feature_gradient=o["dy"], weight_gradient=o["dt"])
    got += [read("dt"), read("dy")]
    ctx.native_cross_entropy_step(o["y"], t, labels, loss=o["loss"], feature_gradient=o["dy"], weight_gradient=o["dt"])
    got += [read("dy"), read("loss"), read("dt")]
    ctx.native_layer_norm_backward(o["x"], o["stats"], up, w, x_gradient=o["dx"], weight_gradient=o["dw"], bias_gradient=o["db"])
    got += [read("db"), read("dw"), read("dx")]
    ctx.native_embedding_backward(up, tokens, t.shape[0], out=o["de"])
    return got + [read("de")]


@pytest.mark.parametrize("rows,vocab,width", [(1, 50, 16), (30, 200, 40), (64, 1000, 64), (300, 4000, 129)])
def test_results_are_there_for_any_stream(ctx, pcu_pkg, rows, vocab, width):
    """What a call returns, small ones that end their own program too, is complete for a copy on another
    stream that starts as soon as the call is back: inputs and results differ from call to call."""
    rng = np.random.default_rng(rows)
    inputs = [_calls(ctx, rng, rows, vocab, width) for _ in range(8)]
    o = _outputs(ctx, rows, vocab, width)
    want = [_run(ctx, i, o, lambda n: o[n].numpy()) for i in inputs]
    with pcu_pkg.Context(0) as reader:
        theirs = {n: pcu_pkg.DeviceArray(reader, a.ptr, a.shape, a.dtype) for n, a in o.items()}
        for _ in range(3):
            for i, w in zip(inputs, want):
                for a, b in zip(_run(ctx, i, o, lambda n: theirs[n].numpy()), w):
                    np.testing.assert_array_equal(a, b)


def test_two_contexts_at_the_same_time(ctx, pcu_pkg):
    """Each context has its own scratch: programs of both, open at once, and calls from two threads."""
    rng = np.random.default_rng(3)
    rows, vocab, width = 500, 3000, 70
    with pcu_pkg.Context(0) as other:
        both = []
        for c in (ctx, other):
            inputs = _calls(c, rng, rows, vocab, width)
            o = _outputs(c, rows, vocab, width)
            both.append((c, inputs, o, _run(c, inputs, o, lambda n, o=o: o[n].numpy())))
        last = ["y", "loss", "dt", "dx", "de"]
        want = [{n: o[n].numpy() for n in last} for _, _, o, _ in both]
        with ctx.program(), other.program():
            for _ in range(3):
                for c, inputs, o, _ in both:
                    _run(c, inputs, o, lambda n: None)
        for (c, _, o, _), w in zip(both, want):
            for n in last:
                np.testing.assert_array_equal(o[n].numpy(), w[n])
        wrong = []

        def work(c, inputs, o, want):
            for _ in range(10):
                for a, b in zip(_run(c, inputs, o, lambda n: o[n].numpy()), want):
                    if not np.array_equal(a, b):
                        wrong.append(c)

        threads = [threading.Thread(target=work, args=a) for a in both]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not wrong


def test_their_kernels_have_their_times(ctx):
    """The profile counts each operator's calls under its own name."""
    rng = np.random.default_rng(4)
    inputs, o = _calls(ctx, rng, 20, 100, 24), _outputs(ctx, 20, 100, 24)
    ctx.profile(True)
    try:
        _run(ctx, inputs, o, lambda n: None)
        times = {n: ctx.kernel_time(n) for n in ("embedding", "layer_norm", "cross_entropy")}
    finally:
        ctx.profile(False)
    assert [times[n][1] for n in ("embedding", "layer_norm", "cross_entropy")] == [2, 2, 3]
    assert all(t[0] > 0 for t in times.values())
