"""A small language model learns ragged sequences, then continues some of them.

    python examples/train_language_model.py

The model reads one token and answers with the next: its row of the table (``native_embedding``),
layer norm (``native_layer_norm``), and the table again as the output layer
(``native_cross_entropy_step``, which keeps no logits). A training step is one program: loss, the
gradients back to the table, where the output layer's is the base that the read rows' gradients are added to
(``native_embedding_backward``), and the update. Sequences shorter than the batch's length are padded
with token -1, which reads zeros, and label -1, which reaches no loss and no gradient.
"""
import importlib.util
import os
import sys

import numpy as np

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _package():
    """The package from its directory, whose name has a hyphen."""
    if "fusion_pcu_amd" not in sys.modules:
        folder = os.path.join(ROOT, "fusion-pcu_amd")
        spec = importlib.util.spec_from_file_location("fusion_pcu_amd", os.path.join(folder, "__init__.py"),
                                                      submodule_search_locations=[folder])
        sys.modules["fusion_pcu_amd"] = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(sys.modules["fusion_pcu_amd"])
    return sys.modules["fusion_pcu_amd"]


def batch(rng, follow, sequences, length):
    """Ragged sequences in which `follow[token]` comes after a token four times of five: the tokens
    read and the labels, int32 [sequences * length], padding -1."""
    tokens = np.full((sequences, length + 1), -1, np.int32)
    for row in tokens:
        row[0] = rng.integers(len(follow))
        for i in range(1, rng.integers(2, length + 2)):
            row[i] = follow[row[i - 1]] if rng.random() < 0.8 else rng.integers(len(follow))
    read = np.where(tokens[:, 1:] >= 0, tokens[:, :-1], -1)
    return np.ascontiguousarray(read).reshape(-1), np.ascontiguousarray(tokens[:, 1:]).reshape(-1)


def gradients(ctx, model, tokens, labels, row_scale, loss=None):
    """Each row's loss, and the gradients of its sum by `row_scale`, like the `model`."""
    table, weight, bias = model["table"], model["weight"], model["bias"]
    x = ctx.native_embedding(table, tokens)
    y, stats = ctx.native_layer_norm(x, weight, bias)
    loss, change, of_table = ctx.native_cross_entropy_step(y, table, labels, row_scale=row_scale, loss=loss)
    change, of_weight, of_bias = ctx.native_layer_norm_backward(x, stats, change, weight, x_gradient=change)
    ctx.native_embedding_backward(change, tokens, table.shape[0], base=of_table, out=of_table)
    return loss, {"table": of_table, "weight": of_weight, "bias": of_bias}


def train(ctx, model, batches, learning_rate):
    """Updates the `model` in place; each step's mean loss."""
    means = []
    for tokens, labels in batches:
        real = int((labels >= 0).sum())
        scale = ctx.upload(np.full(len(labels), 1.0 / real, np.float32))
        loss = ctx.empty((len(labels),), np.float32)
        read, wanted = ctx.upload(tokens), ctx.upload(labels)
        with ctx.program():
            _, change = gradients(ctx, model, read, wanted, scale, loss)
            for name, values in model.items():
                ctx.native_sgd(values, change[name], learning_rate, out=values)
        means.append(float(loss.numpy().sum(dtype=np.float64) / real))
    return means


def write(ctx, model, first, length, rng):
    """Continues each of the `first` tokens by `length` more: int32 [rows, length + 1]."""
    tokens = [np.asarray(first, np.int32)]
    for _ in range(length):
        uniform = ctx.upload(rng.random(len(first), np.float32))
        y, _ = ctx.native_layer_norm(ctx.native_embedding(model["table"], ctx.upload(tokens[-1])), model["weight"], model["bias"])
        logits = ctx.native_matmul(y, model["table"], transpose_right=True)
        tokens.append(ctx.native_sample(logits, uniform, temperature=0.5, top_k=10)[0].numpy())
    return np.stack(tokens, axis=1)


def start(ctx, rng, vocab, width):
    return {"table": ctx.upload(rng.normal(0, 0.02, (vocab, width)).astype(np.float32)),
            "weight": ctx.upload(np.ones(width, np.float32)), "bias": ctx.upload(np.zeros(width, np.float32))}


def run(ctx, vocab=500, width=96, steps=200, seed=0):
    rng = np.random.default_rng(seed)
    follow = rng.permutation(vocab)
    model = start(ctx, rng, vocab, width)
    losses = train(ctx, model, [batch(rng, follow, 32, 24) for _ in range(steps)], learning_rate=4.0)
    return losses, write(ctx, model, np.arange(4), 12, rng)


def main():
    with _package().Context(0) as ctx:
        losses, text = run(ctx)
    print("mean loss %.4f at first, %.4f after %d steps" % (losses[0], losses[-1], len(losses)))
    for row in text:
        print(" ".join(str(t) for t in row))


if __name__ == "__main__":
    main()
