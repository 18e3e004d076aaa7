"""A small next-token student learns from a larger teacher's stored top logits, then writes text.

    python examples/distill_and_sample.py

The teacher's output layer is run once over every context and only its top logits are kept
(``native_top_logits``). A training step is one program: the student's logits, the loss with its
gradient (``native_distill_step``), the weights' gradient and their update. Afterwards the student
continues a batch of sequences, one token a row and step (``native_embedding``, ``native_sample``).
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


def teach(ctx, features, weights, k, temperature):
    """The teacher's top logits, their indices and its log-sum-exp for every context."""
    return ctx.native_top_logits(ctx.native_matmul(features, weights), k, temperature=temperature)


def train(ctx, features, weights, teacher, labels, steps, learning_rate, temperature):
    """Updates `weights` in place; each step's mean loss."""
    values, indices, log_sum = teacher
    rows = features.shape[0]
    scale = ctx.upload(np.full(rows, 1.0 / rows, np.float32))
    logits = ctx.empty((rows, weights.shape[1]), np.float32)
    loss, change = ctx.empty((rows,), np.float32), ctx.empty(weights.shape, np.float32)
    means = []
    for _ in range(steps):
        with ctx.program():
            ctx.native_matmul(features, weights, out=logits)
            # The gradient takes the logits' place.
            ctx.native_distill_step(logits, values, indices, log_sum, labels=labels, temperature=temperature,
                                    label_weight=0.1, row_scale=scale, loss=loss, gradient=logits)
            ctx.native_matmul(features, logits, transpose_left=True, out=change)
            ctx.native_sgd(weights, change, learning_rate, out=weights)
        means.append(float(loss.numpy().mean()))
    return means


def write(ctx, table, weights, first, length, rng):
    """Continues each of the `first` tokens by `length` more: int32 [rows, length + 1]."""
    tokens = [np.asarray(first, np.int32)]
    features, uniform = ctx.empty((len(first), table.shape[1]), np.float32), ctx.empty((len(first),), np.float32)
    for _ in range(length):
        ctx.native_embedding(table, ctx.upload(tokens[-1]), out=features)
        ctx.upload_into(uniform, rng.random(len(first), np.float32))
        logits = ctx.native_matmul(features, weights)
        tokens.append(ctx.native_sample(logits, uniform, temperature=0.8, top_k=40, top_p=0.95, min_p=0.01)[0].numpy())
    return np.stack(tokens, axis=1)


def run(ctx, vocab=1000, steps=60, seed=0):
    rng = np.random.default_rng(seed)
    table = rng.normal(0, 1, (vocab, 64)).astype(np.float32)
    teacher_weights = rng.normal(0, 0.35, (64, vocab)).astype(np.float32)
    contexts = ctx.upload(table)
    teacher = teach(ctx, contexts, ctx.upload(teacher_weights), k=32, temperature=2.0)
    labels = ctx.upload(teacher[1].numpy()[:, 0].copy())  # the teacher's first choice
    student_table = np.ascontiguousarray(table[:, :48])   # the student sees less
    weights = ctx.upload(np.zeros((48, vocab), np.float32))
    student = ctx.upload(student_table)
    losses = train(ctx, student, weights, teacher, labels, steps, learning_rate=20.0, temperature=2.0)
    return losses, write(ctx, student, weights, np.arange(4), 12, rng)


def main():
    with _package().Context(0) as ctx:
        losses, text = run(ctx)
    print("mean loss %.4f at first, %.4f after %d steps" % (losses[0], losses[-1], len(losses)))
    for row in text:
        print(" ".join(str(t) for t in row))


if __name__ == "__main__":
    main()
