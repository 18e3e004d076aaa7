"""Performance cases of the operators around a language model's products: embedding lookup with
its gradient, layer norm with its gradients, and the cross entropy of an output layer whose logits
are not kept, with its gradients.

The plain forms are elementary torch operations in 32 bits (64 for binary64 tensors); the
framework's calls take the same tensors. Inputs that a program keeps between calls, and the buffers
that it lends for the results, are made by prepare().
"""
from __future__ import annotations

import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_TORCH = {"f32": torch.float32, "f64": torch.float64, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "f64": 8, "bf16": 2, "f16": 2}
_EPS = 1e-5


# ------------------------------------------------------------------------- cases


def _embed(kind, rows, vocab, width, dtype="f32", scale=1.0, base=False):
    """`rows` tokens. `base`: the gradient is added to one that the table has already (as the
    output layer's weights)."""
    return {"kind": kind, "rows": rows, "vocab": vocab, "width": width, "dtype": dtype, "scale": scale, "base": base}


def _norm(kind, rows, width, dtype="f32", plain=False):
    """`plain`: without weight and bias."""
    return {"kind": kind, "rows": rows, "width": width, "dtype": dtype, "plain": plain}


def _entropy(kind, rows, vocab, width, dtype="f32", pad=0):
    """`pad`: rows of the weights past the vocabulary."""
    return {"kind": kind, "rows": rows, "vocab": vocab, "width": width, "dtype": dtype, "pad": pad}


def listed():
    return [
        # The inputs of a training batch, scaled by sqrt(width).
        dict(_embed("embed", 16384, 128000, 2048, "bf16", math.sqrt(2048.0)), name="embed_bf16_16384_128000x2048"),
        # The table's gradient: a short batch over a long ragged vocabulary, and a long batch
        # whose gradient joins that of an output layer with the same weights.
        dict(_embed("embed_back", 511, 50257, 768), name="embed_back_f32_511_50257x768"),
        dict(_embed("embed_back", 32768, 32000, 2048, "bf16", math.sqrt(2048.0), True),
             name="embed_back_bf16_32768_32000x2048"),
        # A small batch, where latency counts; a long batch; training's backward passes, odd sizes
        # in halves and the largest.
        dict(_norm("norm", 64, 1000), name="norm_f32_64x1000"),
        dict(_norm("norm", 16384, 4096, "bf16"), name="norm_bf16_16384x4096"),
        dict(_norm("norm_back", 1025, 1000, "f16"), name="norm_back_f16_1025x1000"),
        dict(_norm("norm_back", 16384, 4096, "bf16"), name="norm_back_bf16_16384x4096"),
        # Scoring a few positions under a large vocabulary: the weights are read once.
        dict(_entropy("loss", 8, 128000, 4096, "bf16"), name="loss_bf16_8_128000x4096"),
        # The gradients from losses that were evaluated before, odd sizes, a padded vocabulary.
        dict(_entropy("backward", 777, 32003, 1000, "f16", pad=61), name="backward_f16_777_32003x1000"),
        # Training steps of the output layer: a small model's, an ordinary batch, and the largest.
        dict(_entropy("step", 64, 1000, 64), name="step_f32_64_1000x64"),
        dict(_entropy("step", 1024, 50257, 768), name="step_f32_1024_50257x768"),
        dict(_entropy("step", 4096, 128000, 4096, "bf16"), name="step_bf16_4096_128000x4096"),
    ]


def _log_int(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; some of the larger ones whole multiples of 64."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if v >= 128 and rng.random() < 0.5:
        v = (v + 32) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choices(("embed", "embed_back", "norm", "norm_back", "loss", "backward", "step"),
                       weights=(2, 3, 2, 3, 2, 2, 4))[0]
    dtype = rng.choices(("f32", "bf16", "f16", "f64"), weights=(4, 6, 2, 1))[0]
    if kind in ("embed", "embed_back"):
        vocab = _log_int(rng, 100, 262144)
        width = _log_int(rng, 16, min(8192, (1 << 28) // vocab))
        rows = _log_int(rng, 1, min(65536, (1 << 27) // width))
        return _embed(kind, rows, vocab, width, dtype, rng.choice((1.0, math.sqrt(width))),
                      kind == "embed_back" and rng.random() < 0.4)
    if kind in ("norm", "norm_back"):
        width = _log_int(rng, 16, 32768)
        return _norm(kind, _log_int(rng, 1, min(65536, (1 << 26) // width)), width, dtype, rng.random() < 0.2)
    dtype = rng.choices(("f32", "bf16", "f16"), weights=(3, 6, 2))[0]
    width = _log_int(rng, 32, 4096)
    vocab = _log_int(rng, 100, min(262144, (1 << 29) // width))
    rows = _log_int(rng, 1, max(1, min(8192, (4096 * 128000 * 512) // (vocab * width))))
    return _entropy(kind, rows, vocab, width, dtype, rng.choice((0, 0, 0, 47)))


# ------------------------------------------------------------------------- inputs


def _tensors(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 31)
    rows, width, dtype = case["rows"], case["width"], _TORCH[case["dtype"]]

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=gen)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    def tokens(vocab, absent):
        """Text's tokens: the frequency falls with the rank; ranks lie all over the vocabulary."""
        rank = torch.exp(rand(rows) * math.log(vocab + 1.0)).to(torch.int64) - 1
        place = torch.randperm(vocab, device="cuda", generator=gen)
        t = place[rank.clamp(0, vocab - 1)]
        return torch.where(rand(rows) < absent, -1, t).to(torch.int32)

    kind = case["kind"]
    if kind in ("embed", "embed_back"):
        t = {"tokens": tokens(case["vocab"], 0.02)}
        if kind == "embed":
            t["table"] = randn(case["vocab"], width).mul_(0.02).to(dtype)
        else:
            t["gradient"] = randn(rows, width).mul_(1e-3).to(dtype)
            if case["base"]:
                t["base"] = randn(case["vocab"], width).mul_(1e-3).to(dtype)
        return t
    if kind in ("norm", "norm_back"):
        # Activations with a few columns far larger than the rest.
        columns = torch.where(rand(width) < 0.01, 20.0, 1.0)
        t = {"x": (randn(rows, width) * columns + 0.3 * randn(rows, 1)).to(dtype)}
        if not case["plain"]:
            t["weight"] = (1.0 + 0.2 * randn(width)).to(dtype)
            t["bias"] = (0.1 * randn(width)).to(dtype)
        if kind == "norm_back":
            t["gradient"] = randn(rows, width).mul_(0.01).to(dtype)
            x = _wide(t["x"])
            mean = x.mean(1, keepdim=True)
            t["stats"] = torch.cat([mean, torch.rsqrt((x - mean).square().mean(1, keepdim=True) + _EPS)], 1).contiguous()
        return t
    # Features that have their label's weights in them, more or less, so that some labels are
    # likely; rows without a label (padding at the end of sequences).
    vocab = case["vocab"]
    labels = tokens(vocab, 0.05)
    weights = randn(vocab + case["pad"], width).mul_(2.0 / math.sqrt(width)).to(dtype)
    x = randn(rows, width) + 3.0 * rand(rows, 1) * weights[labels.clamp(min=0).long()].float()
    t = {"features": x.to(dtype), "weights": weights, "labels": labels}
    if kind != "loss":
        # The mean over the rows; binary16 gradients carry a loss scale, as a program's do.
        whole = 1024.0 if case["dtype"] == "f16" else 1.0
        t["row_scale"] = torch.full((rows,), whole / rows, device="cuda")
    if kind == "backward":
        sums = []
        for part in t["features"].split(256):
            sums.append(_log_sum(part.float() @ weights[:vocab].float().T).squeeze(1))
        t["log_sum"] = torch.cat(sums).contiguous()
    return t


def prepare(case, seed):
    t = _tensors(case, seed)
    rows, width, dtype = case["rows"], case["width"], _TORCH[case["dtype"]]
    stat = torch.float64 if case["dtype"] == "f64" else torch.float32
    kind = case["kind"]

    def empty(kind, *shape):
        return torch.empty(shape, dtype=kind, device="cuda")

    if kind in ("embed", "norm"):
        out = [empty(dtype, rows, width)] + ([empty(stat, rows, 2)] if kind == "norm" else [])
    elif kind == "embed_back":
        out = [empty(dtype, case["vocab"], width)]
    elif kind == "norm_back":
        out = [empty(dtype, rows, width)] + ([] if case["plain"] else [empty(dtype, width), empty(dtype, width)])
    elif kind == "loss":
        out = [empty(stat, rows), empty(stat, rows)]
    else:
        out = [empty(dtype, rows, width), empty(dtype, case["vocab"] + case["pad"], width)]
        out = ([empty(stat, rows)] if kind == "step" else []) + out
    torch.cuda.synchronize()  # the inputs exist before the framework's own stream reads them
    return {"case": case, "tensors": t, "out": out}


# -------------------------------------------------------------------- the plain forms


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _log_sum(z):
    m = z.amax(1, keepdim=True)
    return m + torch.log(torch.exp(z - m).sum(1, keepdim=True))


def _plain_embed(case, t):
    there = (t["tokens"] >= 0).unsqueeze(1)
    rows = _wide(t["table"][t["tokens"].clamp(min=0).long()]) * case["scale"]
    return [torch.where(there, rows, 0.0).to(t["table"].dtype)]


def _plain_embed_back(case, t):
    g = _wide(t["gradient"]) * case["scale"]
    g = g * (t["tokens"] >= 0).unsqueeze(1)
    table = _wide(t["base"]).clone() if "base" in t else torch.zeros(case["vocab"], case["width"], dtype=g.dtype, device=g.device)
    table.index_add_(0, t["tokens"].clamp(min=0).long(), g)
    return [table.to(t["gradient"].dtype)]


def _plain_norm(case, t):
    x = _wide(t["x"])
    mean = x.mean(1, keepdim=True)
    near = x - mean
    rstd = torch.rsqrt(near.square().mean(1, keepdim=True) + _EPS)
    y = near * rstd
    if "weight" in t:
        y = y * _wide(t["weight"]) + _wide(t["bias"])
    return [y.to(t["x"].dtype), torch.cat([mean, rstd], 1)]


def _plain_norm_back(case, t):
    x, dy = _wide(t["x"]), _wide(t["gradient"])
    mean, rstd = t["stats"][:, :1], t["stats"][:, 1:]
    near = (x - mean) * rstd
    g = dy * _wide(t["weight"]) if "weight" in t else dy
    dx = rstd * (g - g.mean(1, keepdim=True) - near * (g * near).mean(1, keepdim=True))
    out = [dx.to(t["x"].dtype)]
    if "weight" in t:
        out += [(dy * near).sum(0).to(t["x"].dtype), dy.sum(0).to(t["x"].dtype)]
    return out


def _plain_entropy(case, t):
    vocab, kind = case["vocab"], case["kind"]
    x, w = t["features"].float(), t["weights"][:vocab].float()
    z = x @ w.T
    has = (t["labels"] >= 0).unsqueeze(1)
    label = t["labels"].clamp(min=0).long().unsqueeze(1)
    log_sum = t["log_sum"].unsqueeze(1) if kind == "backward" else _log_sum(z)
    out = []
    if kind != "backward":
        out += [torch.where(has, log_sum - torch.gather(z, 1, label), 0.0).squeeze(1)]
    if kind == "loss":
        return out + [log_sum.squeeze(1)]
    scale = t["row_scale"].unsqueeze(1) * has
    g = torch.exp(z - log_sum) * scale
    g.scatter_add_(1, label, -scale)
    dtype = t["features"].dtype
    change = torch.zeros(t["weights"].shape, dtype=dtype, device=x.device)
    change[:vocab] = (g.T @ x).to(dtype)
    return out + [(g @ w).to(dtype), change]


# ------------------------------------------------------------- the framework's calls


def _framework():
    if "fusion_pcu_amd" not in sys.modules:
        # The package's folder name has a hyphen, so it is loaded by its path.
        folder = os.path.join(_ROOT, "fusion-pcu_amd")
        spec = importlib.util.spec_from_file_location(
            "fusion_pcu_amd", os.path.join(folder, "__init__.py"), submodule_search_locations=[folder])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["fusion_pcu_amd"] = mod
        spec.loader.exec_module(mod)
    import fusion_pcu_amd.graph as graph
    return sys.modules["fusion_pcu_amd"], graph.default_context()


def _lend(state):
    """The program's tensors as the framework's arrays, made once for a state."""
    pcu, ctx = _framework()
    dtype = {torch.float32: np.float32, torch.float64: np.float64, torch.float16: np.float16,
             torch.bfloat16: pcu.bfloat16, torch.int32: np.int32}

    def array(x):
        return pcu.DeviceArray(ctx, x.data_ptr(), tuple(x.shape), dtype[x.dtype])

    state["lent"] = ctx, {n: array(x) for n, x in state["tensors"].items()}, [array(x) for x in state["out"]]
    return state["lent"]


def _own(state):
    case = state["case"]
    ctx, t, out = state.get("lent") or _lend(state)
    kind = case["kind"]
    if kind == "embed":
        ctx.native_embedding(t["table"], t["tokens"], scale=case["scale"], out=out[0])
    elif kind == "embed_back":
        ctx.native_embedding_backward(t["gradient"], t["tokens"], case["vocab"], scale=case["scale"],
                                      base=t.get("base"), out=out[0])
    elif kind == "norm":
        ctx.native_layer_norm(t["x"], t.get("weight"), t.get("bias"), eps=_EPS, out=out[0], stats=out[1])
    elif kind == "norm_back":
        changes = {} if case["plain"] else {"weight_gradient": out[1], "bias_gradient": out[2]}
        ctx.native_layer_norm_backward(t["x"], t["stats"], t["gradient"], t.get("weight"), x_gradient=out[0], **changes)
    elif kind == "loss":
        ctx.native_cross_entropy_loss(t["features"], t["weights"], t["labels"], vocab=case["vocab"],
                                      loss=out[0], log_sum=out[1])
    elif kind == "backward":
        ctx.native_cross_entropy_backward(t["features"], t["weights"], t["labels"], t["log_sum"], vocab=case["vocab"],
                                          row_scale=t["row_scale"], feature_gradient=out[0], weight_gradient=out[1])
    else:
        ctx.native_cross_entropy_step(t["features"], t["weights"], t["labels"], vocab=case["vocab"],
                                      row_scale=t["row_scale"], loss=out[0], feature_gradient=out[1],
                                      weight_gradient=out[2])
    return state["out"]


def run(state):
    if own:
        return _own(state)
    plain = {"embed": _plain_embed, "embed_back": _plain_embed_back, "norm": _plain_norm, "norm_back": _plain_norm_back}
    case = state["case"]
    return plain.get(case["kind"], _plain_entropy)(case, state["tensors"])


# ------------------------------------------------------------------ work and exact values


def work(case):
    rows, width, size = case["rows"], case["width"], _SIZE[case["dtype"]]
    stat = 8 if case["dtype"] == "f64" else 4
    kind, n = case["kind"], case["rows"] * case["width"]
    if kind == "embed":  # every row of the table that occurs, once
        return {"bytes": rows * 4 + n * size + min(rows, case["vocab"]) * width * size, "flops": n}
    if kind == "embed_back":
        whole = case["vocab"] * width * size
        return {"bytes": rows * 4 + n * size + whole * (2 if case["base"] else 1), "flops": n}
    if kind == "norm":
        return {"bytes": 2 * n * size + 2 * rows * stat + (0 if case["plain"] else 2 * width * size), "flops": 8 * n}
    if kind == "norm_back":
        return {"bytes": 3 * n * size + 2 * rows * stat + (0 if case["plain"] else 3 * width * size), "flops": 14 * n}
    product = 2.0 * n * case["vocab"]
    read = (n + case["vocab"] * width) * size + 4 * rows
    if kind == "loss":
        return {"bytes": read + 8 * rows, "flops": product}
    written = (n + (case["vocab"] + case["pad"]) * width) * size
    return {"bytes": read + written + 8 * rows, "flops": 3 * product}


def exact(case, seed):
    t = {n: x.double() if x.is_floating_point() and n != "weights" else x for n, x in _tensors(case, seed).items()}
    kind = case["kind"]
    if kind == "embed":
        picked = torch.nn.functional.pad(t["table"], (0, 0, 0, 1)) * case["scale"]  # index -1: the row of zeros
        return [picked[t["tokens"].long()]]
    if kind == "embed_back":
        order = torch.argsort(t["tokens"], stable=True)
        places, counts = torch.unique_consecutive(t["tokens"][order].long(), return_counts=True)
        ends = torch.cumsum(counts, 0)
        out = t["base"].clone() if "base" in t else torch.zeros(case["vocab"], case["width"], dtype=torch.float64, device="cuda")
        for c in range(0, case["width"], 512):
            upto = torch.cumsum(t["gradient"][order, c: c + 512], 0)
            sums = torch.diff(upto[ends - 1], dim=0, prepend=upto.new_zeros(1, upto.shape[1]))
            real = places >= 0
            out[places[real], c: c + 512] += case["scale"] * sums[real]
        return [out]
    if kind in ("norm", "norm_back"):
        x = t["x"]
        mean = x.sum(1, keepdim=True) / x.shape[1]
        if kind == "norm":
            var = torch.var(x, 1, unbiased=False, keepdim=True)
            y = (x - mean) / torch.sqrt(var + _EPS)
            if not case["plain"]:
                y = torch.addcmul(t["bias"], y, t["weight"])
            return [y, torch.cat([mean, 1 / torch.sqrt(var + _EPS)], 1)]
        near = (x - t["stats"][:, :1]) * t["stats"][:, 1:]
        g = t["gradient"] * (1.0 if case["plain"] else t["weight"])
        ones = x.new_full((x.shape[1], 1), 1.0 / x.shape[1])
        dx = t["stats"][:, 1:] * (g - g @ ones - near * ((near * g) @ ones))
        if case["plain"]:
            return [dx]
        return [dx, (near * t["gradient"]).T @ x.new_ones(x.shape[0]), t["gradient"].T @ x.new_ones(x.shape[0])]
    vocab, width, rows = case["vocab"], case["width"], case["rows"]
    has = t["labels"] >= 0
    label = t["labels"].long().clamp(min=0)
    # Two passes over the vocabulary in pieces.
    piece = 16384
    peak = torch.full((rows,), -math.inf, dtype=torch.float64, device="cuda")
    mass = torch.zeros_like(peak)
    if kind == "backward":
        log_sum = t["log_sum"]
    else:
        for v in range(0, vocab, piece):
            z = t["features"] @ t["weights"][v: min(v + piece, vocab)].double().T
            higher = torch.maximum(peak, z.max(1)[0])
            mass = mass * torch.exp(peak - higher) + torch.exp(z - higher[:, None]).sum(1)
            peak = higher
        log_sum = peak + torch.log(mass)
    own_logit = (t["features"] * t["weights"][label].double()).sum(1)
    loss = torch.where(has, log_sum - own_logit, 0.0)
    if kind == "loss":
        return [loss, log_sum]
    scale = torch.where(has, t["row_scale"], 0.0)[:, None]
    dx = torch.zeros(rows, width, dtype=torch.float64, device="cuda")
    dw = torch.zeros(vocab + case["pad"], width, dtype=torch.float64, device="cuda")
    for v in range(0, vocab, piece):
        w = t["weights"][v: min(v + piece, vocab)].double()
        p = torch.exp(t["features"] @ w.T - log_sum[:, None])
        p -= torch.nn.functional.one_hot(torch.where((label >= v) & (label < v + w.shape[0]), label - v, w.shape[0]),
                                         w.shape[0] + 1)[:, :-1]
        p *= scale
        dx += p @ w
        dw[v: v + w.shape[0]] = p.T @ t["features"]
    return ([loss] if kind == "step" else []) + [dx, dw]
