"""Performance cases of the operators on logits: a teacher's top logits, the distillation
loss with its gradient, and the sampling of tokens.

A case is one call on `rows` rows of `vocab` logits that lie on the GPU. The plain forms are
elementary torch operations in 32 bits (64 for binary64 logits); the framework's calls take
the same tensors. Inputs that a program keeps between calls, and the buffers that it lends
for the results, are made by prepare().
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
_ONE = 1 << 40  # the weight of a row's largest logit in the sampler's integers
_UNIT = 1 << 31  # the fixed point of the sampler's probabilities and random numbers


# ------------------------------------------------------------------------- cases


def _top(rows, vocab, k, dtype="f32", temperature=1.0):
    return {"kind": "top", "rows": rows, "vocab": vocab, "cols": vocab, "k": k, "dtype": dtype,
            "temperature": temperature}


def _distill(kind, rows, vocab, k, dtype="f32", temperature=2.0, full=False, label=0.0, pad=0):
    """`full`: the teacher's log-sum-exp of the whole row comes with its entries. `label`: the
    weight of the hard label's cross entropy (0: no labels). `pad`: columns past the vocabulary."""
    return {"kind": kind, "rows": rows, "vocab": vocab, "cols": vocab + pad, "k": k, "dtype": dtype,
            "temperature": temperature, "full": full, "label": label}


def _sample(rows, vocab, dtype="f32", temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, mixed=False):
    """`mixed`: each row has settings of its own (serving requests batched together)."""
    return {"kind": "sample", "rows": rows, "vocab": vocab, "cols": vocab, "dtype": dtype,
            "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "mixed": mixed}


def listed():
    return [
        # A small teacher's outputs for one batch of an output layer: latency counts.
        dict(_top(64, 1000, 8), name="top_f32_64x1000_k8"),
        # Storing a teacher's targets for a training batch, whole and ragged vocabularies.
        dict(_top(2048, 32000, 64, "bf16"), name="top_bf16_2048x32000_k64"),
        dict(_top(511, 50257, 500, temperature=2.0), name="top_f32_511x50257_k500"),
        # Evaluating a student on held-out rows (loss only).
        dict(_distill("loss", 512, 32000, 32, label=0.3), name="loss_f32_512x32000_k32"),
        # The gradient from a loss that was evaluated before, on a padded vocabulary.
        dict(_distill("backward", 1025, 50257, 100, "f16", full=True, pad=47), name="backward_f16_1025x50257_k100"),
        # Training steps' loss and gradient at once: a small binary64 layer, a few rows of a
        # long vocabulary, an ordinary batch, and the largest.
        dict(_distill("step", 64, 1000, 16, "f64", label=0.5), name="step_f64_64x1000_k16"),
        dict(_distill("step", 16, 200001, 50), name="step_f32_16x200001_k50"),
        dict(_distill("step", 4096, 128000, 64, "bf16", temperature=1.0, label=0.2), name="step_bf16_4096x128000_k64"),
        # One request's next token.
        dict(_sample(1, 128000, "bf16", 0.7, top_k=50, top_p=0.9), name="sample_bf16_1x128000_k50_p90"),
        # A batch with a nucleus alone, a batch with no truncation but min-p, and a batch of
        # requests that each have settings of their own.
        dict(_sample(64, 50257, "f32", 0.9, top_p=0.95), name="sample_f32_64x50257_p95"),
        dict(_sample(32, 32000, "f32", 1.2, min_p=0.05), name="sample_f32_32x32000_min5"),
        dict(_sample(512, 152000, "bf16", mixed=True), name="sample_bf16_512x152000_mixed"),
    ]


def _log_int(rng, lo, hi):
    """A size spread over the logarithm of [lo, hi]; some of the larger ones whole multiples of 64."""
    v = int(round(lo * (hi / lo) ** rng.random()))
    if v >= 512 and rng.random() < 0.4:
        v = (v + 32) // 64 * 64
    return max(lo, min(hi, v))


def draw(rng):
    kind = rng.choices(("top", "loss", "backward", "step", "sample"), weights=(3, 1, 2, 3, 5))[0]
    dtype = rng.choices(("f32", "bf16", "f16", "f64"), weights=(5, 5, 1, 1))[0]
    vocab = _log_int(rng, 100, 262144)
    most = (4096 * 128000 * 2) // _SIZE[dtype] // (2 if kind == "sample" else 1)
    rows = _log_int(rng, 1, max(1, min(512 if kind == "sample" else 4096, most // (vocab + 64))))
    temperature = rng.choice((0.6, 0.8, 1.0, 1.0, 1.5, 2.0, 4.0))
    if kind == "top":
        return _top(rows, vocab, _log_int(rng, 1, min(1024, vocab)), dtype, temperature)
    if kind != "sample":
        return _distill(kind, rows, vocab, _log_int(rng, 1, min(512, vocab)), dtype, temperature,
                        rng.random() < 0.4, rng.choice((0.0, 0.1, 0.5)), rng.choice((0, 0, 1, 64)))
    how = rng.choice(("k", "p", "kp", "min", "all", "none", "mixed", "mixed"))
    return _sample(rows, vocab, dtype, rng.choice((0.5, 0.7, 0.9, 1.0, 1.3)),
                   _log_int(rng, 1, min(1000, vocab)) if how in ("k", "kp", "all") else 0,
                   rng.uniform(0.3, 0.99) if how in ("p", "kp", "all") else 1.0,
                   rng.uniform(0.01, 0.2) if how in ("min", "all") else 0.0, how == "mixed")


# ------------------------------------------------------------------------- inputs


def _log_sum(z):
    m = z.amax(1, keepdim=True)
    return m + torch.log(torch.exp(z - m).sum(1, keepdim=True))


def _tensors(case, seed):
    """Seeded inputs. Logits have the long tail of a language model's: minus a power law of a
    random rank, sharper in some rows than in others, with noise on top."""
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 29)
    rows, vocab, cols = case["rows"], case["vocab"], case["cols"]
    dtype = _TORCH[case["dtype"]]

    def rand(*shape):
        return torch.rand(shape, device="cuda", generator=gen)

    def randn(*shape):
        return torch.randn(shape, device="cuda", generator=gen)

    tail = torch.log1p(rand(rows, cols).mul_(vocab))
    t = {"logits": (randn(rows, cols).mul_(0.5).sub_(tail * (0.8 + 1.2 * rand(rows, 1))).add_(4.0)).to(dtype)}
    if case["kind"] == "sample":
        t["uniform"] = rand(rows)
        # Tokens that a grammar or a user rules out.
        t["logits"].masked_fill_(rand(rows, cols) < 0.02, -math.inf)
        if case["mixed"]:
            pick = rand(4, rows)
            t["temperature"] = torch.where(pick[0] < 0.1, torch.zeros_like(pick[0]), 0.5 + pick[0])
            t["top_k"] = torch.where(pick[1] < 0.6, (pick[1] * 300).to(torch.int32) + 1, 0).to(torch.int32)
            t["top_p"] = torch.where(pick[2] < 0.6, 0.4 + pick[2], torch.ones_like(pick[2]))
            t["min_p"] = torch.where(pick[3] < 0.3, 0.3 * pick[3], torch.zeros_like(pick[3]))
        return t
    if case["kind"] == "top":
        return t
    # A teacher that agrees with the student in part, its entries, and rows that carry nothing
    # (padding at the end of sequences).
    stat = torch.float64 if case["dtype"] == "f64" else torch.float32
    teacher = t["logits"][:, :vocab].to(stat).mul(0.7).sub_(0.3 * torch.log1p(rand(rows, vocab).mul_(vocab)).to(stat))
    values, indices = torch.topk(teacher, case["k"], dim=1)
    empty = (rand(rows) < 0.05).unsqueeze(1)
    t["values"] = values.to(dtype).contiguous()
    t["indices"] = torch.where(empty, -1, indices).to(torch.int32).contiguous()
    if case["full"]:
        t["teacher_log_sum"] = _log_sum(teacher / case["temperature"]).squeeze(1).contiguous()
    del teacher
    if case["label"]:
        labels = torch.where(rand(rows) < 0.7, indices[:, 0], (rand(rows) * (vocab - 1)).to(torch.int64))
        t["labels"] = torch.where(empty.squeeze(1), -1, labels).to(torch.int32)
    if case["kind"] != "loss":
        # The mean over the rows; binary16 gradients carry a loss scale, as a program's do.
        whole = 1024.0 if case["dtype"] == "f16" else 1.0
        t["row_scale"] = ((~empty.squeeze(1)).to(stat) * (whole / max(1, rows))).contiguous()
    if case["kind"] == "backward":
        s = t["logits"][:, :vocab].to(stat)
        t["log_sums"] = torch.cat([_log_sum(s / case["temperature"]), _log_sum(s)], 1).contiguous()
    return t


def prepare(case, seed):
    t = _tensors(case, seed)
    rows, dtype = case["rows"], _TORCH[case["dtype"]]
    stat = torch.float64 if case["dtype"] == "f64" else torch.float32

    def empty(kind, *shape):
        return torch.empty(shape, dtype=kind, device="cuda")

    if case["kind"] == "top":
        out = [empty(dtype, rows, case["k"]), empty(torch.int32, rows, case["k"]), empty(stat, rows)]
    elif case["kind"] == "loss":
        out = [empty(stat, rows), empty(stat, rows, 2)]
    elif case["kind"] == "backward":
        out = [empty(dtype, rows, case["cols"])]
    elif case["kind"] == "step":
        out = [empty(stat, rows), empty(dtype, rows, case["cols"])]
    else:
        out = [empty(torch.int32, rows), empty(torch.float32, rows)]
    torch.cuda.synchronize()  # the inputs exist before the framework's own stream reads them
    return {"case": case, "tensors": t, "out": out}


# -------------------------------------------------------------------- the plain forms


def _wide(x):
    return x if x.dtype == torch.float64 else x.float()


def _plain_top(case, t):
    x = _wide(t["logits"])
    values, indices = torch.sort(x, dim=1, descending=True, stable=True)
    k = case["k"]
    return [values[:, :k].to(t["logits"].dtype), indices[:, :k].to(torch.int32),
            _log_sum(x / case["temperature"]).squeeze(1)]


def _teacher(case, t):
    """The teacher's probabilities (0 for absent entries), their logarithms and places."""
    there = t["indices"] >= 0
    z = _wide(t["values"]) / case["temperature"]
    z = torch.where(there, z, -math.inf)
    if "teacher_log_sum" in t:
        log_sum = t["teacher_log_sum"].unsqueeze(1)
    else:
        m = z.amax(1, keepdim=True)
        m = torch.where(m == -math.inf, torch.zeros_like(m), m)
        log_sum = m + torch.log(torch.exp(z - m).sum(1, keepdim=True))
    log_q = torch.where(there, z - log_sum, -math.inf)
    return torch.exp(log_q), log_q, torch.where(there, t["indices"], 0).long()


def _plain_distill(case, t, forward, backward):
    s = _wide(t["logits"][:, : case["vocab"]])
    tau, b = case["temperature"], case["label"]
    a = 1.0 - b
    q, log_q, at = _teacher(case, t)
    labelled = "labels" in t
    if "log_sums" in t:
        log_sum, log_sum1 = t["log_sums"][:, :1], t["log_sums"][:, 1:]
    else:
        log_sum = _log_sum(s / tau)
        log_sum1 = _log_sum(s) if (labelled or case["kind"] == "loss") and tau != 1.0 else log_sum
    out = []
    if labelled:
        has = (t["labels"] >= 0).unsqueeze(1)
        label = torch.where(has, t["labels"].unsqueeze(1), 0).long()
    if forward:
        log_p = torch.gather(s, 1, at) / tau - log_sum
        loss = a * tau * tau * torch.where(q > 0, q * (log_q - log_p), torch.zeros_like(q)).sum(1)
        if labelled:
            loss = loss + b * torch.where(has, log_sum1 - torch.gather(s, 1, label), 0.0).squeeze(1)
        out += [loss]
        if not backward:
            out += [torch.cat([log_sum, log_sum1], 1)]
    if backward:
        scale = t["row_scale"].unsqueeze(1)
        g = torch.zeros(case["rows"], case["cols"], dtype=s.dtype, device=s.device)
        inner = g[:, : case["vocab"]]
        inner += torch.exp(s / tau - log_sum) * (a * tau * q.sum(1, keepdim=True) * scale)
        inner.scatter_add_(1, at, q * (-a * tau * scale))
        if labelled:
            inner += torch.exp(s - log_sum1) * (b * has * scale)
            inner.scatter_add_(1, label, -b * has * scale)
        out += [g.to(t["logits"].dtype)]
    return out


def _mul_shift(mass, part):
    """floor(mass * part / 2^31) for masses below 2^62 and parts of up to 31 bits."""
    return ((mass >> 32) * part * 2) + (((mass & 0xFFFFFFFF) * part) >> 31)


def _settings(case, t):
    """The rows' settings as columns."""
    rows = case["rows"]

    def column(name, dtype):
        if name in t:
            return t[name].unsqueeze(1)
        return torch.full((rows, 1), case[name], dtype=dtype, device="cuda")

    return [column("temperature", torch.float32), column("top_k", torch.int32),
            column("top_p", torch.float32), column("min_p", torch.float32)]


def _plain_sample(case, t):
    x = _wide(t["logits"])
    temperature, top_k, top_p, min_p = _settings(case, t)
    m = x.amax(1, keepdim=True)
    inverse = 1.0 / temperature
    greedy = torch.isinf(inverse)
    z = (x - m).float() * torch.where(greedy, torch.ones_like(inverse), inverse)
    w = torch.where(x == m, _ONE, (torch.exp(z) * float(_ONE)).to(torch.int64))
    keep = w >= torch.ceil(min_p.double() * _ONE).to(torch.int64)
    if case["mixed"] or case["top_k"] or case["top_p"] < 1.0:
        # In the order of the logits: the first top_k, then the shortest prefix with top_p of
        # their mass; back in the order of the tokens afterwards.
        order = torch.sort(x, dim=1, descending=True, stable=True)[1]
        rank = torch.arange(x.shape[1], device=x.device).unsqueeze(0)
        most = torch.where(greedy, 1, torch.where(top_k > 0, top_k, x.shape[1]))
        ws = torch.where(rank < most, torch.gather(w, 1, order), 0)
        upto = torch.cumsum(ws, 1)
        need = _mul_shift(upto[:, -1:], (top_p.clamp(max=1.0).double() * _UNIT).to(torch.int64))
        sorted_keep = (rank < most) & ((upto - ws < need) | (rank == 0))
        keep &= torch.zeros_like(keep).scatter_(1, order, sorted_keep)
    w = torch.where(keep, w, 0)
    upto = torch.cumsum(w, 1)
    mass = upto[:, -1:]
    target = _mul_shift(mass, (t["uniform"].double() * _UNIT).to(torch.int64).unsqueeze(1))
    token = (upto > target).to(torch.uint8).argmax(1, keepdim=True)
    log_prob = torch.log(torch.gather(w, 1, token).float() / mass.float())
    return [token.squeeze(1).to(torch.int32), log_prob.squeeze(1)]


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
    kind, logits = case["kind"], t["logits"]
    if kind == "top":
        ctx.native_top_logits(logits, case["k"], temperature=case["temperature"],
                              values=out[0], indices=out[1], log_sum=out[2])
    elif kind == "sample":
        ctx.native_sample(logits, t["uniform"], temperature=t.get("temperature", case["temperature"]),
                          top_k=t.get("top_k", case["top_k"]), top_p=t.get("top_p", case["top_p"]),
                          min_p=t.get("min_p", case["min_p"]), tokens=out[0], log_prob=out[1])
    else:
        loss = {"temperature": case["temperature"], "teacher_log_sum": t.get("teacher_log_sum"),
                "labels": t.get("labels"), "distill_weight": 1.0 - case["label"],
                "label_weight": case["label"], "vocab": case["vocab"]}
        args = (logits, t["values"], t["indices"])
        if kind == "loss":
            ctx.native_distill_loss(*args, **loss, loss=out[0], log_sums=out[1])
        elif kind == "backward":
            ctx.native_distill_backward(*args, t["log_sums"], **loss, row_scale=t["row_scale"], gradient=out[0])
        else:
            ctx.native_distill_step(*args, **loss, row_scale=t["row_scale"], loss=out[0], gradient=out[1])
    return state["out"]


def run(state):
    if own:
        return _own(state)
    case, t = state["case"], state["tensors"]
    if case["kind"] == "top":
        return _plain_top(case, t)
    if case["kind"] == "sample":
        return _plain_sample(case, t)
    return _plain_distill(case, t, case["kind"] != "backward", case["kind"] != "loss")


# ------------------------------------------------------------------ work and exact values


def work(case):
    rows, vocab, size = case["rows"], case["vocab"], _SIZE[case["dtype"]]
    stat = 8 if case["dtype"] == "f64" else 4
    n = rows * vocab
    if case["kind"] == "top":  # a comparison, a difference, an exponential and a sum a logit
        return {"bytes": n * size + rows * (case["k"] * (size + 4) + stat), "flops": 4 * n}
    if case["kind"] == "sample":
        return {"bytes": n * size + rows * (12 + (16 if case["mixed"] else 0)), "flops": 4 * n}
    extra = rows * (case["k"] * (size + 4) + stat * (1 + int(case["full"])) + (4 if case["label"] else 0))
    if case["kind"] == "loss":
        return {"bytes": n * size + extra + 2 * rows * stat, "flops": 4 * n}
    moved = n * size + rows * case["cols"] * size + extra
    return {"bytes": moved + (2 * rows * stat if case["kind"] == "backward" else rows * stat),
            "flops": (4 if case["kind"] == "backward" else 7) * n}


def _exact_sample(case, t):
    """Row by row: the definition's integer weights, the kept tokens by a lexicographic order,
    and the logarithm of the drawn token's share in binary64."""
    log_prob, tokens = [], []
    settings = [c.squeeze(1).tolist() for c in _settings(case, t)]
    for r in range(case["rows"]):
        x = t["logits"][r].double().cpu().numpy()
        temperature, top_k, top_p, min_p = (s[r] for s in settings)
        peak = x.max()
        inverse = np.float32(np.inf) if temperature == 0 else np.float32(1) / np.float32(temperature)
        if np.isinf(inverse):
            top_k, inverse = 1, np.float32(1)
        near = x - peak if case["dtype"] == "f64" else x.astype(np.float32) - np.float32(peak)
        z = torch.from_numpy(near.astype(np.float32) * inverse).cuda()
        w = (torch.exp(z).double() * 2.0**40).floor().cpu().numpy().astype(np.int64)
        w[x == peak] = _ONE
        by = np.lexsort((np.arange(x.size), -x))
        if top_k > 0:
            by = by[:top_k]
        mass = int(w[by].sum())
        before = np.cumsum(w[by]) - w[by]
        n = max(1, int((before < mass * int(min(float(np.float32(top_p)), 1.0) * 2**31) // 2**31).sum()))
        kept = np.sort(by[:n])
        kept = kept[w[kept] >= math.ceil(float(np.float32(min_p)) * 2**40)]
        upto = np.cumsum(w[kept])
        target = int(upto[-1]) * int(float(t["uniform"][r]) * 2**31) // 2**31
        token = int(kept[np.searchsorted(upto, target, side="right")])
        tokens.append(token)
        log_prob.append(math.log(int(w[token])) - math.log(int(upto[-1])))
    return [np.array(tokens, dtype=np.int32), np.array(log_prob)]


def exact(case, seed):
    t = _tensors(case, seed)
    if case["kind"] == "sample":
        return None if case["rows"] * case["vocab"] > 100_000_000 else _exact_sample(case, t)
    rows, vocab, k, tau = case["rows"], case["vocab"], case["k"], case["temperature"]
    if case["kind"] == "top":
        lse = torch.cat([torch.logsumexp(c.double() / tau, 1) for c in t["logits"].split(256)])
        return [torch.cat([torch.topk(c.double(), k, dim=1)[0] for c in t["logits"].split(256)]), None, lse]
    b, losses, stats, grads = case["label"], [], [], []
    for lo in range(0, rows, 256):
        part = {n: x[lo: lo + 256] for n, x in t.items()}
        s = part["logits"][:, :vocab].double()
        full = torch.log_softmax(s / tau, 1)
        hard = torch.log_softmax(s, 1)
        target = part["values"].double() / tau
        gone = part["indices"] < 0
        target = target.masked_fill(gone, -math.inf)
        base = part["teacher_log_sum"].double()[:, None] if "teacher_log_sum" in t else torch.logsumexp(target, 1, keepdim=True)
        q = torch.exp(target - base).masked_fill(gone, 0.0)
        where = part["indices"].long().clamp(min=0)
        dense = torch.zeros_like(s).scatter_add_(1, where, q)
        parts = q * (target - base - full.gather(1, where))
        loss = (1 - b) * tau**2 * parts.masked_fill(gone, 0.0).nansum(1)
        grad = (1 - b) * tau * (dense.sum(1, keepdim=True) * full.exp() - dense)
        if b:
            on = part["labels"] >= 0
            one = torch.zeros_like(s).scatter_(1, part["labels"].long().clamp(min=0)[:, None], 1.0)
            loss = loss - b * torch.where(on, (one * hard).sum(1), 0.0)
            grad = grad + b * on[:, None] * (hard.exp() - one)
        losses.append(loss)
        stats.append(torch.stack([torch.logsumexp(s / tau, 1), torch.logsumexp(s, 1)], 1))
        if case["kind"] != "loss":
            grad = grad * part["row_scale"].double()[:, None]
            grads.append(torch.nn.functional.pad(grad, (0, case["cols"] - vocab)))
    if case["kind"] == "loss":
        return [torch.cat(losses), torch.cat(stats)]
    return [torch.cat(grads)] if case["kind"] == "backward" else [torch.cat(losses), torch.cat(grads)]
