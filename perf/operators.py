"""Measured cases of the trainable front of an index: embedding tables and linear adapters.

Four operators, the two directions of each:

* ``lookup``: rows of an embedding table by id, times a scale; a negative id (an unfilled search
  result slot) gives a row of zeros.
* ``grad``: the table's gradient, ``grad[r] = scale * sum of upstream[i] over ids[i] == r``, dense,
  with zeros where no id points.
* ``linear``: ``act(x W^T + bias) + residual``, the adapter that maps vectors before they are
  added to an index or searched for.
* ``train``: ``linear`` and its backward pass, as one training step runs it.

Where ``own`` is false the operators are computed from elementary torch operations in float32.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
GLOVE_ROWS = 1183514  # the GloVe-100 collection of the benchmark


def listed():
    return [
        # The tokens of one short query: latency.
        dict(name="lookup.query", op="lookup", rows=32000, dim=768, n=19, dtype="bf16", ids="i64"),
        # The vectors behind 10,000 answers of 10 neighbours each, for a re-ranker: float32 rows
        # of 400 bytes, some result slots unfilled.
        dict(name="lookup.neighbours", op="lookup", rows=GLOVE_ROWS, dim=100, n=100000,
             dtype="f32", ids="i64"),
        # A training batch of text: frequent tokens repeat.
        dict(name="lookup.batch", op="lookup", rows=131072, dim=1024, n=131072, dtype="bf16",
             ids="i32"),
        # The gradient of a handful of sentences.
        dict(name="grad.few", op="grad", rows=32000, dim=768, n=509, dtype="bf16", ids="i64"),
        # Item vectors of a whole collection, trained by sampled neighbours; odd batch.
        dict(name="grad.items", op="grad", rows=GLOVE_ROWS, dim=100, n=50001, dtype="f32",
             ids="i64"),
        # The gradient of a training batch of text, frequent tokens thousands of times in it.
        dict(name="grad.batch", op="grad", rows=131072, dim=1024, n=131072, dtype="bf16",
             ids="i32"),
        # One query through a query adapter: latency.
        dict(name="linear.one", op="linear", m=1, k=768, n=768, dtype="bf16", act="gelu",
             bias=True, residual=True),
        # The benchmark's 10,000-query batch of 768-dimensional float32 vectors.
        dict(name="linear.queries", op="linear", m=10000, k=768, n=768, dtype="f32", act="none",
             bias=True, residual=True),
        # Small odd sizes whose rows are not multiples of 16 bytes.
        dict(name="linear.odd", op="linear", m=1003, k=100, n=100, dtype="f16", act="relu",
             bias=True, residual=True),
        # The wide layer of an encoder over a large batch.
        dict(name="linear.wide", op="linear", m=32768, k=1024, n=4096, dtype="bf16", act="gelu",
             bias=True, residual=False),
        # Training an adapter of GloVe-100 queries, float32, with its skip connection.
        dict(name="train.adapter", op="train", m=4097, k=100, n=100, dtype="f32", act="silu",
             bias=True, residual=True),
        # Training the wide layer of an encoder.
        dict(name="train.wide", op="train", m=8192, k=1024, n=4096, dtype="bf16", act="gelu",
             bias=True, residual=False),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm; odd ones as likely as any,
    and every third one rounded to a multiple of 8."""
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.randrange(3) == 0:
        v = (v + 7) // 8 * 8
    return max(lo, min(hi, v))


def draw(rng):
    op = rng.choice(("lookup", "grad", "linear", "train"))
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    if op in ("lookup", "grad"):
        while True:
            c = dict(op=op, rows=_spread(rng, 1000, GLOVE_ROWS), dim=_spread(rng, 32, 1024),
                     n=_spread(rng, 1, 131072), dtype=dtype, ids=rng.choice(("i64", "i32")))
            if (c["rows"] + c["n"]) * c["dim"] * SIZE[dtype] <= 262144 * 1024 * 2:
                return c
    while True:
        c = dict(op=op, m=_spread(rng, 1, 32768), k=_spread(rng, 32, 4096),
                 n=_spread(rng, 32, 4096), dtype=dtype,
                 act=rng.choice(("none", "relu", "gelu", "gelu_tanh", "silu")),
                 bias=rng.random() < 0.8, residual=rng.random() < 0.5)
        most = 32768 * 1024 * 4096 if op == "linear" else 8192 * 1024 * 4096
        if c["m"] * c["k"] * c["n"] <= most:
            return c


def _ids(case, g):
    """Ids as they come: neighbours of a collection spread evenly, some slots unfilled; tokens by
    a power law (token r about as often as 1/(r+1)), a few of a batch padded with -1."""
    rows, n = case["rows"], case["n"]
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    if rows > 200000:
        ids = (u * rows).long()
    else:
        ids = (torch.exp(u * math.log(rows + 1.0)) - 1.0).long()
    ids = ids.clamp(0, rows - 1)
    ids[torch.rand(n, generator=g, device="cuda") < 0.01] = -1
    return ids if case["ids"] == "i64" else ids.int()


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    t = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(t)

    s = dict(case)
    if case["op"] in ("lookup", "grad"):
        s["scale"] = math.sqrt(case["dim"])
        s["ids"] = _ids(case, g)
        if case["op"] == "lookup":
            s["table"] = normal(case["rows"], case["dim"], scale=case["dim"] ** -0.5)
        else:
            s["upstream"] = normal(case["n"], case["dim"], scale=0.02)
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s["x"] = normal(m, k)
    s["w"] = normal(n, k, scale=k ** -0.5)
    s["b"] = normal(n, scale=0.1) if case["bias"] else None
    s["r"] = normal(m, n) if case["residual"] else None
    if case["op"] == "train":
        s["dy"] = normal(m, n, scale=0.02)
        for name in ("x", "w", "b", "r"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return (0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
                + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi))
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        q = 1 / (1 + torch.exp(-z))
        return q * (1 + z * (1 - q))
    return torch.ones_like(z)


def _plain_lookup(s):
    ids = s["ids"].long()
    rows = s["table"][ids.clamp(min=0)].float() * s["scale"]
    return torch.where((ids >= 0)[:, None], rows, 0.0).to(s["table"].dtype)


def _plain_grad(s):
    ids = s["ids"].long()
    up = s["upstream"].float()
    total = torch.zeros(s["rows"] + 1, s["dim"], device=up.device)
    total.index_add_(0, torch.where(ids >= 0, ids, s["rows"]), up)
    return (total[:s["rows"]] * s["scale"]).to(s["upstream"].dtype)


def _plain_linear(s):
    z = s["x"].float() @ s["w"].float().t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y = _act(z, s["act"])
    if s["r"] is not None:
        y = y + s["r"].float()
    return y.to(s["x"].dtype), z


def _plain_train(s):
    t = s["x"].dtype
    with torch.no_grad():
        y, z = _plain_linear(s)
        dz = s["dy"].float() * _act_grad(z, s["act"])
        out = {"y": y, "dx": (dz @ s["w"].float()).to(t), "dw": (dz.t() @ s["x"].float()).to(t)}
        if s["b"] is not None:
            out["db"] = dz.sum(0).to(t)
        if s["r"] is not None:
            out["dr"] = s["dy"]
    return out


def _own_train(s):
    from quiver_b200 import embed
    y = embed.linear(s["x"], s["w"], s["b"], residual=s["r"], activation=s["act"])
    names = [k for k in ("x", "w", "b", "r") if s[k] is not None]
    grads = torch.autograd.grad(y, [s[k] for k in names], s["dy"])
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(names, grads)}}


def run(state):
    s = state
    if own:
        from quiver_b200 import embed
        if s["op"] == "lookup":
            return embed.embedding_lookup(s["table"], s["ids"], s["scale"])
        if s["op"] == "grad":
            return embed.embedding_grad(s["upstream"], s["ids"], s["rows"], s["scale"])
        if s["op"] == "linear":
            return embed.linear(s["x"], s["w"], s["b"], residual=s["r"], activation=s["act"])
        return _own_train(s)
    if s["op"] == "lookup":
        return _plain_lookup(s)
    if s["op"] == "grad":
        return _plain_grad(s)
    if s["op"] == "linear":
        return _plain_linear(s)[0]
    return _plain_train(s)


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] in ("lookup", "grad"):
        rows, n, d = case["rows"], case["n"], case["dim"]
        ids = n * (8 if case["ids"] == "i64" else 4)
        if case["op"] == "lookup":
            # The rows that are read: each distinct one once (its expected number under _ids).
            if rows > 200000:
                distinct = rows * -math.expm1(n * math.log1p(-1.0 / rows))
            else:
                r = np.arange(rows, dtype=np.float64)
                p = np.log1p(1.0 / (r + 1)) / math.log(rows + 1.0)
                distinct = float(-np.expm1(n * np.log1p(-p)).sum())
            return {"bytes": ids + (distinct + n) * d * e, "flops": n * d}
        return {"bytes": ids + (n + rows) * d * e, "flops": n * d + rows * d}
    m, k, n = case["m"], case["k"], case["n"]
    bias = n * e if case["bias"] else 0
    res = m * n * e if case["residual"] else 0
    forward = (m * k + n * k + m * n) * e + bias + res
    if case["op"] == "linear":
        return {"bytes": forward, "flops": 2 * m * n * k}
    # The backward pass reads dy and writes dx, dw and db; x and w are read once for the step.
    return {"bytes": forward + (m * n + m * k + n * k) * e + bias, "flops": 6 * m * n * k}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "lookup":
        ids = s["ids"].long()
        out = torch.zeros(case["n"], case["dim"], dtype=torch.float64, device=ids.device)
        held = torch.nonzero(ids >= 0)[:, 0]
        out[held] = s["table"].double().index_select(0, ids[held]) * s["scale"]
        return out
    if case["op"] == "grad":
        ids = s["ids"].long()
        held = torch.nonzero(ids >= 0)[:, 0]
        out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device=ids.device)
        out.index_put_((ids[held],), s["upstream"][held].double() * s["scale"], accumulate=True)
        return out
    leaves = {k: s[k].detach().double().requires_grad_(case["op"] == "train")
              for k in ("x", "w", "b", "r") if s[k] is not None}
    z = torch.einsum("mk,nk->mn", leaves["x"], leaves["w"])
    if "b" in leaves:
        z = z + leaves["b"]
    cdf = {"none": lambda: 1.0, "relu": lambda: (z > 0).double(),
           "gelu": lambda: torch.special.ndtr(z),
           "gelu_tanh": lambda: torch.sigmoid(
               2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)),
           "silu": lambda: torch.sigmoid(z)}[case["act"]]()
    y = z * cdf
    if "r" in leaves:
        y = y + leaves["r"]
    if case["op"] == "linear":
        return y
    grads = torch.autograd.grad(y, list(leaves.values()), s["dy"].double())
    return {"y": y.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}
