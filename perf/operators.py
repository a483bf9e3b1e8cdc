"""Workloads of the training operators: embedding lookup and its gradient, LayerNorm forward and backward, AdamW.

``listed()`` names the workloads, ``draw(rng)`` gives more of the same ranges, ``prepare(case, seed)`` makes the tensors a
training program holds before the call, ``run(state)`` makes one pass: the plain form (elementary torch operations in
32 bits) or, with ``own`` set, the call of this package's kernel.  ``exact(case, seed)`` is the same result in 64 bits,
``work(case)`` the bytes and operations that a pass cannot do without.
"""
from __future__ import annotations

import functools
import json
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "i32": torch.int32, "i64": torch.int64}
BYTES = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i64": 8}
BETAS, EPSILON, DECAY = (0.9, 0.999), 1e-8, 0.1
ALIGN = 64  # elements between the starts of two tensors of the optimizer's storage


def listed():
    return [
        # one decoding step of sixteen sequences: a handful of rows, only latency counts
        dict(name="lookup 16 x 4096", op="lookup", tokens=16, vocab=32768, hidden=4096, table="bf16", out="bf16", ids="i32",
             scale=1.0, spread="even"),
        # a long packed batch through a table kept in 32 bits, scaled by sqrt(hidden)
        dict(name="lookup 65536 x 4096 scaled", op="lookup", tokens=65536, vocab=50257, hidden=4096, table="f32", out="bf16",
             ids="i64", scale=64.0, spread="zipf"),
        # a micro-batch with padding, accumulated into the 32-bit gradient of the table
        dict(name="lookup grad 4096 added", op="lookup_grad", tokens=4096, vocab=32768, hidden=2048, grad="bf16", table="f32",
             ids="i32", scale=1.0, spread="zipf", padded=0.2, accumulate=True),
        # the whole gradient of a large vocabulary, written once
        dict(name="lookup grad 65536 x 4096", op="lookup_grad", tokens=65536, vocab=131072, hidden=4096, grad="bf16",
             table="bf16", ids="i64", scale=1.0, spread="zipf", padded=0.0, accumulate=False),
        # a few rows, as in evaluation between steps
        dict(name="norm 16 x 4096", op="norm", rows=16, hidden=4096, dtype="bf16", weight="bf16", residual=False, bias=True),
        # rows of no vector's length
        dict(name="norm 4099 x 1535", op="norm", rows=4099, hidden=1535, dtype="f16", weight="f16", residual=False, bias=True),
        # a block's norm over a large batch, with the residual added on the way and 32-bit weights
        dict(name="norm 65536 x 8192 residual", op="norm", rows=65536, hidden=8192, dtype="bf16", weight="f32", residual=True,
             bias=True),
        dict(name="norm grad 64 x 1024", op="norm_grad", rows=64, hidden=1024, dtype="f32", weight="f32", residual=False, bias=True),
        dict(name="norm grad 8191 x 1001", op="norm_grad", rows=8191, hidden=1001, dtype="f16", weight="f32", residual=False, bias=True),
        dict(name="norm grad 65536 x 8192", op="norm_grad", rows=65536, hidden=8192, dtype="bf16", weight="f32", residual=True,
             bias=True),
        # the parameters of a small head, all in 32 bits
        dict(name="adamw 1 M in 24", op="adamw", matrices=8, rows=256, cols=512, vectors=16, length=511, param="f32", grad="f32", masters=False),
        # the blocks of a mid-sized model: 16-bit parameters with 32-bit copies
        dict(name="adamw 400 M in 144", op="adamw", matrices=48, rows=2048, cols=4096, vectors=96, length=2047, param="bf16", grad="bf16", masters=True),
    ]


MOST_BYTES = 4 * 2 * 65536 * 8192  # of a drawn case: what the largest listed one moves


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["lookup", "lookup_grad", "norm", "norm_grad", "adamw"])
    if op == "adamw":
        case = dict(op=op, matrices=rng.randint(1, 48), rows=_spread(rng, 1, 4096), cols=_spread(rng, 16, 4099), vectors=rng.randint(0, 96),
                    length=_spread(rng, 1, 8192), param=rng.choice(["f32", "bf16", "f16"]), grad=rng.choice(["param", "f32"]), masters=False)
        case["grad"] = case["param"] if case["grad"] == "param" else "f32"
        case["masters"] = case["param"] != "f32" and rng.random() < 0.6
    elif op in ("norm", "norm_grad"):
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        case = dict(op=op, rows=_spread(rng, 1, 65536), hidden=_spread(rng, 16, 8192), dtype=dtype, weight=rng.choice([dtype, "f32"]),
                    residual=rng.random() < 0.5, bias=rng.random() < 0.8)
        if rng.random() < 0.6:  # most models' widths are whole vectors; the others stay as drawn
            case["hidden"] = max(16, case["hidden"] // 64 * 64) if case["hidden"] >= 64 else 16
    else:
        case = dict(op=op, tokens=_spread(rng, 1, 65536), vocab=_spread(rng, 16, 131072), hidden=_spread(rng, 16, 8192),
                    table=rng.choice(["f32", "bf16", "f16"]), ids=rng.choice(["i32", "i64"]), scale=rng.choice([1.0, 0.5, 11.25]),
                    spread=rng.choice(["zipf", "even"]))
        if rng.random() < 0.7:
            case["hidden"] = max(16, case["hidden"] // 16 * 16)
        case["vocab"] = max(2, min(case["vocab"], (1 << 29) // case["hidden"]))
        if op == "lookup":
            case["out"] = rng.choice([case["table"], "bf16"])
        else:
            case.update(grad=rng.choice([case["table"], "bf16"]), padded=rng.choice([0.0, 0.25]), accumulate=rng.random() < 0.5)
    size = "cols" if op == "adamw" else "rows" if "rows" in case else "tokens"
    while work(case)["bytes"] > MOST_BYTES:
        case[size] = max(1, case[size] // 2)
    return case


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _tokens(case, generator):
    """Token numbers: evenly spread, or with the 1/rank frequencies of a vocabulary (ranks scattered over the numbers)."""
    count, vocab = case["tokens"], case["vocab"]
    u = torch.rand(count, device="cuda", dtype=torch.float64, generator=generator)
    rank = (u * vocab).long() if case["spread"] == "even" else torch.exp(u * math.log(vocab + 1)).long() - 1
    tokens = (rank.clamp_(0, vocab - 1) * 7919 + 13) % vocab
    if case.get("padded"):  # the tail of every sequence of 64 is padding
        tail = torch.arange(count, device="cuda") % 64 >= round(64 * (1 - case["padded"]))
        tokens = torch.where(tail, torch.zeros_like(tokens), tokens)
    return tokens.to(DTYPES[case["ids"]])


def _padding(case):
    return 0 if case.get("padded") else None


def _shapes(case):
    shapes = [(case["rows"], case["cols"])] * case["matrices"]
    return shapes + [(case["length"] + index,) for index in range(case["vectors"])]


def _places(case):
    """Start of every tensor of the optimizer in its storage, the first place without decay (the vectors), and the end."""
    starts, at, first_vector = [], 0, 0
    for index, shape in enumerate(_shapes(case)):
        if index == case["matrices"]:
            first_vector = at
        starts.append(at)
        at += -(-math.prod(shape) // ALIGN) * ALIGN
    return starts, first_vector if case["vectors"] else at, at


def _views(flat, case):
    starts, _, _ = _places(case)
    return [flat[start:start + math.prod(shape)].view(shape) for start, shape in zip(starts, _shapes(case))]


def prepare(case, seed):
    generator = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype="f32", scale=1.0, shift=0.0):
        return torch.randn(shape, device="cuda", generator=generator).mul_(scale).add_(shift).to(DTYPES[dtype])

    op = case["op"]
    state = {"case": case}
    if op == "lookup":
        state.update(tokens=_tokens(case, generator), table=normal(case["vocab"], case["hidden"], dtype=case["table"], scale=0.02),
                     out=torch.empty(case["tokens"], case["hidden"], device="cuda", dtype=DTYPES[case["out"]]))
    elif op == "lookup_grad":
        state.update(grad_out=normal(case["tokens"], case["hidden"], dtype=case["grad"]), tokens=_tokens(case, generator))
        shape = (case["vocab"], case["hidden"])
        state["grad_table"] = normal(*shape, dtype=case["table"]) if case["accumulate"] else torch.empty(shape, device="cuda", dtype=DTYPES[case["table"]])
    elif op in ("norm", "norm_grad"):
        rows, hidden, dtype = case["rows"], case["hidden"], case["dtype"]
        x = normal(rows, hidden, scale=1.5).add_(normal(rows, 1, scale=0.5, shift=0.5))
        x[:, ::97] *= 8.0  # a few channels are far larger than the others, as trained networks have them
        state.update(x=x.to(DTYPES[dtype]), weight=normal(hidden, dtype=case["weight"], scale=0.1, shift=1.0),
                     bias=normal(hidden, dtype=case["weight"], scale=0.1) if case["bias"] else None)
        del x
        state["residual"] = normal(rows, hidden, dtype=dtype) if case["residual"] else None
        if op == "norm":
            state.update(out=torch.empty_like(state["x"]), out_resid=torch.empty_like(state["x"]) if case["residual"] else None,
                         mean=torch.empty(rows, device="cuda"), rstd=torch.empty(rows, device="cuda"))
        else:
            wide = state["x"].double()
            variance, mean = torch.var_mean(wide, dim=-1, correction=0)
            state.update(grad_out=normal(rows, hidden, dtype=dtype), mean=mean.float(), rstd=(variance + 1e-5).rsqrt().float(),
                         grad_x=torch.empty_like(state["x"]), grad_weight=torch.empty_like(state["weight"]),
                         grad_bias=torch.empty_like(state["weight"]) if case["bias"] else None)
    else:
        _, _, total = _places(case)
        mask = torch.zeros(total, device="cuda")
        for view in _views(mask, case):
            view.fill_(1.0)

        def flat(dtype, scale, positive=False):
            values = normal(total, scale=scale).mul_(mask)
            return (values.square_() if positive else values).to(DTYPES[dtype])

        params = flat("f32", 0.02)
        state.update(params=params.to(DTYPES[case["param"]]), masters=params if case["masters"] else None, grads=flat(case["grad"], 1e-2),
                     exp_avgs=flat("f32", 1e-3), exp_avg_sqs=flat("f32", 1e-2, positive=True),
                     schedule=torch.tensor([1e-3, 100.0 + seed % 64, 0.5], device="cuda"))  # learning rate, step, factor on the gradients
    if own:
        state["call"] = _program(state)
    return state


# ---------------------------------------------------------------------------------------------
# this package's kernels
# ---------------------------------------------------------------------------------------------
ORDER = {
    "lookup": ("tokens", "table", "out"),
    "lookup_grad": ("grad_out", "tokens", "grad_table"),
    "norm": ("x", "out", "mean", "rstd", "weight", "bias", "residual", "out_resid"),
    "norm_grad": ("grad_out", "x", "mean", "rstd", "weight", "grad_x", "grad_weight", "grad_bias", "residual"),
    "adamw": ("params", "grads", "exp_avgs", "exp_avg_sqs", "schedule", "masters"),
}


def _kernel(case):
    import baybridge_b200 as cute

    op = case["op"]
    if op == "lookup":
        def body(tokens, table, out):
            cute.embedding(tokens, table, out, scale=case["scale"])
    elif op == "lookup_grad":
        def body(grad_out, tokens, grad_table):
            cute.embedding_backward(grad_out, tokens, grad_table, scale=case["scale"], padding_token=_padding(case),
                                    accumulate=case["accumulate"])
    elif op == "norm":
        def body(x, out, mean, rstd, weight, bias, residual, out_resid):
            cute.layernorm_forward(x, out, mean, rstd, weight, bias, residual=residual, out_resid=out_resid, epsilon=1e-5)
    elif op == "norm_grad":
        def body(grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias, grad_resid):
            cute.layernorm_backward(grad_out, x, mean, rstd, weight, grad_x, grad_weight, grad_bias, grad_resid=grad_resid)
    else:
        decay = [DECAY] * case["matrices"] + [0.0] * case["vectors"]

        def body(params, grads, exp_avgs, exp_avg_sqs, schedule, masters):
            cute.adamw(params, grads, exp_avgs, exp_avg_sqs, schedule, masters=masters, betas=BETAS, epsilon=EPSILON, weight_decay=decay)
    return cute.kernel(body)


_ARTIFACTS = {}


def _program(state):
    """The compiled kernel of the case (compiled once per case, as a program does) bound to handles of the state's tensors."""
    import baybridge_b200 as cute

    case = state["case"]
    arguments = []
    for name in ORDER[case["op"]]:
        value = state[name]
        if case["op"] == "adamw" and name != "schedule" and value is not None:
            arguments.append(cute.tensor_group(_views(value, case)))
        else:
            arguments.append(None if value is None else cute.from_dlpack(value))
    key = json.dumps({k: v for k, v in case.items() if k != "name"}, sort_keys=True)
    if key not in _ARTIFACTS:
        _ARTIFACTS[key] = cute.compile(_kernel(case), *arguments, backend=cute.B200Backend(synchronize=False))
    return functools.partial(_ARTIFACTS[key], *arguments)


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def _plain_lookup(s, case):
    return {"out": (s["table"][s["tokens"].long()].float() * case["scale"]).to(s["out"].dtype)}


def _plain_lookup_grad(s, case):
    tokens, given = s["tokens"].long(), s["grad_out"].float() * case["scale"]
    if _padding(case) is not None:
        given = torch.where((tokens != _padding(case))[:, None], given, torch.zeros((), device="cuda"))
    sums = s["grad_table"].float() if case["accumulate"] else torch.zeros(s["grad_table"].shape, device="cuda")
    if sums is s["grad_table"]:
        sums = sums.clone()
    sums.index_add_(0, tokens, given)
    s["grad_table"].copy_(sums)
    return {"grad_table": s["grad_table"]}


def _plain_norm(s, case):
    x = s["x"].float()
    if case["residual"]:
        x = x + s["residual"].float()
    mean = x.mean(-1, keepdim=True)
    centred = x - mean
    rstd = 1.0 / torch.sqrt((centred * centred).mean(-1, keepdim=True) + 1e-5)
    out = centred * rstd * s["weight"].float()
    if case["bias"]:
        out = out + s["bias"].float()
    kind = s["x"].dtype
    return {"out": out.to(kind), "mean": mean[:, 0], "rstd": rstd[:, 0], "out_resid": x.to(kind) if case["residual"] else None}


def _plain_norm_grad(s, case):
    given, rstd = s["grad_out"].float(), s["rstd"][:, None]
    normal = (s["x"].float() - s["mean"][:, None]) * rstd
    inner = given * s["weight"].float()
    grad_x = (inner - inner.mean(-1, keepdim=True) - normal * (inner * normal).mean(-1, keepdim=True)) * rstd
    if case["residual"]:
        grad_x = grad_x + s["residual"].float()
    kind = s["weight"].dtype
    return {"grad_x": grad_x.to(s["x"].dtype), "grad_weight": (given * normal).sum(0).to(kind),
            "grad_bias": given.sum(0).to(kind) if case["bias"] else None}


def _plain_adamw(s, case):
    _, decayed, _ = _places(case)
    rate, step, factor = s["schedule"].unbind()
    step = step.double()
    first, second = 1 - BETAS[0] ** step, 1 - BETAS[1] ** step  # 64 bits: 1 - beta^t is small at first
    grad = s["grads"].float() * factor
    s["exp_avgs"].mul_(BETAS[0]).add_(grad * (1 - BETAS[0]))
    s["exp_avg_sqs"].mul_(BETAS[1]).add_(grad * grad * (1 - BETAS[1]))
    values = s["masters"] if case["masters"] else s["params"].float()
    values[:decayed] *= 1 - rate * DECAY
    values -= rate * (s["exp_avgs"] / first.float()) / (torch.sqrt(s["exp_avg_sqs"] / second.float()) + EPSILON)
    s["params"].copy_(values)
    return {"params": s["params"], "exp_avgs": s["exp_avgs"], "exp_avg_sqs": s["exp_avg_sqs"], "masters": s["masters"]}


PLAIN = {"lookup": _plain_lookup, "lookup_grad": _plain_lookup_grad, "norm": _plain_norm, "norm_grad": _plain_norm_grad, "adamw": _plain_adamw}
OUTPUTS = {
    "lookup": ("out",), "lookup_grad": ("grad_table",), "norm": ("out", "mean", "rstd", "out_resid"),
    "norm_grad": ("grad_x", "grad_weight", "grad_bias"), "adamw": ("params", "exp_avgs", "exp_avg_sqs", "masters"),
}


def run(state):
    op = state["case"]["op"]
    if own:
        state["call"]()
        return {name: state[name] for name in OUTPUTS[op]}
    return PLAIN[op](state, state["case"])


# ---------------------------------------------------------------------------------------------
# the same in 64 bits, and what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    op = case["op"]
    if op == "lookup":
        return {"out": s["table"].double().index_select(0, s["tokens"].long()).mul_(case["scale"])}
    if op == "lookup_grad":
        order = torch.argsort(s["tokens"].long())
        if _padding(case) is not None:
            order = order[s["tokens"][order] != _padding(case)]
        total = s["grad_table"].double() if case["accumulate"] else torch.zeros(s["grad_table"].shape, device="cuda", dtype=torch.float64)
        for part in order.split(8192):
            total.index_add_(0, s["tokens"][part].long(), s["grad_out"][part].double(), alpha=case["scale"])
        return {"grad_table": total}
    if op == "norm":
        x = s["x"].double() + s["residual"].double() if case["residual"] else s["x"].double()
        variance, mean = torch.var_mean(x, dim=-1, correction=0, keepdim=True)
        scale = torch.rsqrt(variance + 1e-5)
        out = torch.addcmul(s["bias"].double() if case["bias"] else torch.zeros((), device="cuda", dtype=torch.float64),
                            (x - mean) * scale, s["weight"].double())
        return {"out": out, "mean": mean.squeeze(-1), "rstd": scale.squeeze(-1), "out_resid": x if case["residual"] else None}
    if op == "norm_grad":
        grads = {"grad_x": torch.empty(case["rows"], case["hidden"], device="cuda", dtype=torch.float64),
                 "grad_weight": torch.zeros(case["hidden"], device="cuda", dtype=torch.float64),
                 "grad_bias": torch.zeros(case["hidden"], device="cuda", dtype=torch.float64) if case["bias"] else None}
        for at in range(0, case["rows"], 8192):
            rows = slice(at, min(at + 8192, case["rows"]))
            given, scale = s["grad_out"][rows].double(), s["rstd"][rows].double()[:, None]
            unit = (s["x"][rows].double() - s["mean"][rows].double()[:, None]) * scale
            grads["grad_weight"] += torch.einsum("rh,rh->h", given, unit)
            if case["bias"]:
                grads["grad_bias"] += given.sum(0)
            given = given * s["weight"].double()
            along = torch.einsum("rh,rh->r", given, unit)[:, None] / case["hidden"]
            grads["grad_x"][rows] = scale * (given - given.sum(-1, keepdim=True) / case["hidden"] - unit * along)
            if case["residual"]:
                grads["grad_x"][rows] += s["residual"][rows].double()
        return grads
    rate, step, factor = (float(value) for value in s["schedule"])
    grad = s["grads"].double() * factor
    exp_avg = torch.lerp(grad, s["exp_avgs"].double(), BETAS[0])
    exp_avg_sq = torch.lerp(grad.square(), s["exp_avg_sqs"].double(), BETAS[1])
    values = (s["masters"] if case["masters"] else s["params"]).double()
    decay = torch.zeros_like(values)
    decay[:_places(case)[1]] = DECAY
    denominator = (exp_avg_sq / -math.expm1(step * math.log(BETAS[1]))).sqrt() + EPSILON
    values = values - rate * decay * values - rate / -math.expm1(step * math.log(BETAS[0])) * exp_avg / denominator
    return {"params": values, "exp_avgs": exp_avg, "exp_avg_sqs": exp_avg_sq, "masters": values if case["masters"] else None}


@functools.lru_cache(maxsize=None)
def _distinct(tokens, vocab, spread):
    """How many rows of the table a batch is expected to name."""
    if spread == "even":
        return vocab * -math.expm1(tokens * math.log1p(-1.0 / vocab)) if vocab > 1 else 1
    rank = torch.arange(1, vocab + 1, dtype=torch.float64)
    share = torch.log1p(1.0 / rank) / math.log(vocab + 1)
    return float(-torch.expm1(tokens * torch.log1p(-share.clamp(max=1 - 1e-12))).sum())


def work(case):
    op = case["op"]
    if op == "adamw":
        count = sum(math.prod(shape) for shape in _shapes(case))
        each = BYTES[case["grad"]] + 16 + (8 + BYTES[case["param"]] if case["masters"] else 2 * BYTES[case["param"]])
        return {"bytes": count * each, "flops": count * 16}
    if op in ("norm", "norm_grad"):
        rows, hidden, size = case["rows"], case["hidden"], BYTES[case["dtype"]]
        vectors = (1 + case["bias"]) * hidden * BYTES[case["weight"]]
        if op == "norm":
            return {"bytes": (4 if case["residual"] else 2) * rows * hidden * size + vectors + 8 * rows, "flops": rows * hidden * 9}
        vectors += hidden * BYTES[case["weight"]]  # the weight is read, its gradient and the bias's are written
        return {"bytes": (4 if case["residual"] else 3) * rows * hidden * size + vectors + 8 * rows, "flops": rows * hidden * 14}
    tokens, vocab, hidden = case["tokens"], case["vocab"], case["hidden"]
    distinct = _distinct(tokens, vocab, case["spread"])
    if op == "lookup":
        return {"bytes": distinct * hidden * BYTES[case["table"]] + tokens * (hidden * BYTES[case["out"]] + BYTES[case["ids"]]), "flops": tokens * hidden}
    kept = tokens * (1 - case["padded"])
    rows = 2 * distinct if case["accumulate"] else vocab
    return {"bytes": rows * hidden * BYTES[case["table"]] + kept * hidden * BYTES[case["grad"]] + tokens * BYTES[case["ids"]],
            "flops": 2 * kept * hidden}
