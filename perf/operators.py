"""The operators of a large model's last layers that are timed: block-scaled 8-bit floating-point quantisation, the dense layer on
such operands, and the log-probabilities of given classes with entropy and the best alternatives.

Sizes stand for a model's layers one token at a time, a few sequences at a time and whole prompts at a time, and for classifiers with
a thousand to a quarter of a million classes.  Inputs come from the seed; activations have a few columns that are much larger than the rest,
logits have peaks, masked classes and rows whose mask leaves nothing.
"""
import math

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTIVATIONS = {"none": 0, "relu": 1, "leaky": 2}
SLOPE = 0.1


def listed():
    return [
        # One token of one sequence through a square projection: latency, and the weights' bytes.
        dict(name="dense_1x4096x4096_bf16", op="dense", rows=1, outputs=4096, inputs=4096, dtype="bf16", bias=False, act="none"),
        # A few sequences decoded together, a wide layer: the weights' bytes.
        dict(name="dense_24x8192x8192_bf16", op="dense", rows=24, outputs=8192, inputs=8192, dtype="bf16", bias=False, act="none"),
        # A classifier head on odd sizes: rows, outputs and the last block are all cut short.
        dict(name="dense_333x1001x2064_f32", op="dense", rows=333, outputs=1001, inputs=2064, dtype="f32", bias=True, act="leaky"),
        # A prompt of two thousand tokens, with bias and activation.
        dict(name="dense_2048x8192x4096_f16", op="dense", rows=2048, outputs=8192, inputs=4096, dtype="f16", bias=True, act="relu"),
        # Several prompts at once: the tensor cores.
        dict(name="dense_8192x8192x8192_bf16", op="dense", rows=8192, outputs=8192, inputs=8192, dtype="bf16", bias=False, act="none"),
        # The activations of one token, before its dense layer.
        dict(name="quantize_1x4096_bf16", op="quantize", rows=1, columns=4096, block_rows=1, dtype="bf16"),
        # The activations of several prompts.
        dict(name="quantize_8192x8192_bf16", op="quantize", rows=8192, columns=8192, block_rows=1, dtype="bf16"),
        # A weight matrix as it is loaded: square blocks, the last ones cut short.
        dict(name="quantize_weights_5000x4112_f32", op="quantize", rows=5000, columns=4112, block_rows=128, dtype="f32"),
        # One image's thousand classes.
        dict(name="logprobs_1x1000_f32", op="logprobs", rows=1, classes=1000, dtype="f32", top=5, masked=False),
        # A few sequences under a grammar that masks classes, some rows whole.
        dict(name="logprobs_6x131072_f32", op="logprobs", rows=6, classes=131072, dtype="f32", top=20, masked=True),
        # A batch of sequences, an odd number of classes.
        dict(name="logprobs_160x50257_f16", op="logprobs", rows=160, classes=50257, dtype="f16", top=10, masked=True),
        # Scoring a whole text: memory bandwidth.
        dict(name="logprobs_2048x131072_bf16", op="logprobs", rows=2048, classes=131072, dtype="bf16", top=8, masked=False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["dense", "dense", "dense", "quantize", "logprobs", "logprobs"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "dense":
        return dict(op=op, rows=_log_int(rng, 1, 8192), outputs=_log_int(rng, 64, 8192), inputs=16 * _log_int(rng, 16, 512), dtype=dtype,
                    bias=rng.random() < 0.5, act=rng.choice(["none", "none", "relu", "leaky"]))
    if op == "quantize":
        return dict(op=op, rows=_log_int(rng, 1, 8192), columns=16 * _log_int(rng, 16, 512), block_rows=rng.choice([1, 1, 128]), dtype=dtype)
    classes = _log_int(rng, 64, 262144)
    rows = _log_int(rng, 1, min(4096, 2048 * 131072 // (2 if dtype == "f32" else 1) // classes))
    return dict(op=op, rows=rows, classes=classes, dtype=dtype, top=rng.choice([0, 1, 5, 8, 20, 32]), masked=rng.random() < 0.5)


# --------------------------------------------------------------------------- shared arithmetic
def _blocks(n):
    return (n + 127) // 128


def _spread(scales, rows, columns, block_rows):
    """The scale of every element from the scale of every block."""
    s = scales.repeat_interleave(128, 1)[:, :columns]
    return s if block_rows == 1 else s.repeat_interleave(128, 0)[:rows]


def _quantize(x, block_rows):
    """The codes and scales of a matrix: scale = largest magnitude / 448 in fp32 (1 for a block of zeros), code = x / scale to the nearest
    e4m3 value, ties to even.  The quotient is taken in 64 bits: in 32 it can land on the border between two codes."""
    rows, columns = x.shape
    r, c = _blocks(rows) if block_rows == 128 else rows, _blocks(columns)
    whole = torch.zeros(r * block_rows, c * 128, dtype=torch.float32, device=x.device)
    whole[:rows, :columns] = x
    amax = whole.view(r, block_rows, c, 128).abs().amax((1, 3))
    # a division by a tensor: one by a number is a product with its rounded inverse
    scales = torch.where(amax > 0, (amax / torch.full_like(amax, 448)).clamp_min(2.0 ** -126), torch.ones_like(amax))
    q = (whole.view(r, block_rows, c, 128).double() / scales.double()[:, None, :, None]).view(r * block_rows, c * 128)[:rows, :columns]
    step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
    # log2 may round up to the next whole number just below a power of two, where the step is the smaller one
    step = torch.where(q.abs() < step * 8, (step / 2).clamp_min(2.0 ** -9), step)
    return (torch.round(q / step) * step).clamp(-448, 448).float().to(F8), scales


# --------------------------------------------------------------------------- inputs
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _activations(rows, columns, g):
    x = torch.randn(rows, columns, generator=g, device="cuda")
    loud = torch.rand(columns, generator=g, device="cuda") < 0.004
    return x * torch.where(loud, 25.0, 1.0)


def prepare(case, seed):
    g = _generator(seed)
    rows, kind = case["rows"], TYPES[case["dtype"]]
    state = dict(case)
    if case["op"] == "dense":
        K, C = case["outputs"], case["inputs"]
        state["x"], state["x_scales"] = _quantize(_activations(rows, C, g), 1)
        state["w"], state["w_scales"] = _quantize(torch.randn(K, C, generator=g, device="cuda") * (0.6 / math.sqrt(C)), 128)
        state["b"] = torch.randn(K, generator=g, device="cuda") * 0.1 if case["bias"] else None
        state["y"] = torch.empty(rows, K, dtype=kind, device="cuda")
        if own:
            from smallframework_b200 import interface as S
            state["buffers"] = (S.Float8Buffer(rows, C, data=state["x"], scales=state["x_scales"]),
                                S.Float8Buffer(K, C, 128, data=state["w"], scales=state["w_scales"]),
                                S.FloatBuffer(data=state["b"]) if case["bias"] else None, _buffer(S, state["y"]))
    elif case["op"] == "quantize":
        C, m = case["columns"], case["block_rows"]
        state["x"] = (_activations(rows, C, g) if m == 1 else torch.randn(rows, C, generator=g, device="cuda") / math.sqrt(C)).to(kind)
        state["q"] = torch.empty(rows, C, dtype=F8, device="cuda")
        state["scales"] = torch.empty(rows if m == 1 else _blocks(rows), _blocks(C), device="cuda")
        if own:
            from smallframework_b200 import interface as S
            state["buffers"] = (_buffer(S, state["x"]), S.Float8Buffer(rows, C, m, data=state["q"], scales=state["scales"]))
    else:
        V, top = case["classes"], case["top"]
        x = torch.randn(rows, V, generator=g, device="cuda") * 2.5
        # peaks: a few classes stand out in every row, by little or by much
        at = torch.randint(V, (rows, 8), generator=g, device="cuda")
        x.scatter_add_(1, at, torch.rand(rows, 8, generator=g, device="cuda") * 14)
        tokens = torch.randint(V, (rows,), generator=g, device="cuda")
        tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.5, at[:, 0], tokens)
        if case["masked"]:
            # by rows: all classes allowed, a tenth of them, a few, none; masks are the type's lowest value or minus infinity
            low = torch.finfo(kind).min
            kinds = torch.randint(6, (rows, 1), generator=g, device="cuda")
            u = torch.rand(rows, V, generator=g, device="cuda")
            x = torch.where((kinds == 1) & (u > 0.1), low, x)
            x = torch.where((kinds == 2) & (u > 0.1), -math.inf, x)
            x = torch.where((kinds == 3) & (u > 4 / V), -math.inf, x)
            x = torch.where(kinds == 4, -math.inf, x)
            # positions that no token is given for
            tokens = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.1, -1, tokens)
        state["x"], state["tokens"] = x.to(kind), tokens
        state["out"] = (torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda"),
                        torch.empty(rows, top, device="cuda"), torch.empty(rows, top, dtype=torch.int32, device="cuda"))
        if own:
            from smallframework_b200 import interface as S
            lp, h, tv, ti = state["out"]
            state["buffers"] = (_buffer(S, state["x"]), S.FloatBuffer(data=lp), S.FloatBuffer(data=h), S.FloatBuffer(data=tv) if top else None)
    return state


def _buffer(S, t):
    return {torch.float32: S.FloatBuffer, torch.bfloat16: S.BFloat16Buffer, torch.float16: S.HalfBuffer}[t.dtype](data=t)


# --------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    if state["op"] == "dense":
        x = state["x"].float() * _spread(state["x_scales"], state["rows"], state["inputs"], 1)
        w = state["w"].float() * _spread(state["w_scales"], state["outputs"], state["inputs"], 128)
        y = x @ w.t()
        if state["b"] is not None:
            y = y + state["b"]
        if state["act"] != "none":
            y = torch.where(y > 0, y, y * (SLOPE if state["act"] == "leaky" else 0.0))
        return y.to(TYPES[state["dtype"]])
    if state["op"] == "quantize":
        q, scales = _quantize(state["x"].float(), state["block_rows"])
        return {"q": q, "scales": scales}
    x = state["x"].float()
    m = x.amax(1, keepdim=True)
    empty = m == -math.inf
    t = x - torch.where(empty, 0.0, m)
    p = torch.exp(t)
    s = p.sum(1, keepdim=True)
    log_s = torch.log(torch.where(empty, 1.0, s))
    entropy = (log_s - torch.where(p > 0, p * t, 0.0).sum(1, keepdim=True) / torch.where(empty, 1.0, s)).squeeze(1)
    tokens = state["tokens"]
    given = torch.where(tokens >= 0, (t.gather(1, tokens.clamp_min(0)[:, None]) - log_s).squeeze(1), 0.0)
    out = {"logprobs": given, "entropy": torch.where(empty.squeeze(1), 0.0, entropy)}
    if state["top"]:
        # the value in whole-number order above, the class below: no two keys are alike, and of equal values the lowest class is best
        bits = (x + 0.0).view(torch.int32).long()
        order = torch.where(bits < 0, -(bits & 0x7fffffff) - 1, bits)
        key = order * (1 << 31) + ((1 << 31) - 1 - torch.arange(x.shape[1], device=x.device))
        best = (1 << 31) - 1 - (key.topk(state["top"], dim=1).values & ((1 << 31) - 1))
        out["top_logprobs"] = t.gather(1, best) - log_s
        out["top_tokens"] = best.int()
    return out


def _run_own(state):
    from smallframework_b200 import interface as S
    if state["op"] == "dense":
        x, w, b, y = state["buffers"]
        S.Dense_Bias_Activation(state["outputs"], state["inputs"], x, w, b, y, activation=ACTIVATIONS[state["act"]],
                                negative_slope=SLOPE, batch=state["rows"])
        return state["y"]
    if state["op"] == "quantize":
        x, q = state["buffers"]
        S.QuantizeBlocks(state["rows"], state["columns"], x, q)
        return {"q": state["q"], "scales": state["scales"]}
    x, lp, h, tv = state["buffers"]
    top = state["top"]
    S.LogProbabilities(state["rows"], state["classes"], x, state["tokens"], lp, h, tv, state["out"][3] if top else None, top=top)
    out = {"logprobs": state["out"][0], "entropy": state["out"][1]}
    if top:
        out["top_logprobs"], out["top_tokens"] = state["out"][2], state["out"][3]
    return out


# --------------------------------------------------------------------------- work and exact results
def work(case):
    rows, size = case["rows"], TYPES[case["dtype"]].itemsize
    if case["op"] == "dense":
        K, C = case["outputs"], case["inputs"]
        scales = 4 * _blocks(C) * (rows + _blocks(K))
        return {"bytes": rows * C + K * C + scales + rows * K * size + (4 * K if case["bias"] else 0), "flops": 2 * rows * K * C}
    if case["op"] == "quantize":
        C = case["columns"]
        blocks = (rows if case["block_rows"] == 1 else _blocks(rows)) * _blocks(C)
        return {"bytes": rows * C * (size + 1) + 4 * blocks, "flops": 3 * rows * C}
    # largest value, difference, exponential, two sums
    return {"bytes": rows * case["classes"] * size + rows * (16 + 8 * case["top"]), "flops": 6 * rows * case["classes"]}


def _e4m3_values():
    """All non-negative e4m3 values in ascending order: 2^-9 times the subnormals' whole numbers, then (8 + m) * 2^(e - 10)."""
    return torch.tensor([m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1],
                        dtype=torch.float64, device="cuda")


def _exact_quantize(x, block_rows):
    rows, columns = x.shape
    table = _e4m3_values()
    middle = (table[1:] + table[:-1]) / 2
    q = torch.empty(rows, columns, dtype=torch.float64, device="cuda")
    scales = torch.empty(rows if block_rows == 1 else _blocks(rows), _blocks(columns), dtype=torch.float64, device="cuda")
    for c in range(_blocks(columns)):
        at = slice(128 * c, min(columns, 128 * c + 128))
        v = x[:, at].double()
        a = v.abs().amax(1)
        if block_rows == 128:
            a = torch.nn.functional.pad(a, (0, -rows % 128)).view(-1, 128).amax(1)
        s = (a / 448).float().double().clamp_min(2.0 ** -126)  # the scale that is stored is an fp32 number
        s[a == 0] = 1
        scales[:, c] = s
        if block_rows == 128:
            s = s.repeat_interleave(128)[:rows]
        quotient = v.abs() / s[:, None]
        below = torch.searchsorted(middle, quotient)               # the value below a middle that is met exactly
        above = torch.searchsorted(middle, quotient, right=True)   # the value above it
        code = torch.where(below % 2 == 0, below, above)           # of the two, the even code
        q[:, at] = torch.copysign(table[code], v)
    return q, scales


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "dense":
        K, C = case["outputs"], case["inputs"]
        y = torch.zeros(case["rows"], K, dtype=torch.float64, device="cuda")
        for c in range(_blocks(C)):
            at = slice(128 * c, min(C, 128 * c + 128))
            ws = state["w_scales"][:, c].double().repeat_interleave(128)[:K]
            y += (state["x"][:, at].double() @ state["w"][:, at].double().t()) * state["x_scales"][:, c].double()[:, None] * ws
        if case["bias"]:
            y += state["b"].double()
        if case["act"] == "relu":
            y = y.clamp_min(0)
        elif case["act"] == "leaky":
            y = torch.where(y < 0, y * SLOPE, y)
        return y
    if case["op"] == "quantize":
        q, scales = _exact_quantize(state["x"], case["block_rows"])
        return {"q": q, "scales": scales}
    parts = []
    rows_at_once = max(1, (1 << 25) // case["classes"])
    for r in range(0, case["rows"], rows_at_once):
        x = state["x"][r:r + rows_at_once].double()
        tokens = state["tokens"][r:r + rows_at_once]
        m = x.amax(1, keepdim=True)
        nothing = m == -math.inf
        t = x - torch.where(nothing, 0.0, m)  # before the logarithm: beside a mask of the type's lowest value that would be lost
        logp = t - torch.where(nothing, 1.0, t.exp().sum(1, keepdim=True)).log()
        p = logp.exp()
        h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
        given = logp.gather(1, tokens.clamp(min=0)[:, None]).squeeze(1)
        given[tokens < 0] = 0
        part = [given, h]
        if case["top"]:
            best = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :case["top"]]
            part += [logp.gather(1, best), best.int()]
        parts.append(part)
    whole = [torch.cat(p) for p in zip(*parts)]
    return dict(zip(("logprobs", "entropy", "top_logprobs", "top_tokens"), whole))
