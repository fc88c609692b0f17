"""The operators at the end of a decode step, and beside the packed linears: the 8-bit floating-point linear with a scale
for every block of 128, and drawing a token from logits.  Cases, inputs, the operators' plain forms and the calls.

    listed()               the fixed cases
    draw(rng)              one more case of the same ranges
    prepare(case, seed)    inputs and quantized weights: what the program holds before a call
    run(state)             one pass: the plain form, or with `own` the framework's operators
    work(case)             bytes and floating-point operations that a pass cannot do without
    exact(case, seed)      what run() returns, in 64 bits

A case's "kind" says which path it takes:

    linear    `fp8_linear` on new activations: quantize them by blocks of 128 along K, multiply with the weight
    shared    activations quantized once (`quantize_fp8_activations`) for the three weights that read them
    convert   `quantize_fp8_weight`: a dense weight to codes and a scale for every 128 x 128 block
    sample    `sample_logits`: one token a row from temperature, top-k, top-p and min-p and a given random number
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
LARGEST = 448.0                          # of E4M3
HIDDEN, KV, FFN, VOCAB = 4096, 1024, 14336, 128256      # the benchmark's decoder


def listed():
    return [
        # one token through the smallest projection of a decoder layer: latency
        {"name": "kv_1", "kind": "linear", "m": 1, "n": KV, "k": HIDDEN, "x": "bf16", "out": "bf16"},
        # one token through the output head: half a gigabyte of weight
        {"name": "head_1", "kind": "linear", "m": 1, "n": VOCAB, "k": HIDDEN, "x": "bf16", "out": "f32"},
        # sixteen sequences through the down projection, few rows and a long K
        {"name": "down_16", "kind": "linear", "m": 16, "n": HIDDEN, "k": FFN, "x": "bf16", "out": "bf16"},
        # a decode batch through the gate projection
        {"name": "gate_48", "kind": "linear", "m": 48, "n": FFN, "k": HIDDEN, "x": "bf16", "out": "bf16"},
        # a ragged batch through an adapter-sized layer whose sides are no multiple of the block, half precision
        {"name": "ragged_333", "kind": "linear", "m": 333, "n": 1000, "k": 1500, "x": "f16", "out": "f16"},
        # a long prompt through the gate projection
        {"name": "gate_4096", "kind": "linear", "m": 4096, "n": FFN, "k": HIDDEN, "x": "bf16", "out": "bf16"},
        # a prompt through q, k and v, which read the same activations
        {"name": "qkv_777", "kind": "shared", "m": 777, "hidden": HIDDEN, "kv": KV, "x": "bf16", "out": "bf16"},
        # loading a model: a gate projection from bf16 to blocks
        {"name": "convert_gate", "kind": "convert", "n": FFN, "k": HIDDEN, "x": "bf16"},
        # one conversation, the usual chat settings
        {"name": "sample_1", "kind": "sample", "rows": 1, "vocab": VOCAB, "x": "bf16", "masked": 0.0, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # a serving batch whose requests each bring their own settings (temperature -1: a value for each row)
        {"name": "sample_64", "kind": "sample", "rows": 64, "vocab": VOCAB, "x": "bf16", "masked": 0.0, "temperature": -1.0, "top_k": -1, "top_p": -1.0, "min_p": -1.0},
        # pure sampling of a small vocabulary, for rollouts: no filter at all
        {"name": "sample_rollout", "kind": "sample", "rows": 16, "vocab": 32000, "x": "f32", "masked": 0.0, "temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0},
        # output bound to a grammar: most of an odd-sized vocabulary is masked
        {"name": "sample_masked", "kind": "sample", "rows": 7, "vocab": 50001, "x": "f16", "masked": 0.97, "temperature": 1.2, "top_k": 0, "top_p": 0.9, "min_p": 0.05},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _side(rng, lo, hi):
    value = _log(rng, lo, hi)
    return value if rng.random() < 0.3 else max(128, value // 128 * 128)      # most layers have round sizes


def draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "shared", "convert", "sample", "sample", "sample"])
    if kind == "linear":
        m, k = _log(rng, 1, 4096), _side(rng, 128, FFN)
        n = _side(rng, 64, VOCAB) if rng.random() < 0.3 else _side(rng, 64, 28672)
        while n * k > VOCAB * HIDDEN or 2.0 * m * n * k > 4.8e11 or m * n > 4096 * FFN:
            if m > 64:
                m = m * 2 // 3
            else:
                n = max(64, n // 2)
        x = rng.choice(["bf16", "bf16", "bf16", "f16", "f32"])
        return {"kind": kind, "m": m, "n": n, "k": k, "x": x, "out": rng.choice([x, "bf16", "f32"])}
    if kind == "shared":
        hidden = max(256, _log(rng, 1024, 8192) // 128 * 128)
        m = _log(rng, 1, 3000)
        while 4.0 * m * hidden * hidden > 4.8e11:
            m //= 2
        x = rng.choice(["bf16", "bf16", "f16"])
        return {"kind": kind, "m": m, "hidden": hidden, "kv": max(64, hidden // rng.choice([1, 4, 8]) // 64 * 64), "x": x, "out": x}
    if kind == "convert":
        n, k = _side(rng, 64, 28672), _side(rng, 128, 14336)
        while n * k > FFN * HIDDEN:
            n = max(1, n // 2)
        return {"kind": kind, "n": n, "k": k, "x": rng.choice(["bf16", "bf16", "f16", "f32"])}
    rows, vocab = _log(rng, 1, 256), _log(rng, 1000, 262144)
    while rows * vocab > 64 * VOCAB:
        rows = max(1, rows // 2)
    own_settings = rng.random() < 0.3
    return {"kind": kind, "rows": rows, "vocab": vocab, "x": rng.choice(["bf16", "bf16", "f32", "f16"]),
            "masked": rng.choice([0.0, 0.0, 0.5, 0.99]),
            "temperature": -1.0 if own_settings else round(rng.uniform(0.3, 1.5), 2),
            "top_k": -1 if own_settings else rng.choice([0, 0, 1, 20, 50, 200, 1000]),
            "top_p": -1.0 if own_settings else rng.choice([1.0, 1.0, 0.99, 0.95, 0.9, 0.5]),
            "min_p": -1.0 if own_settings else rng.choice([0.0, 0.0, 0.02, 0.1])}


# ------------------------------------------------------------------------------------------ inputs
def _weight(n, k, gen, dtype=torch.bfloat16):
    """Heavy-tailed weight, Student-t with 4 degrees of freedom times 0.02 (the benchmark's)."""
    z = torch.randn((n, k), generator=gen, device="cuda")
    chi = torch.zeros((n, k), device="cuda")
    for _ in range(4):
        d = torch.randn((n, k), generator=gen, device="cuda")
        chi.addcmul_(d, d)
    return (z / torch.sqrt(chi / 4) * 0.02).to(dtype)


def _tokens(m, k, gen, dtype):
    """Activations as a layer's norm leaves them, with a few channels that stand out."""
    x = torch.randn((m, k), generator=gen, device="cuda")
    x[:, torch.randperm(k, generator=gen, device="cuda")[: max(1, k // 200)]] *= 20.0
    return x.to(dtype)


def _packed(n, k, gen):
    codes, scales = _by_tiles(_weight(n, k, gen))
    if own:
        import mixfp4_b200 as mx

        return mx.FP8Weight.from_tensors(codes, scales)
    return codes, scales


def _settings(case, gen):
    """Numbers for every row, or with -1 a tensor that has each row's own."""
    rows, got = case["rows"], {}
    for name, choices, dtype in (("temperature", (0.0, 0.6, 0.8, 1.0, 1.3), torch.float32), ("top_k", (0, 1, 20, 64, 500), torch.int32),
                                 ("top_p", (1.0, 0.99, 0.95, 0.9, 0.5), torch.float32), ("min_p", (0.0, 0.0, 0.02, 0.1), torch.float32)):
        got[name] = case[name]
        if case[name] == -1:
            which = torch.randint(0, len(choices), (rows,), generator=gen, device="cuda")
            got[name] = torch.tensor(choices, dtype=dtype, device="cuda")[which]
    return got


@torch.no_grad()
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, state = case["kind"], {"kind": case["kind"]}
    if kind == "linear":
        state.update(w=_packed(case["n"], case["k"], gen), x=_tokens(case["m"], case["k"], gen, DTYPES[case["x"]]), out=DTYPES[case["out"]])
    elif kind == "shared":
        h, kv = case["hidden"], case["kv"]
        state.update(w=[_packed(n, h, gen) for n in (h, kv, kv)], x=_tokens(case["m"], h, gen, DTYPES[case["x"]]), out=DTYPES[case["out"]])
    elif kind == "convert":
        state.update(w=_weight(case["n"], case["k"], gen, DTYPES[case["x"]]))
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = 3.0 * torch.randn((rows, vocab), generator=gen, device="cuda")
        # a few tokens ahead of the rest, as a trained model's head puts them
        at = torch.randint(0, vocab, (rows, 8), generator=gen, device="cuda")
        logits.scatter_add_(1, at, 12.0 * torch.rand((rows, 8), generator=gen, device="cuda"))
        if case["masked"]:
            logits[torch.rand((rows, vocab), generator=gen, device="cuda") < case["masked"]] = -math.inf
        state.update(logits=logits.to(DTYPES[case["x"]]), uniform=torch.rand(rows, generator=gen, device="cuda"), settings=_settings(case, gen))
    return state


# -------------------------------------------------------------------------------------------- pass
def _blocks(x, rows):
    """x in 32 bits as [row blocks, rows, column blocks, 128], padded with zeros."""
    r, k = x.shape
    x = torch.nn.functional.pad(x.float(), (0, -k % 128, 0, -r % rows))
    return x.reshape(-1, rows, x.shape[1] // 128, 128)


def _quantized(x, rows):
    """Codes and scales: the block's largest magnitude becomes 448; a block whose scale would be zero has the scale 1."""
    b = _blocks(x, rows)
    largest = b.abs().amax(dim=(1, 3), keepdim=True)
    scale = largest / torch.full_like(largest, LARGEST)                        # by a tensor: a number would multiply with 1/448
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    codes = (b / scale).clamp(-LARGEST, LARGEST).to(torch.float8_e4m3fn)
    codes = codes.reshape(b.shape[0] * rows, -1)[: x.shape[0], : x.shape[1]]
    return codes.contiguous(), scale[:, 0, :, 0].contiguous()


def _by_rows(x):
    return _quantized(x, 1)


def _by_tiles(w):
    return _quantized(w, 128)


def _values(codes, scales, rows):
    """The 32-bit values that codes and scales stand for."""
    s = scales.repeat_interleave(rows, 0)[: codes.shape[0]].repeat_interleave(128, 1)[:, : codes.shape[1]]
    return codes.float() * s


def _linear(x, weight, out):
    return (_values(*_by_rows(x), 1) @ _values(*weight, 128).T).to(out)


def _sample(logits, u, temperature, top_k, top_p, min_p):
    """In 64 bits: the kept set and the token hang on comparisons of sums."""
    rows, vocab = logits.shape
    setting = lambda v, dtype: (v if isinstance(v, torch.Tensor) else torch.full((rows,), v, device=logits.device)).to(dtype)[:, None]
    t, k = setting(temperature, torch.float64), setting(top_k, torch.int64)
    p, floor = setting(top_p, torch.float64), setting(min_p, torch.float64)
    x = logits.double()
    x = torch.where(x.isnan(), -math.inf, x)
    x, index = torch.sort(x, dim=1, descending=True, stable=True)
    largest = x[:, :1]
    w = torch.where(x == largest, 1.0, torch.exp((x - largest) / torch.where(t > 0, t, 1.0)))
    w = torch.where((x == -math.inf) | ((t == 0) & (x < largest)), 0.0, w)
    rank = torch.arange(vocab, device=x.device)
    first = torch.where(t == 0, 1, torch.where(k <= 0, vocab, k))             # temperature zero: the first of the largest
    w = torch.where(rank < first, w, 0.0)
    before = torch.cumsum(w, 1)
    total = before[:, -1:]
    before = torch.nn.functional.pad(before[:, :-1], (1, 0))
    keep = (w >= floor) & ((rank == 0) | (p >= 1.0) | (before < p * total))
    w = torch.where(keep, w, 0.0)
    w = torch.zeros_like(w).scatter_(1, index, w)                              # back in the vocabulary's order
    run_up = torch.cumsum(w, 1)
    total = run_up[:, -1:]
    token = torch.searchsorted(run_up, u.double()[:, None] * total, right=True).clamp(max=vocab - 1)
    weight = torch.gather(w, 1, token)
    empty = total[:, 0] == 0
    token = torch.where(empty, -1, token[:, 0])
    return token, torch.where(empty, -math.inf, torch.log(weight[:, 0] / total[:, 0])).float()


@torch.no_grad()
def run(state):
    kind = state["kind"]
    if own:
        import mixfp4_b200 as mx

        if kind == "linear":
            return mx.fp8_linear(state["x"], state["w"], out_dtype=state["out"])
        if kind == "shared":
            x = mx.quantize_fp8_activations(state["x"])
            return [mx.fp8_linear(x, w, out_dtype=state["out"]) for w in state["w"]]
        if kind == "convert":
            w = mx.quantize_fp8_weight(state["w"])
            return [w.codes, w.scales]
        return mx.sample_logits(state["logits"], state["uniform"], return_logprob=True, **state["settings"])
    if kind == "linear":
        return _linear(state["x"], state["w"], state["out"])
    if kind == "shared":
        x = _values(*_by_rows(state["x"]), 1)
        return [(x @ _values(*w, 128).T).to(state["out"]) for w in state["w"]]
    if kind == "convert":
        return list(_by_tiles(state["w"]))
    return _sample(state["logits"], state["uniform"], **state["settings"])


# ------------------------------------------------------------------------------------ what it takes
def work(case):
    kind = case["kind"]
    if kind == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * BYTES[case["x"]] + 4 + 12), "flops": 0}
    size = BYTES[case["x"]]
    weight = lambda n, k: n * k + 4 * -(-n // 128) * -(-k // 128)
    if kind == "convert":
        return {"bytes": size * case["n"] * case["k"] + weight(case["n"], case["k"]), "flops": 0}
    m, out = case["m"], BYTES[case["out"]]
    if kind == "shared":
        n, k = case["hidden"] + 2 * case["kv"], case["hidden"]
    else:
        n, k = case["n"], case["k"]
    return {"bytes": size * m * k + weight(n, k) + out * m * n, "flops": 2.0 * m * n * k}


# ---------------------------------------------------------------------------------------- in 64 bits
def _e4m3(v):
    """Doubles to the nearest E4M3 value, ties to the even mantissa: spacing 2^(e-3), and 2^-9 below 2^-6."""
    _, e = torch.frexp(v)                                                      # |v| in [2^(e-1), 2^e)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _exact_blocks(x, rows):
    """(values of the codes, scales) with the block's scale held in 32 bits, and the quotient too: that is the operator's definition."""
    r, k = x.shape
    values = torch.empty((r, k), dtype=torch.float64, device=x.device)
    scales = torch.empty((-(-r // rows), -(-k // 128)), dtype=torch.float64, device=x.device)
    for b in range(scales.shape[1]):
        part = x[:, 128 * b: 128 * b + 128].double()
        padded = torch.zeros((scales.shape[0] * rows, part.shape[1]), dtype=torch.float64, device=x.device)
        padded[:r] = part
        top = padded.abs().reshape(scales.shape[0], -1).max(dim=1).values
        s = (top / 448).float().double()
        s[s == 0] = 1.0
        scales[:, b] = s
        values[:, 128 * b: 128 * b + 128] = _e4m3((part / s[torch.arange(r, device=x.device) // rows, None]).float().double())
    return values, scales


def _exact_product(x, codes, scales):
    """Rows of x against the weight, 8192 rows of the weight at a time."""
    q, s = _exact_blocks(x, 1)
    block = torch.arange(x.shape[1], device=x.device) // 128
    q = q * s[:, block]
    parts = []
    for n in range(0, codes.shape[0], 8192):
        c = codes[n: n + 8192].double()
        parts.append(q @ (c * scales.double()[torch.arange(n, n + c.shape[0], device=x.device) // 128][:, block]).T)
    return torch.cat(parts, 1)


def _exact_row(x, u, t, k, p, floor):
    """One row of sample_logits with numpy: (token, log probability)."""
    x = np.where(np.isnan(x), -np.inf, x)
    top = x.max()
    if top == -np.inf:
        return -1, -np.inf
    order = np.lexsort((np.arange(len(x)), -x))
    if t == 0:
        return int(order[0]), 0.0
    order = order[: k if k > 0 else None]
    order = order[x[order] > -np.inf]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == top, 1.0, np.exp((x[order] - top) / t))
    if p < 1.0:
        w = w[: max(1, int(np.searchsorted(np.cumsum(w), p * w.sum(), side="left")) + 1)]
    w = w[w >= floor]
    kept = np.sort(order[: len(w)])
    weight = dict(zip(order[: len(w)].tolist(), w.tolist()))
    w = np.array([weight[i] for i in kept.tolist()])
    up = np.cumsum(w)
    at = min(int(np.searchsorted(up, u * up[-1], side="right")), len(kept) - 1)
    return int(kept[at]), math.log(w[at] / up[-1])


@torch.no_grad()
def exact(case, seed):
    global own
    before, own = own, False                                                   # the same codes and scales, as tensors
    try:
        s = prepare(case, seed)
    finally:
        own = before
    if s["kind"] == "linear":
        return _exact_product(s["x"], *s["w"])
    if s["kind"] == "shared":
        return [_exact_product(s["x"], *w) for w in s["w"]]
    if s["kind"] == "convert":
        return list(_exact_blocks(s["w"], 128))
    rows = case["rows"]
    each = {k: v.double().cpu().numpy() if isinstance(v, torch.Tensor) else np.full(rows, v) for k, v in s["settings"].items()}
    logits, u = s["logits"].double().cpu().numpy(), s["uniform"].double().cpu().numpy()
    got = [_exact_row(logits[r], u[r], each["temperature"][r], int(each["top_k"][r]), each["top_p"][r], each["min_p"][r]) for r in range(rows)]
    return torch.tensor([g[0] for g in got], device="cuda"), torch.tensor([g[1] for g in got], dtype=torch.float64, device="cuda")
