"""What is timed of the INT8 operators: matrix products of 8-bit integers with a scale for each
token and each output channel (dense, and grouped by expert with ragged rows; plain or with a
gated pair of weight halves), the per-token quantiser in front of them, and the norms around a
block with its gate and residual scale.

``own`` false: the operators in elementary torch operations; ``own`` true: the framework's own
entry points (``harness.int8``). Both take the same state."""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
#: The largest listed product: no drawn case multiplies more than this.
MOST_PRODUCTS = 8192 ** 3
MOST_WEIGHTS = 32 * 2 * 2048 * 7168
MOST_ELEMENTS = 8192 * 7168


@functools.lru_cache(None)
def _int8():
    package = str(Path(__file__).resolve().parents[1] / "flashinfer-cubins_b200")
    if package not in sys.path:
        sys.path.append(package)
    from harness import int8

    return int8


# -- cases ----------------------------------------------------------------------------------


def listed():
    return [
        # One token through an attention output projection: the weights' bytes are everything.
        dict(name="gemm_token", op="gemm", m=1, n=8192, k=8192, gated=False, bias=False, out="bf16"),
        # A decode batch, odd in tokens and channels, with a bias.
        dict(name="gemm_batch_odd", op="gemm", m=67, n=5121, k=5120, gated=False, bias=True, out="fp16"),
        # Gate and up projections of a dense feed-forward for a thousand prompt tokens.
        dict(name="gemm_gated", op="gemm", m=1000, n=14336, k=4096, gated=True, bias=False, out="bf16"),
        # The square that the framework's own headline is quoted on.
        dict(name="gemm_square", op="gemm", m=8192, n=8192, k=8192, gated=False, bias=False, out="bf16"),
        # Experts of a decode step: eight tokens of eight choices over 32 local experts.
        dict(name="grouped_decode", op="grouped", experts=32, rows=64, n=2048, k=7168, gated=True, out="bf16", skew=1),
        # Their down projections for a small prompt.
        dict(name="grouped_down", op="grouped", experts=32, rows=1024, n=7168, k=2048, gated=False, out="fp16", skew=2),
        # Prompt tokens over few experts: the tensor cores are everything.
        dict(name="grouped_prefill", op="grouped", experts=16, rows=8192, n=1536, k=4096, gated=True, out="bf16", skew=3),
        # Activations of a long prompt on their way into a product.
        dict(name="quantize_prefill", op="quantize", tokens=8192, rows=0, k=7168, type="bf16"),
        # Eight decode tokens, each into the rows of eight experts.
        dict(name="quantize_gather", op="quantize", tokens=8, rows=64, k=7168, type="fp32"),
        # The end of one block and the start of the next for a long prompt.
        dict(name="norm_prefill", op="norm", tokens=8192, hidden=5120, x="fp32", residual="bf16", gates=1, scale=0.5, post=True, next=True, codes=False),
        # The same for a single token, straight into the next product's codes.
        dict(name="norm_token", op="norm", tokens=1, hidden=7168, x="bf16", residual="bf16", gates=0, scale=1.0, post=True, next=True, codes=True),
        # Seven sequences with a gate each, an odd number of tokens.
        dict(name="norm_sequences", op="norm", tokens=2051, hidden=2880, x="fp16", residual="fp16", gates=7, scale=1.0, post=True, next=True, codes=True),
    ]


def _log(rng, low, high):
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("gemm", "gemm", "grouped", "grouped", "quantize", "norm", "norm"))
    if op in ("gemm", "grouped"):
        gated = rng.random() < 0.4
        k = _log(rng, 16, 16384)
        if rng.random() < 0.75:
            k = -(-k // 16) * 16
        n = _log(rng, 8, 16384)
        if rng.random() < 0.6:
            n = -(-n // 8) * 8
        out = rng.choice(("bf16", "fp16", "fp32"))
        width = 2 * n if gated else n
        if op == "gemm":
            m = _log(rng, 1, max(1, min(8192, MOST_PRODUCTS // (width * k))))
            return dict(op=op, m=m, n=n, k=k, gated=gated, bias=not gated and rng.random() < 0.4, out=out)
        experts = _log(rng, 1, max(1, min(128, MOST_WEIGHTS // (width * k))))
        rows = _log(rng, 1, max(1, min(8192, MOST_PRODUCTS // (4 * width * k))))
        return dict(op=op, experts=experts, rows=rows, n=n, k=k, gated=gated, out=out, skew=rng.randrange(1000))
    if op == "quantize":
        k = _log(rng, 1, 16384)
        tokens = _log(rng, 1, MOST_ELEMENTS // k if k > 4096 else 8192)
        rows = 0 if rng.random() < 0.5 else _log(rng, 1, min(8192, max(1, MOST_ELEMENTS // k)))
        return dict(op=op, tokens=tokens, rows=rows, k=k, type=rng.choice(tuple(DTYPES)))
    hidden = _log(rng, 1, 16384)
    gates = rng.choice((0, 1, 1, 2, 5))
    tokens = _log(rng, 1, min(8192, max(1, 8192 * 5120 // hidden)))
    tokens = max(1, tokens // max(gates, 1)) * max(gates, 1)
    kind = rng.choice(("bf16", "fp16", "fp32"))
    post = rng.random() < 0.7
    return dict(op=op, tokens=tokens, hidden=hidden, x=rng.choice((kind, "fp32")), residual=kind, gates=gates,
                scale=rng.choice((1.0, 0.5, 0.22)), post=post, next=not post or rng.random() < 0.8,
                codes=rng.random() < 0.5)


def counts_of(case):
    """Rows of every expert: log-normal shares of ``rows``, some of them empty."""
    rng = random.Random(case["skew"])
    weights = [rng.lognormvariate(0.0, 1.0) for _ in range(case["experts"])]
    total, left = sum(weights), case["rows"]
    counts = [int(case["rows"] * w / total) for w in weights]
    for e in range(case["rows"] - sum(counts)):
        counts[rng.randrange(case["experts"])] += 1
    assert sum(counts) == left
    return counts


# -- inputs ---------------------------------------------------------------------------------


def _codes(shape, g):
    """INT8 codes as a symmetric quantiser leaves them: bell-shaped, the extremes at +-127. Rows
    of a width that is no multiple of 16 bytes lie 16 bytes apart at least, padded as a user pads
    them."""
    *lead, k = shape
    pitch = -(-k // 16) * 16
    flat = torch.empty((math.prod(lead), pitch), dtype=torch.int8, device="cuda")
    for block in flat.split(max(1, (1 << 27) // pitch)):
        block.copy_(torch.randn(block.shape, device="cuda", generator=g, dtype=torch.float16).mul_(30.0).round_().clamp_(-127, 127))
    return flat.view(*lead, pitch)[..., :k]


def _activations(rows, k, dtype, g):
    """Normal activations whose tokens differ in size and of which some channels stand out."""
    x = torch.randn((rows, k), device="cuda", generator=g)
    x *= torch.exp(0.5 * torch.randn((rows, 1), device="cuda", generator=g))
    x *= torch.where(torch.rand((k,), device="cuda", generator=g) < 0.01, 8.0, 1.0)
    return x.to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *shape: torch.rand(shape, device="cuda", generator=g)  # noqa: E731
    s = {"case": case}
    if case["op"] in ("gemm", "grouped"):
        m = case["m"] if case["op"] == "gemm" else case["rows"]
        lead = () if case["op"] == "gemm" else (case["experts"],)
        width = (2 if case["gated"] else 1) * case["n"]
        s["a"] = _codes((m, case["k"]), g)
        s["b"] = _codes((*lead, width, case["k"]), g)
        s["a_scales"] = 0.01 + 0.05 * rand(m)
        # Products of unit size whatever the depth.
        s["b_scales"] = (0.5 + rand(*lead, width)) / (30.0 * math.sqrt(case["k"]))
        s["bias"] = torch.randn((width,), device="cuda", generator=g) if case.get("bias") else None
        if lead:
            counts = torch.tensor(counts_of(case), dtype=torch.int64)
            s["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(device="cuda", dtype=torch.int32)
            s["most"] = int(counts.max())
    elif case["op"] == "quantize":
        s["x"] = _activations(case["tokens"], case["k"], DTYPES[case["type"]], g)
        s["rows"] = torch.randint(0, case["tokens"], (case["rows"],), device="cuda", generator=g, dtype=torch.int32) if case["rows"] else None
    else:
        tokens, hidden = case["tokens"], case["hidden"]
        s["x"] = _activations(tokens, hidden, DTYPES[case["x"]], g)
        s["residual"] = (2.0 * torch.randn((tokens, hidden), device="cuda", generator=g)).to(DTYPES[case["residual"]])
        s["post_weight"] = 0.5 + rand(hidden) if case["post"] else None
        s["next_weight"] = 0.5 + rand(hidden) if case["next"] else None
        s["gate"] = torch.randn((case["gates"], hidden), device="cuda", generator=g) if case["gates"] else None
    return s


# -- one pass -------------------------------------------------------------------------------


def run(state):
    return {"gemm": _gemm, "grouped": _grouped, "quantize": _quantize, "norm": _norm}[state["case"]["op"]](state)


def _silu(x):
    return x / (1.0 + torch.exp(-x))


def _scaled(products, a_scales, b_scales, bias, gated):
    """FP32 sums of code products [..., rows, width] -> FP32 results."""
    y = products * a_scales.unsqueeze(-1) * b_scales.unsqueeze(-2)
    if bias is not None:
        y = y + bias
    if gated:
        half = y.shape[-1] // 2
        y = _silu(y[..., :half]) * y[..., half:]
    return y


def _gemm(s):
    case = s["case"]
    out = DTYPES[case["out"]]
    if own:
        return _int8().gemm(s["a"], s["b"], s["a_scales"], s["b_scales"], bias=s["bias"], gated=case["gated"], out_dtype=out)
    products = s["a"].float() @ s["b"].float().T
    return _scaled(products, s["a_scales"], s["b_scales"], s["bias"], case["gated"]).to(out)


def _grouped(s):
    case = s["case"]
    out = DTYPES[case["out"]]
    if own:
        return _int8().grouped_gemm(s["a"], s["b"], s["a_scales"], s["b_scales"], s["offsets"], gated=case["gated"], out_dtype=out)
    # Every expert's rows in a slab of the fullest one's height, one batched product.
    rows = torch.arange(case["rows"], device="cuda")
    offsets = s["offsets"].long()
    expert = torch.searchsorted(offsets[1:], rows, right=True)
    place = rows - offsets[expert]
    a = torch.zeros((case["experts"], s["most"], case["k"]), device="cuda")
    scales = torch.zeros((case["experts"], s["most"]), device="cuda")
    a[expert, place] = s["a"].float()
    scales[expert, place] = s["a_scales"]
    products = torch.bmm(a, s["b"].float().transpose(1, 2))
    return _scaled(products, scales, s["b_scales"], None, case["gated"])[expert, place].to(out)


def _codes_of(x):
    """FP32 rows -> (INT8 codes, FP32 scales): the scale is the row's largest magnitude over 127
    and the code the nearest integer of the quotient, ties to even. The divisors are tensors, so
    that both quotients are rounded once."""
    scales = x.abs().amax(-1) / torch.full((), 127.0, device=x.device)
    q = torch.where(scales.unsqueeze(-1) > 0, x / scales.unsqueeze(-1), torch.zeros((), device=x.device))
    return q.round().clamp(-127, 127).to(torch.int8), scales


def _quantize(s):
    if own:
        return _int8().quantize_tokens(s["x"], rows=s["rows"])
    x = s["x"] if s["rows"] is None else s["x"][s["rows"].long()]
    return _codes_of(x.float())


def _normed(x, weight, eps):
    """Codes lie next to a border: the statistic is taken in 64 bits and rounded once."""
    mean = x.double().square().sum(-1, keepdim=True) / x.shape[-1]
    return x * (mean + eps).sqrt().reciprocal().float() * weight


def _norm(s):
    case = s["case"]
    eps = 1e-6
    if own:
        r, y, scales = _int8().residual_norm(
            s["x"], s["residual"], post_weight=s["post_weight"], gate=s["gate"], residual_scale=case["scale"],
            next_weight=s["next_weight"], eps=eps, quantize=case["codes"] and case["next"])
        return [v for v in (r, y, scales) if v is not None]
    h = s["x"].float()
    if s["post_weight"] is not None:
        h = _normed(h, s["post_weight"], eps)
    if s["gate"] is not None:
        h = (h.view(case["gates"], -1, case["hidden"]) * s["gate"].unsqueeze(1)).view(h.shape)
    r = s["residual"].float() * case["scale"] + h
    kind = s["residual"].dtype
    if s["next_weight"] is None:
        return [r.to(kind)]
    y = _normed(r, s["next_weight"], eps)
    return [r.to(kind), *_codes_of(y)] if case["codes"] else [r.to(kind), y.to(kind)]


# -- what a pass cannot do without ----------------------------------------------------------


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] in ("gemm", "grouped"):
        width = (2 if case["gated"] else 1) * case["n"]
        if case["op"] == "gemm":
            m, used = case["m"], 1
        else:
            m, used = case["rows"], sum(c > 0 for c in counts_of(case))
        moved = m * case["k"] + 4 * m + used * width * (case["k"] + 4) + m * case["n"] * size[case["out"]]
        return {"bytes": moved + (4 * width if case.get("bias") else 0), "flops": 2 * m * width * case["k"]}
    if case["op"] == "quantize":
        rows = case["rows"] or case["tokens"]
        read = min(rows, case["tokens"]) * case["k"] * size[case["type"]]
        return {"bytes": read + rows * (case["k"] + 4), "flops": 4 * rows * case["k"]}
    elements = case["tokens"] * case["hidden"]
    written = size[case["residual"]]
    if case["next"]:
        written += 1 if case["codes"] else size[case["residual"]]
    vectors = 4 * case["hidden"] * (case["gates"] + case["post"] + case["next"])
    return {"bytes": elements * (size[case["x"]] + size[case["residual"]] + written) + vectors, "flops": 12 * elements}


# -- the operators' definitions in 64 bits --------------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    f = lambda t: t.to(torch.float64)  # noqa: E731

    def product(a, b, sa, sb, bias):
        z = torch.einsum("mk,nk->mn", f(a), f(b)) * torch.outer(f(sa), f(sb))
        z = z if bias is None else z + f(bias)
        if not case["gated"]:
            return z
        gate, up = z.chunk(2, dim=1)
        return gate * torch.sigmoid(gate) * up

    if case["op"] == "gemm":
        return product(s["a"], s["b"], s["a_scales"], s["b_scales"], s["bias"])
    if case["op"] == "grouped":
        edges = s["offsets"].tolist()
        parts = [product(s["a"][lo:hi], s["b"][e], s["a_scales"][lo:hi], s["b_scales"][e], None)
                 for e, (lo, hi) in enumerate(zip(edges, edges[1:])) if hi > lo]
        return torch.cat(parts)
    if case["op"] == "quantize":
        x = f(s["x"]) if s["rows"] is None else f(s["x"]).index_select(0, s["rows"].long())
        return (None, torch.linalg.vector_norm(x, ord=math.inf, dim=1) / 127)

    def rms(x, w):
        return x / torch.sqrt(torch.mean(x ** 2, dim=1, keepdim=True) + 1e-6) * f(w)

    h = f(s["x"])
    h = h if s["post_weight"] is None else rms(h, s["post_weight"])
    if s["gate"] is not None:
        h = h * f(s["gate"]).repeat_interleave(case["tokens"] // case["gates"], dim=0)
    r = case["scale"] * f(s["residual"]) + h
    if s["next_weight"] is None:
        return [r]
    y = rms(r, s["next_weight"])
    return [r, None, torch.linalg.vector_norm(y, ord=math.inf, dim=1) / 127] if case["codes"] else [r, y]
