"""The block norms and the 8-bit integer products: their cases, plain forms and exact values.

``run`` computes them from elementary torch operations, or, where ``own`` is
true, through the framework's entry points (``qcc_b200.runtime.block_norm``
and ``qcc_b200.runtime.int8_dense``).
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6
SMALLEST_AMAX = 2.0 ** -119  # rows below this are stored as zeros (their scale would not be a normal fp32 number)


def listed():
    return [
        # The norm before the FFN of one decode step: latency.
        dict(name="norm_one_token", op="norm", tokens=1, hidden=5120, kind="rms", dtype="bf16"),
        # The same norm, with means and biases, over a prompt in fp16.
        dict(name="norm_prompt_layer", op="norm", tokens=2048, hidden=5120, kind="layer", dtype="fp16"),
        # Decode of a batch: the FFN's output is normed, gated per token and added, and the next block's norm taken.
        dict(name="join_batch", op="join", tokens=8, hidden=5120, kind="rms", gate="token", dtype="bf16",
             residual="bf16"),
        # A small model of odd width in fp32, gated per channel.
        dict(name="join_odd", op="join", tokens=517, hidden=1111, kind="layer", gate="channel", dtype="fp32",
             residual="fp32"),
        # A long prompt's residual stream kept in bf16.
        dict(name="join_prompt", op="join", tokens=8192, hidden=5120, kind="rms", gate="none", dtype="bf16",
             residual="bf16"),
        # The down projection of one decode step, quantising its input: reads the weight once.
        dict(name="linear_one_token", op="linear", tokens=1, rows=5120, cols=17408, source="rows", dtype="bf16",
             bias=False),
        # Odd sizes with a bias, from rows that are int8 already, fp32 out.
        dict(name="linear_odd", op="linear", tokens=77, rows=1000, cols=1111, source="int8", dtype="fp32", bias=True),
        # The down projection of a prompt.
        dict(name="linear_prompt", op="linear", tokens=4096, rows=5120, cols=17408, source="rows", dtype="bf16",
             bias=False),
        # Gate and up of one decode step behind the block's norm.
        dict(name="gated_one_token", op="gated", tokens=1, rows=17408, cols=5120, source="norm", dtype="bf16"),
        # Gate and up of a serving batch behind the block's norm.
        dict(name="gated_batch", op="gated", tokens=64, rows=17408, cols=5120, source="norm", dtype="bf16"),
        # Ragged in every direction.
        dict(name="gated_odd", op="gated", tokens=301, rows=1023, cols=517, source="rows", dtype="fp16"),
        # Gate and up of a prompt behind the block's norm.
        dict(name="gated_prompt", op="gated", tokens=4096, rows=17408, cols=5120, source="norm", dtype="bf16"),
    ]


def _spread(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["norm", "join", "linear", "gated"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op in ("norm", "join"):
        case = dict(op=op, tokens=_spread(rng, 1, 8192), hidden=_spread(rng, 64, 8192),
                    kind=rng.choice(["rms", "layer"]), dtype=dtype)
        while case["tokens"] * case["hidden"] * (4 if dtype == "fp32" else 2) > 8192 * 5120 * 2:
            case["tokens"] = (case["tokens"] + 1) // 2
        if op == "join":
            case.update(gate=rng.choice(["none", "token", "channel", "full"]), residual=rng.choice([dtype, "fp32"]))
            if case["residual"] == "fp32" and dtype != "fp32":
                case["tokens"] = (case["tokens"] + 1) // 2
            if case["gate"] == "full":
                case["tokens"] = (case["tokens"] + 1) // 2
        return case
    most = 4096 * 5120 * 17408 * (2 if op == "gated" else 1)
    case = dict(op=op, tokens=_spread(rng, 1, 4096), rows=_spread(rng, 64, 17408), cols=_spread(rng, 64, 17408),
                dtype=dtype)
    while case["rows"] * case["cols"] > 5120 * 17408:
        case["rows"] = (case["rows"] + 1) // 2
    while case["tokens"] * case["rows"] * case["cols"] * (2 if op == "gated" else 1) > most:
        case["tokens"] = (case["tokens"] + 1) // 2
    # fp32 results come from rows that are int8 already: a value next to a rounding border of the quantisation would
    # otherwise say more than the product.
    case["source"] = "int8" if dtype == "fp32" else rng.choice(["int8", "rows"] + (["norm"] if op == "gated" else []))
    if op == "linear":
        case["bias"] = rng.choice([True, False])
    return case


def _int8(rows, cols, gen, device):
    """Gaussian values as int8, rows padded to 16 bytes as the framework's quantiser stores them."""
    q = torch.zeros((rows, (cols + 15) // 16 * 16), dtype=torch.int8, device=device)
    q[:, :cols] = (torch.randn((rows, cols), generator=gen, device=device) * 32).round_().clamp_(-127, 127)
    return q[:, :cols]


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)

    def randn(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(shape, generator=gen, device=device) * scale).to(dtype)

    state = dict(case)
    dtype = DTYPES[case["dtype"]]
    state["out_dtype"] = dtype
    if case["op"] in ("norm", "join"):
        t, h = case["tokens"], case["hidden"]
        names = ["next"] if case["op"] == "norm" else ["post", "next"]
        for name in names:
            state[name + "_weight"] = (1 + randn(h, scale=0.1)).to(dtype)
            state[name + "_bias"] = randn(h, scale=0.1, dtype=dtype) if case["kind"] == "layer" else None
        state["x"] = randn(t, h, dtype=dtype)
        if case["op"] == "join":
            state["residual_in"] = randn(t, h, scale=3.0, dtype=DTYPES[case["residual"]])
            shape = {"none": None, "token": (t, 1), "channel": (h,), "full": (t, h)}[case["gate"]]
            state["gate_in"] = None if shape is None else randn(*shape, dtype=dtype)
        return state
    t, n, k = case["tokens"], case["rows"], case["cols"]
    weights = 2 * n if case["op"] == "gated" else n
    state["wq"] = _int8(weights, k, gen, device)
    state["ws"] = (0.5 + torch.rand(weights, generator=gen, device=device)) / (32 * math.sqrt(k))
    state["bias_in"] = randn(n, scale=0.1, dtype=dtype) if case.get("bias") else None
    if case["source"] == "int8":
        state["xq"] = _int8(t, k, gen, device)
        state["xs"] = (0.5 + torch.rand(t, generator=gen, device=device)) / 32
    else:
        state["x"] = randn(t, k, dtype=dtype)
        if case["source"] == "norm":
            state["norm_weight"] = (1 + randn(k, scale=0.1)).to(dtype)
    return state


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "norm":
        t, h = case["tokens"], case["hidden"]
        return {"bytes": 2 * t * h * es + h * es, "flops": 6 * t * h}
    if case["op"] == "join":
        t, h = case["tokens"], case["hidden"]
        rs = 4 if case["residual"] == "fp32" else 2
        gate = {"none": 0, "token": t, "channel": h, "full": t * h}[case["gate"]]
        return {"bytes": 2 * t * h * (es + rs) + gate * es + 2 * h * es, "flops": 14 * t * h}
    t, n, k = case["tokens"], case["rows"], case["cols"]
    weights = 2 * n if case["op"] == "gated" else n
    read = t * k * (1 if case["source"] == "int8" else es)
    return {"bytes": weights * k + 4 * weights + read + t * n * es, "flops": 2 * t * weights * k}


# ---------------------------------------------------------------------------
# The plain forms.
# ---------------------------------------------------------------------------

def _norm(x, weight, bias, kind):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.float()
    return y if bias is None else y + bias.float()


def _quantize(x):
    amax = x.abs().amax(-1, keepdim=True)
    inverse = torch.where(amax >= SMALLEST_AMAX, 127 / amax, torch.zeros_like(amax))
    return torch.round(x * inverse), torch.where(amax >= SMALLEST_AMAX, amax / 127, torch.zeros_like(amax))


def _plain(s):
    if s["op"] == "norm":
        return _norm(s["x"].float(), s["next_weight"], s["next_bias"], s["kind"]).to(s["out_dtype"])
    if s["op"] == "join":
        branch = _norm(s["x"].float(), s["post_weight"], s["post_bias"], s["kind"])
        if s["gate_in"] is not None:
            branch = branch / (1 + torch.exp(-s["gate_in"].float()))
        residual = s["residual_in"].float() + 0.5 * branch
        out = _norm(residual, s["next_weight"], s["next_bias"], s["kind"])
        return residual.to(s["residual_in"].dtype), out.to(s["out_dtype"])
    if s["source"] == "int8":
        xq, xs = s["xq"].float(), s["xs"][:, None]
    elif s["source"] == "rows":
        xq, xs = _quantize(s["x"].float())
    else:
        xq, xs = _quantize(_norm(s["x"].float(), s["norm_weight"], None, "rms"))
    y = (xq @ s["wq"].float().t()) * xs * s["ws"]
    if s["op"] == "gated":
        gate, up = y.chunk(2, dim=1)
        y = gate / (1 + torch.exp(-gate)) * up
    if s["bias_in"] is not None:
        y = y + s["bias_in"].float()
    return y.to(s["out_dtype"])


# ---------------------------------------------------------------------------
# The framework's calls.
# ---------------------------------------------------------------------------

def _own(s):
    from qcc_b200.runtime.block_norm import BlockNorm, residual_norm
    from qcc_b200.runtime.int8_dense import int8_gated_linear, int8_linear, quantize_rows

    if s["op"] == "norm":
        return BlockNorm(s["next_weight"], s["next_bias"], kind=s["kind"], eps=EPS)(s["x"])
    if s["op"] == "join":
        post = BlockNorm(s["post_weight"], s["post_bias"], kind=s["kind"], eps=EPS)
        following = BlockNorm(s["next_weight"], s["next_bias"], kind=s["kind"], eps=EPS)
        return residual_norm(s["x"], s["residual_in"], post=post, gate=s["gate_in"],
                             gate_activation="sigmoid", branch_scale=0.5, next_norm=following)
    if s["source"] == "int8":
        xq, xs = s["xq"], s["xs"]
    elif s["source"] == "rows":
        xq, xs = quantize_rows(s["x"])
    else:
        xq, xs = BlockNorm(s["norm_weight"], kind="rms", eps=EPS)(s["x"], quantize=True)
    if s["op"] == "gated":
        return int8_gated_linear(xq, xs, s["wq"], s["ws"], out_dtype=s["out_dtype"])
    return int8_linear(xq, xs, s["wq"], s["ws"], bias=s["bias_in"], out_dtype=s["out_dtype"])


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# The definitions, in 64 bits.
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)

    def normed(v, weight, bias):
        n = v.shape[1]
        centre = torch.einsum("th->t", v) / n if case.get("kind") == "layer" else torch.zeros_like(v[:, 0])
        v = v - centre[:, None]
        size = torch.sqrt(torch.einsum("th,th->t", v, v) / n + EPS)
        v = v / size[:, None] * weight.double()
        return v if bias is None else v + bias.double()

    if case["op"] == "norm":
        return normed(s["x"].double(), s["next_weight"], s["next_bias"])
    if case["op"] == "join":
        branch = normed(s["x"].double(), s["post_weight"], s["post_bias"])
        if s["gate_in"] is not None:
            branch = branch * torch.sigmoid(s["gate_in"].double())
        residual = torch.add(s["residual_in"].double(), branch, alpha=0.5)
        return residual, normed(residual, s["next_weight"], s["next_bias"])
    if case["source"] == "int8":
        x = s["xq"].double() * s["xs"].double()[:, None]
    else:
        v = s["x"].double()
        if case["source"] == "norm":
            v = normed(v, s["norm_weight"], None)
        step = v.abs().max(dim=1, keepdim=True).values / 127
        x = torch.where(step > 0, torch.round(v / step.clamp_min(1e-300)) * step, 0.0)
    pieces = []
    for rows in torch.arange(s["wq"].shape[0], device=x.device).split(4096):  # bounds the weight's copy in 64 bits
        pieces.append(torch.einsum("tk,nk->tn", x, s["wq"][rows].double() * s["ws"][rows].double()[:, None]))
    y = torch.cat(pieces, dim=1)
    if case["op"] == "gated":
        n = case["rows"]
        y = torch.nn.functional.silu(y[:, :n]) * y[:, n:]
    return y if s["bias_in"] is None else y + s["bias_in"].double()
