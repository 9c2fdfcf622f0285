"""Cases of the 8-bit projection operators: what is timed, on which inputs, and what the right answer is.

A decoder layer around the quantised attention is four matrix products with codes of 8 bits on both sides and one scale
a token and one a channel (queries/keys/values, attention output, gate and up, down), and the kernels that make the
tokens' codes: the root-mean-square norm with the residual's addition, the gated activation, and plain rows.

    norm     rms_norm(x, weight, eps, residual)   -> codes and scales of the normed rows, and the new residual
    gated    silu_mul(gate, up)                   -> codes and scales of silu(gate) * up
    rows     quantize_rows(x)                     -> codes and scales of x
    linear   linear(rows, weight, bias, residual) -> (codes . codes^T) * scale_token * scale_channel + bias + residual

The operators that end in codes are followed by what turns codes back into values, so that both forms return numbers of the
inputs' type.
"""
import math

import torch

own = False

EPS = 1e-5
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


# ---- cases -----------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one token of one sequence on its way into a layer: latency alone
        dict(name="norm token", op="norm", tokens=1, width=4096, type="bf16", residual=True, padding=0),
        # a prompt batch of 16,384 tokens, width of 28 heads
        dict(name="norm prompt", op="norm", tokens=16384, width=3584, type="bf16", residual=True, padding=0),
        # a ragged batch with padded rows behind the last sequence, odd width, no residual (first layer)
        dict(name="norm ragged", op="norm", tokens=333, width=5001, type="fp16", residual=False, padding=13),
        # the gated activation of a decode step of 16 sequences
        dict(name="gated batch", op="gated", tokens=16, width=8192, type="bf16", padding=0),
        # the same in a prompt pass
        dict(name="gated prompt", op="gated", tokens=8192, width=14336, type="bf16", padding=0),
        # attention outputs of a decode step of 32 sequences, before the output projection
        dict(name="rows batch", op="rows", tokens=32, width=3584, type="bf16", padding=0),
        # attention outputs of a prompt batch, 32 heads of 128
        dict(name="rows prompt", op="rows", tokens=16384, width=4096, type="bf16", padding=0),
        # one token through the merged query, key and value projection (32 + 2 * 8 heads of 128)
        dict(name="linear token", op="linear", tokens=1, outputs=6144, width=4096, type="bf16", bias=False, residual=False),
        # a decode step of 32 sequences through a projection with biases (28 + 2 * 4 heads of 128)
        dict(name="linear batch", op="linear", tokens=32, outputs=4608, width=3584, type="bf16", bias=True, residual=False),
        # logits of 16 sequences over the whole vocabulary
        dict(name="linear logits", op="linear", tokens=16, outputs=128256, width=4096, type="fp32", bias=False, residual=False),
        # nothing is a multiple of anything
        dict(name="linear ragged", op="linear", tokens=777, outputs=5003, width=2051, type="fp16", bias=True, residual=False),
        # the down projection of a prompt batch, added to the residual stream
        dict(name="linear prompt", op="linear", tokens=16384, outputs=4096, width=14336, type="bf16", bias=False, residual=True),
    ]


def draw(rng):
    def spread(lo, hi):
        n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
        if rng.random() < 0.5:            # half of the sizes as models have them, half as they come
            unit = 128 if n >= 1024 else 16 if n >= 64 else 1
            n = max(unit, n // unit * unit)
        return min(max(n, lo), hi)

    op = rng.choice(("linear", "linear", "linear", "norm", "gated", "rows"))
    kind = rng.choice(("bf16", "bf16", "fp16"))
    if op == "linear":
        while True:
            tokens, outputs, width = spread(1, 16384), spread(96, 32768), spread(96, 16384)
            if tokens * outputs * width <= 16384 * 4096 * 14336 // 2 and tokens * outputs <= 16384 * 8192:
                break
        return dict(op=op, tokens=tokens, outputs=outputs, width=width, type=rng.choice((kind, "fp32")),
                    bias=rng.random() < 0.4, residual=rng.random() < 0.4)
    while True:
        tokens, width = spread(1, 16384), spread(96, 16384)
        if tokens * width <= 8192 * 6144:
            break
    case = dict(op=op, tokens=tokens, width=width, type=kind, padding=rng.choice((0, 0, tokens // 8)))
    if op == "norm":
        case["residual"] = rng.random() < 0.7
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _pitched(rows, width, dtype, device):
    """Rows of codes lie a multiple of 16 bytes apart."""
    return torch.zeros(rows, -(-width // 16) * 16, dtype=dtype, device=device)[:, :width]


def _codes_of(x):
    """Symmetric codes of 8 bits and one scale a row."""
    scales = x.abs().amax(1, keepdim=True).clamp(min=1e-20) / 127
    codes = _pitched(x.shape[0], x.shape[1], torch.int8, x.device)
    codes.copy_(torch.round(x / scales).clamp(-127, 127))
    return codes, scales[:, 0].contiguous()


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    dtype, tokens, width = TYPES[case["type"]], case["tokens"], case["width"]
    # activations: N(0,1) with one channel in a hundred twenty times as wide
    outliers = torch.where(torch.rand(width, generator=gen, device="cuda") < 0.01, 20.0, 1.0)
    state = dict(case=case)
    if case["op"] == "linear":
        state["codes"], state["scales"] = _codes_of(normal(tokens, width) * outliers)
        state["wcodes"] = _pitched(case["outputs"], width, torch.int8, "cuda")
        state["wscales"] = torch.empty(case["outputs"], device="cuda")
        for lo in range(0, case["outputs"], 16384):
            part = slice(lo, min(lo + 16384, case["outputs"]))
            codes, state["wscales"][part] = _codes_of(0.02 * normal(part.stop - lo, width))
            state["wcodes"][part].copy_(codes)
        state["bias"] = normal(case["outputs"]).to(dtype) if case["bias"] else None
        state["residual"] = (2 * normal(tokens, case["outputs"])).to(dtype) if case["residual"] else None
        return state
    live = (torch.arange(tokens, device="cuda") < tokens - case["padding"])[:, None]
    if case["op"] == "norm":
        state["x"] = (normal(tokens, width) * live).to(dtype)
        state["weight"] = (1 + 0.1 * normal(width)).to(dtype)
        state["residual"] = (3 * normal(tokens, width) * outliers * live).to(dtype) if case["residual"] else None
    elif case["op"] == "gated":
        # gate and up come side by side out of one product
        both = torch.empty(tokens, 2 * width, dtype=dtype, device="cuda")
        both[:, :width] = 2 * normal(tokens, width) * live
        both[:, width:] = normal(tokens, width) * outliers * live
        state["gate"], state["up"] = both[:, :width], both[:, width:]
    else:
        state["x"] = (normal(tokens, width) * outliers * live).to(dtype)
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

_kept = {}


def _ops():
    if "ops" not in _kept:
        from triattention_b200.kernels.extension import load_extension
        from triattention_b200.kernels.linear import Int8Ops, Int8Rows
        _kept["ops"], _kept["rows"] = Int8Ops(load_extension()), Int8Rows
    return _kept["ops"], _kept["rows"]


def _run_own(state):
    ops, rows = _ops()
    op = state["case"]["op"]
    if op == "linear":
        return ops.linear(rows(state["codes"], state["scales"]), rows(state["wcodes"], state["wscales"]), bias=state["bias"],
                          residual=state["residual"], dtype=TYPES[state["case"]["type"]])
    if op == "norm":
        if state["residual"] is None:
            return dict(values=ops.dequantize(ops.rms_norm(state["x"], state["weight"], EPS)))
        normed, residual = ops.rms_norm(state["x"], state["weight"], EPS, residual=state["residual"])
        return dict(values=ops.dequantize(normed), residual=residual)
    if op == "gated":
        return dict(values=ops.dequantize(ops.silu_mul(state["gate"], state["up"])))
    return dict(values=ops.dequantize(ops.quantize_rows(state["x"])))


def _through_codes(y, dtype):
    scales = y.abs().amax(1, keepdim=True) / 127
    codes = torch.round(y / torch.where(scales > 0, scales, 1.0))
    return (codes * scales).to(dtype)


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    dtype = TYPES[case["type"]]
    if case["op"] == "linear":
        y = (state["codes"].float() @ state["wcodes"].float().T) * state["wscales"] * state["scales"][:, None]
        if state["bias"] is not None:
            y = y + state["bias"].float()
        if state["residual"] is not None:
            y = y + state["residual"].float()
        return y.to(dtype)
    if case["op"] == "norm":
        h = state["x"] if state["residual"] is None else (state["x"].float() + state["residual"].float()).to(dtype)
        wide = h.float()
        y = wide * torch.rsqrt(wide.square().mean(1, keepdim=True) + EPS) * state["weight"].float()
        values = dict(values=_through_codes(y, dtype))
        return values if state["residual"] is None else dict(values, residual=h)
    if case["op"] == "gated":
        gate = state["gate"].float()
        return dict(values=_through_codes(gate / (1 + torch.exp(-gate)) * state["up"].float(), dtype))
    return dict(values=_through_codes(state["x"].float(), dtype))


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    tokens, width, size = case["tokens"], case["width"], SIZE[case["type"]]
    if case["op"] == "linear":
        outputs = case["outputs"]
        moved = tokens * width + outputs * width + 4 * (tokens + outputs) + tokens * outputs * size
        moved += outputs * size * case["bias"] + tokens * outputs * size * case["residual"]
        return dict(bytes=moved, flops=2 * tokens * outputs * width)
    cells = tokens * width
    read = {"norm": 1 + case.get("residual", False), "gated": 2, "rows": 1}[case["op"]]
    moved = cells * size * read + cells + 4 * tokens + cells * size     # inputs, codes, scales, the codes' values
    if case["op"] == "norm":
        moved += width * size + cells * size * case["residual"]
    return dict(bytes=moved, flops=cells * {"norm": 8, "gated": 10, "rows": 4}[case["op"]])


# ---- the definition in 64 bits ---------------------------------------------------------------------------------------

def _nearest_step(y):
    """Each row on the grid of 255 even steps that spans its largest magnitude."""
    largest = y.abs().max(dim=1).values[:, None]
    step = torch.where(largest > 0, largest, torch.ones_like(largest)) / 127.0
    return torch.floor(y / step + 0.5) * step


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        x, w = s["codes"].double() * s["scales"].double()[:, None], s["wcodes"].double() * s["wscales"].double()[:, None]
        y = x @ w.T
        for more in (s["bias"], s["residual"]):
            if more is not None:
                y += more.double()
        return y
    if case["op"] == "norm":
        total = s["x"].double() if s["residual"] is None else s["x"].double() + s["residual"].double()
        kept = total.to(TYPES[case["type"]]).double()       # the stream that later layers see is what is normed
        power = (kept * kept).sum(1, keepdim=True) / case["width"]
        values = _nearest_step(kept / (power + EPS).sqrt() * s["weight"].double())
        return dict(values=values) if s["residual"] is None else dict(values=values, residual=total)
    if case["op"] == "gated":
        return dict(values=_nearest_step(s["gate"].double() * torch.sigmoid(s["gate"].double()) * s["up"].double()))
    return dict(values=_nearest_step(s["x"].double()))
