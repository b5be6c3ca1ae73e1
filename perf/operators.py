"""Cases of the four-bit (MXFP4) operators and of the mixture-of-experts layer.

Four-bit matrices hold blocks of 32 values along a row: 16 bytes of e2m1 codes (value 2i in the
low half of byte i) and one power-of-two scale byte (2^(b - 127)); a ragged last block is filled
with zeros. ``run`` computes an operator in its plain form, elementary torch operations in 32 bits
rounded once at the end (router logits in 64 bits: an expert next to the border of the selection
is decided there), or, where ``own`` is set, through the framework's calls.
"""
import sys
from pathlib import Path

import torch

own = False

TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = 32
CODES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
_package = None


def _framework():
    global _package
    if _package is None:
        path = str(Path(__file__).resolve().parents[1] / "cuda-kernel_b200")
        if path not in sys.path:
            sys.path.insert(1, path)
        import swiglu_b200
        _package = swiglu_b200
    return _package


# ------------------------------------------------------------------ cases

def listed():
    return [
        # one token's activations, as they are rounded before a product: the smallest call
        {"name": "quantize-token", "op": "quantize", "type": "fp16", "rows": 1, "cols": 14336},
        # a layer's gate matrix, rounded once when a model is loaded, and read back
        {"name": "quantize-weights", "op": "quantize", "type": "bf16", "rows": 14336, "cols": 4096},
        # decode of one token: the up projection of the large layer, read once at four bits
        {"name": "project-token", "op": "project", "type": "fp16", "out": "fp16", "tokens": 1, "rows": 14336,
         "cols": 4096, "bias": False, "residual": False},
        # eight sequences decoded together: a down projection with bias and residual, fp32 out as the layer gives it
        {"name": "project-batch", "op": "project", "type": "bf16", "out": "fp32", "tokens": 8, "rows": 4096,
         "cols": 14336, "bias": True, "residual": True},
        # a prompt through the smaller layer
        {"name": "project-prompt", "op": "project", "type": "fp16", "out": "fp16", "tokens": 512, "rows": 5632,
         "cols": 2048, "bias": False, "residual": False},
        # both sides in four bits: a few tokens, a ragged batch, and a long prompt
        {"name": "matmul-few", "op": "matmul", "type": "fp16", "tokens": 16, "rows": 14336, "cols": 4096,
         "bias": False, "residual": False},
        {"name": "matmul-ragged", "op": "matmul", "type": "bf16", "tokens": 333, "rows": 5631, "cols": 2047,
         "bias": True, "residual": False},
        {"name": "matmul-prompt", "op": "matmul", "type": "bf16", "tokens": 4096, "rows": 14336, "cols": 4096,
         "bias": False, "residual": True},
        # decode of one token through a small layer, where the call's latency counts
        {"name": "moe-small", "op": "moe", "type": "fp16", "weights": "fp16", "tokens": 1, "experts": 8, "topk": 2,
         "hidden": 512, "inter": 1376, "renormalize": True},
        # decode of one token through few experts of the smaller layer's size
        {"name": "moe-token", "op": "moe", "type": "fp16", "weights": "fp16", "tokens": 1, "experts": 8, "topk": 2,
         "hidden": 2048, "inter": 5632, "renormalize": True},
        # many narrow experts, a batch of decoded tokens that reaches most of them
        {"name": "moe-narrow", "op": "moe", "type": "bf16", "weights": "bf16", "tokens": 16, "experts": 64, "topk": 8,
         "hidden": 2048, "inter": 1376, "renormalize": False},
        # the large layer as experts in four bits: the most that a call reads
        {"name": "moe-four-bit", "op": "moe", "type": "fp16", "weights": "mx4", "tokens": 32, "experts": 8, "topk": 2,
         "hidden": 4096, "inter": 14336, "renormalize": True},
    ]


def _size(rng, low, high):
    """Spread over the logarithm; two in three rounded to a multiple of 32 where that fits."""
    n = int(round(low * (high / low) ** rng.random()))
    if n > BLOCK and rng.random() < 0.67:
        n = n // BLOCK * BLOCK
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(["quantize", "project", "matmul", "moe"])
    if op == "quantize":
        rows, cols = _size(rng, 1, 16384), _size(rng, 1, 16384)
        rows = max(1, min(rows, 14336 * 4096 // cols))
        return {"op": op, "type": rng.choice(["fp16", "bf16", "fp32"]), "rows": rows, "cols": cols}
    if op == "project":
        rows, cols = _size(rng, 64, 14336), _size(rng, 64, 14336)
        rows = max(1, min(rows, 14336 * 4096 // cols))
        tokens = max(1, min(_size(rng, 1, 512), 512 * 5632 * 2048 // (rows * cols)))
        kind = rng.choice(["fp16", "bf16"])
        return {"op": op, "type": kind, "out": rng.choice([kind, "fp32"]), "tokens": tokens, "rows": rows,
                "cols": cols, "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    if op == "matmul":
        rows, cols = _size(rng, 64, 14336), _size(rng, 64, 14336)
        rows = max(1, min(rows, 14336 * 4096 // cols))
        return {"op": op, "type": rng.choice(["fp16", "bf16"]), "tokens": _size(rng, 1, 4096), "rows": rows,
                "cols": cols, "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    experts = _size(rng, 2, 128)
    hidden, inter = _size(rng, 64, 4096), _size(rng, 64, 14336)
    inter = max(1, min(inter, 8 * 4096 * 14336 // (experts * hidden)))
    kind = rng.choice(["fp16", "bf16"])
    return {"op": op, "type": kind, "weights": rng.choice([kind, "mx4"]), "tokens": _size(rng, 1, 64),
            "experts": experts, "topk": rng.randint(1, min(8, experts)), "hidden": hidden, "inter": inter,
            "renormalize": rng.random() < 0.5}


# ------------------------------------------------------------------ inputs

def _normal(g, shape, scale, kind):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(TYPES[kind])


def _four_bit(g, shape, scale):
    """A normal matrix in four bits, as a model's weights are after loading: (codes, scales)."""
    lead, cols = shape[:-1], shape[-1]
    return _encode(torch.randn((*lead, cols), generator=g, device="cuda", dtype=torch.float32) * scale)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, kind = case["op"], case.get("type")
    state = {"case": case}
    if op == "quantize":
        rows, cols = case["rows"], case["cols"]
        blocks = -(-cols // BLOCK)
        state["x"] = _normal(g, (rows, cols), 1.0 if rows == 1 else cols ** -0.5, kind)
        state["codes"] = torch.empty((rows, blocks * 16), dtype=torch.uint8, device="cuda")
        state["scales"] = torch.empty((rows, blocks), dtype=torch.uint8, device="cuda")
        state["out"] = torch.empty_like(state["x"])
        return state
    if op in ("project", "matmul"):
        tokens, rows, cols = case["tokens"], case["rows"], case["cols"]
        if op == "project":
            state["x"] = _normal(g, (tokens, cols), 1.0, kind)
        else:
            state["xq"], state["xs"] = _four_bit(g, (tokens, cols), 1.0)
        state["wq"], state["ws"] = _four_bit(g, (rows, cols), cols ** -0.5)
        state["bias"] = _normal(g, (rows,), 0.02, kind) if case["bias"] else None
        state["residual"] = _normal(g, (tokens, rows), 1.0, kind) if case["residual"] else None
        state["out"] = torch.empty((tokens, rows), dtype=TYPES[case.get("out", kind)], device="cuda")
        return state
    tokens, experts, hidden, inter = case["tokens"], case["experts"], case["hidden"], case["inter"]
    state["x"] = _normal(g, (tokens, hidden), 1.0, kind)
    state["router"] = _normal(g, (experts, hidden), hidden ** -0.5, kind)
    for name, rows, cols in (("gate", inter, hidden), ("up", inter, hidden), ("down", hidden, inter)):
        state[name + "_scales"] = None
        if case["weights"] == "mx4":
            blocks = -(-cols // BLOCK)
            state[name] = torch.empty((experts, rows, blocks * 16), dtype=torch.uint8, device="cuda")
            state[name + "_scales"] = torch.empty((experts, rows, blocks), dtype=torch.uint8, device="cuda")
            for e in range(experts):
                state[name][e], state[name + "_scales"][e] = _four_bit(g, (rows, cols), cols ** -0.5)
        else:
            state[name] = torch.empty((experts, rows, cols), dtype=TYPES[kind], device="cuda")
            for e in range(experts):
                state[name][e] = _normal(g, (rows, cols), cols ** -0.5, kind)
    state["y"] = torch.empty_like(state["x"])
    state["ids"] = torch.empty((tokens, case["topk"]), dtype=torch.int32, device="cuda")
    state["weights"] = torch.empty((tokens, case["topk"]), dtype=torch.float32, device="cuda")
    return state


# ------------------------------------------------------------------ plain forms

def _encode(x):
    """Rows of fp32 values to (codes, scales): the block's scale is 2^(floor(log2 max) - 2), a
    value goes to the nearest of +-{0, .5, 1, 1.5, 2, 3, 4, 6}, ties to the even code, larger ones
    to 6; a block that holds a NaN or an infinity is NaN as a whole (scale byte 255)."""
    lead, cols = x.shape[:-1], x.shape[-1]
    blocks = -(-cols // BLOCK)
    v = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).reshape(*lead, blocks, BLOCK)
    bits = v.view(torch.int32) & 0x7FFFFFFF
    top = bits.amax(-1)
    byte = torch.where(top >= 0x7F800000, 255, torch.clamp((top >> 23) - 2, min=0))
    up = torch.where(byte == 255, 0, (254 - byte) << 23).to(torch.int32).view(torch.float32)  # 2^(127 - byte)
    a = bits.view(torch.float32) * up.unsqueeze(-1)
    steps = torch.where(a < 2, torch.round(a * 2), torch.where(a < 4, torch.round(a) + 2, torch.round(a / 2) + 4))
    code = torch.clamp(steps, max=7).to(torch.uint8) | torch.where(v.view(torch.int32) < 0, 8, 0).to(torch.uint8)
    code = torch.where((byte == 255).unsqueeze(-1), torch.zeros_like(code), code)
    packed = code[..., 0::2] | (code[..., 1::2] << 4)
    return packed.reshape(*lead, blocks * 16), byte.to(torch.uint8)


def _decode(q, s, cols):
    """The fp32 values that codes and scales stand for."""
    table = torch.tensor(CODES + tuple(-c for c in CODES), dtype=torch.float32, device=q.device)
    pairs = torch.stack((table.repeat(16), table.repeat_interleave(16)), -1)
    v = pairs[q.int()].reshape(*s.shape, BLOCK)
    scale = torch.where(s == 0, 0x00400000, torch.where(s == 255, 0x7FC00000, s.int() << 23)).to(torch.int32)
    scale = scale.view(torch.float32)  # 2^(s - 127), NaN for 255
    return (v * scale.unsqueeze(-1)).flatten(-2)[..., :cols]


def _product(x, w, bias, residual):
    y = x @ w.transpose(-1, -2)
    if bias is not None:
        y = y + bias.float()
    if residual is not None:
        y = y + residual.float()
    return y


def _moe(s, case):
    x, topk = s["x"].float(), case["topk"]
    tokens, experts = x.shape[0], case["experts"]
    logits = s["x"].double() @ s["router"].double().T
    value, order = torch.sort(logits, dim=-1, descending=True, stable=True)
    ids = order[:, :topk]
    weight = torch.exp(value[:, :topk] - value[:, :1])
    weight = weight / (weight if case["renormalize"] else torch.exp(value - value[:, :1])).sum(-1, keepdim=True)
    weight = weight.float()
    few = tokens * topk < experts
    pick = ids.reshape(-1) if few else slice(None)

    def matrix(name, cols):
        if case["weights"] == "mx4":
            return _decode(s[name][pick], s[name + "_scales"][pick], cols)
        return s[name][pick].float()

    if few:  # only the selected experts' weights, one copy for each token and place
        row = x.repeat_interleave(topk, 0).unsqueeze(-1)
        g, u = (matrix("gate", case["hidden"]) @ row), (matrix("up", case["hidden"]) @ row)
        h = g / (1 + torch.exp(-g)) * u
        y = (matrix("down", case["inter"]) @ h).reshape(tokens, topk, -1)
        y = (y * weight.unsqueeze(-1)).sum(1)
    else:  # every expert on every token, those not selected with weight zero
        mix = torch.zeros((tokens, experts), device=x.device).scatter_(1, ids, weight)
        g, u = x @ matrix("gate", case["hidden"]).transpose(1, 2), x @ matrix("up", case["hidden"]).transpose(1, 2)
        h = g / (1 + torch.exp(-g)) * u * mix.T.unsqueeze(-1)
        y = (h @ matrix("down", case["inter"]).transpose(1, 2)).sum(0)
    return y.to(s["x"].dtype), ids.int(), weight


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        f = _framework()
        if op == "quantize":
            f.mx4_quantize_out(state["x"], state["codes"], state["scales"])
            f.mx4_dequantize_out(state["codes"], state["scales"], state["out"])
            return state["out"]
        if op == "project":
            f.mx4_project_out(state["x"], state["wq"], state["ws"], state["out"], state["bias"], state["residual"])
            return state["out"]
        if op == "matmul":
            f.mx4_matmul_out(state["xq"], state["xs"], state["wq"], state["ws"], state["out"], state["bias"],
                             state["residual"])
            return state["out"]
        if "workspace" not in state:
            state["workspace"] = f.moe_workspace(case["tokens"], case["experts"], case["topk"], case["inter"])
        f.moe_out(state["x"], state["router"], state["gate"], state["up"], state["down"], state["y"],
                  state["workspace"], case["topk"], renormalize=case["renormalize"],
                  gate_scales=state["gate_scales"], up_scales=state["up_scales"], down_scales=state["down_scales"],
                  ids=state["ids"], weights=state["weights"])
        return state["y"], state["ids"], state["weights"]
    if op == "quantize":
        return _decode(*_encode(state["x"].float()), case["cols"]).to(state["x"].dtype)
    if op == "project":
        w = _decode(state["wq"], state["ws"], case["cols"])
        return _product(state["x"].float(), w, state["bias"], state["residual"]).to(TYPES[case["out"]])
    if op == "matmul":
        x = _decode(state["xq"], state["xs"], case["cols"])
        w = _decode(state["wq"], state["ws"], case["cols"])
        return _product(x, w, state["bias"], state["residual"]).to(TYPES[case["type"]])
    return _moe(state, case)


# ------------------------------------------------------------------ least work

def _matrix_bytes(rows, cols, kind):
    return rows * -(-cols // BLOCK) * 17 if kind == "mx4" else rows * cols * (4 if kind == "fp32" else 2)


def work(case):
    op = case["op"]
    if op == "quantize":  # written in four bits, read back from them
        rows, cols = case["rows"], case["cols"]
        return {"bytes": 2 * _matrix_bytes(rows, cols, case["type"]) + 2 * _matrix_bytes(rows, cols, "mx4"),
                "flops": 4 * rows * cols}
    if op in ("project", "matmul"):
        tokens, rows, cols = case["tokens"], case["rows"], case["cols"]
        size = _matrix_bytes(tokens, cols, case["type"] if op == "project" else "mx4") + _matrix_bytes(rows, cols, "mx4")
        size += _matrix_bytes(tokens, rows, case.get("out", case["type"]))
        size += 2 * rows * case["bias"] + 2 * tokens * rows * case["residual"]
        return {"bytes": size, "flops": 2 * tokens * rows * cols}
    tokens, experts, topk = case["tokens"], case["experts"], case["topk"]
    hidden, inter = case["hidden"], case["inter"]
    # experts that a batch reaches, expected for independent selections
    reached = experts * (1 - (1 - topk / experts) ** tokens)
    expert = 2 * _matrix_bytes(inter, hidden, case["weights"]) + _matrix_bytes(hidden, inter, case["weights"])
    return {"bytes": int(reached * expert) + 2 * (2 * tokens + experts) * hidden + 8 * tokens * topk,
            "flops": 2 * tokens * (topk * 3 * hidden * inter + experts * hidden)}


# ------------------------------------------------------------------ the definitions in 64 bits

def _values64(q, s, cols):
    low, high = (q & 15).long(), (q >> 4).long()
    code = torch.stack((low, high), -1).flatten(-2)
    exponent, half = (code & 7) >> 1, (code & 1).double()
    size = torch.where(exponent == 0, half * 0.5, (1 + half * 0.5) * torch.ones_like(exponent).bitwise_left_shift(exponent) / 2)
    v = torch.where(code >= 8, -size, size)
    scale = ((s.long() + (1023 - 127)) << 52).view(torch.float64)
    scale[s == 255] = float("nan")
    return (v * scale.repeat_interleave(BLOCK, -1))[..., :cols]


def _rounded64(x):
    """Each value to the nearest one that its block can hold, by distance: rows of 64-bit values."""
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros((rows, blocks * BLOCK), dtype=torch.float64, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, blocks, BLOCK)
    top = v.abs().amax(-1, keepdim=True)
    _, e = torch.frexp(torch.where(top == 0, torch.ones_like(top), top))  # top = m 2^e, m in [.5, 1)
    unit = ((torch.clamp(e.long() - 1 - 2, min=-127) + 1023) << 52).view(torch.float64)
    a = v.abs() / unit
    best = torch.zeros_like(a)
    lower = CODES[0]
    for i, upper in enumerate(CODES[1:], 1):
        middle = (lower + upper) / 2
        best = torch.where((a > middle) | ((a == middle) & (i % 2 == 0)), torch.full_like(a, upper), best)
        lower = upper
    return (torch.sign(v) * best * unit).reshape(rows, blocks * BLOCK)[:, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "quantize":
        return torch.cat([_rounded64(part.double()) for part in s["x"].split(2048)])
    if op in ("project", "matmul"):
        x = s["x"].double() if op == "project" else _values64(s["xq"], s["xs"], case["cols"])
        y = torch.matmul(x, _values64(s["wq"], s["ws"], case["cols"]).T)
        if case["bias"]:
            y += s["bias"].double()
        if case["residual"]:
            y += s["residual"].double()
        return y
    x = s["x"].double()
    logits = torch.matmul(x, s["router"].double().T)
    share = torch.softmax(logits, -1)
    rank = torch.argsort(-logits, dim=-1, stable=True)[:, :case["topk"]]
    weight = torch.gather(share, 1, rank)
    if case["renormalize"]:
        weight = weight / weight.sum(-1, keepdim=True)
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, place = torch.nonzero(rank == e, as_tuple=True)
        if token.numel() == 0:
            continue
        m = {}
        for name, cols in (("gate", case["hidden"]), ("up", case["hidden"]), ("down", case["inter"])):
            scales = s[name + "_scales"]
            m[name] = s[name][e].double() if scales is None else _values64(s[name][e], scales[e], cols)
        g, u = x[token] @ m["gate"].T, x[token] @ m["up"].T
        out = (g * torch.sigmoid(g) * u) @ m["down"].T
        y.index_add_(0, token, out * weight[token, place].unsqueeze(-1))
    return y, rank.int(), weight
