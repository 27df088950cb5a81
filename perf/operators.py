"""Measured cases of the operators around 4-bit feed-forwards and of expert layers for a few tokens.

Four kinds of pass, by the case's ``op``:

quantize  a matrix to microscaled 4-bit numbers (blocks of 32 elements along the width share a power of two, an element is
          sign, two bits of exponent, one of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and back to the values these stand for
linear    act(x W^T + b) + residual with W in that form: one token's step, a batch's, a prompt's
grouped   the same product over rows sorted by expert, in row tiles that meet one expert's matrix each, with the gated unit or
          an activation as its epilogue
moe       a whole expert layer for one to eight tokens: routing, the chosen units, the shared unit, the weighted sum

How the 4-bit matrices lie in memory is part of the operators' interface: four blocks of 32 elements (128 of a row; a row is
padded with zeros to whole groups) are 64 bytes, sixteen 32-bit words; word 4 t + b holds elements 8 t .. 8 t + 7 of block b,
its elements 0, 2, 4, 6 in bits 0 .. 15 and 1, 3, 5, 7 in bits 16 .. 31, four bits each, from the lowest up. A block's scale is
one byte s, standing for 2^(s - 127); scales lie in block order.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16}
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
GROUP, BLOCK = 128, 32
TILES = (16, 32, 64, 128)


# ------------------------------------------------------------------ the cases

def _quantize(rows, width, dtype):
    return {"op": "quantize", "rows": rows, "width": width, "dtype": dtype}


def _linear(rows, out, width, activation="none", bias=False, residual=False, out_dtype="bfloat16"):
    return {"op": "linear", "rows": rows, "out": out, "width": width, "activation": activation, "bias": bias, "residual": residual,
            "out_dtype": out_dtype}


def _grouped(tokens, top, experts, out, width, unit, out_dtype="bfloat16", row_scale=False):
    return {"op": "grouped", "tokens": tokens, "top": top, "experts": experts, "out": out, "width": width, "unit": unit,
            "out_dtype": out_dtype, "row_scale": row_scale}


def _moe(tokens, width, inner, experts, top, weights, unit, score="sigmoid", groups=1, keep=1, scale=1.0, correction=False,
         renormalize=False, identity=0, weight_input=False, shared=0, shared_gate=False):
    return {"op": "moe", "tokens": tokens, "width": width, "inner": inner, "experts": experts, "top": top, "weights": weights,
            "unit": unit, "score": score, "groups": groups, "keep": keep, "scale": scale, "correction": correction,
            "renormalize": renormalize, "identity": identity, "weight_input": weight_input, "shared": shared,
            "shared_gate": shared_gate}


def listed():
    return [
        # loading a model: one up matrix of a GPT-2 XL layer; the stacked gate and up matrices of sixteen experts
        {"name": "quantize_up_6400x1600", **_quantize(6400, 1600, "bfloat16")},
        {"name": "quantize_stack_51200x1600", **_quantize(51200, 1600, "float32")},
        # a decode step of one request: GPT-2 XL's up product with its activation
        {"name": "linear_1_up", **_linear(1, 6400, 1600, "gelu_new", bias=True)},
        # ... of eight requests: its down product, added into the float32 stream
        {"name": "linear_8_down", **_linear(8, 1600, 6400, bias=True, residual=True, out_dtype="float32")},
        # a mixed step of a model of odd sizes
        {"name": "linear_61_odd", **_linear(61, 1030, 1000, "gelu", bias=True)},
        # a prompt of 2,048 tokens: the up product
        {"name": "linear_prompt_up", **_linear(2048, 6400, 1600, "gelu_new", bias=True)},
        # 64 requests decoding in an expert model: gate and up with the silu unit, sixteen experts, two a token
        {"name": "grouped_64_silu", **_grouped(64, 2, 16, 1600, 1600, "silu")},
        # a prompt of 2,048 tokens in the wider one: the experts' down product
        {"name": "grouped_prompt_down", **_grouped(2048, 2, 16, 2048, 2048, "none", out_dtype="float32")},
        # one request decoding: router within groups, gated shared unit
        {"name": "moe_1_shared", **_moe(1, 1600, 1600, 16, 2, "bfloat16", "silu", groups=4, keep=2, scale=2.5, shared=1600, shared_gate=True)},
        # eight requests: experts by a table of token ids, clamped units
        {"name": "moe_8_table", **_moe(8, 2048, 2048, 16, 2, "bfloat16", "clamped_swish", score="table", shared=2048)},
        # eight requests, many small 4-bit experts, softmax scores with identity outputs
        {"name": "moe_8_mx4", **_moe(8, 2048, 1024, 64, 8, "mx4", "silu", score="softmax", correction=True, renormalize=True, identity=4)},
        # five requests of the float32 engine: plain units, weights on their inputs
        {"name": "moe_5_float32", **_moe(5, 1600, 1600, 16, 2, "float32", "relu2", weight_input=True)},
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("quantize", "linear", "linear", "grouped", "moe", "moe"))
    if op == "quantize":
        return _quantize(_log(rng, 1, 16384), _log(rng, 16, 4900), rng.choice(("float32", "bfloat16")))
    if op == "linear":
        rows, out, width = _log(rng, 1, 2048), _log(rng, 48, 6400), _log(rng, 48, 1600)
        if rows <= 64 and rng.random() < 0.5:
            width = _log(rng, 1600, 6400)
        if rng.random() < 0.5:
            width = -(-width // 32) * 32
        residual = rng.random() < 0.5
        return _linear(rows, out, width, "none" if residual else rng.choice(("none", "gelu_new", "gelu", "relu2")),
                       bias=rng.random() < 0.5, residual=residual, out_dtype="float32" if residual else rng.choice(("bfloat16", "float32")))
    experts = rng.choice((4, 8, 16, 24, 32))
    top = rng.randint(1, 4)
    if op == "grouped":
        unit = rng.choice(("none", "relu2", "silu", "clamped_swish", "gelu_tanh"))
        plain = unit in ("none", "relu2")
        return _grouped(_log(rng, 1, 2048), top, experts, _log(rng, 64, 1600), 8 * _log(rng, 8, 200), unit,
                        out_dtype=rng.choice(("bfloat16", "float32")), row_scale=plain and rng.random() < 0.5)
    weights = rng.choice(("bfloat16", "bfloat16", "mx4", "mx4", "float32"))
    tokens, width, inner = rng.randint(1, 8), 8 * _log(rng, 8, 256), 8 * _log(rng, 8, 256)
    kind = rng.choice(("groups", "table", "identity", "input"))
    if kind == "groups":
        return _moe(tokens, width, inner, experts, min(top, experts // 2), weights, "silu", groups=4, keep=2, scale=2.5,
                    shared=8 * _log(rng, 8, 256), shared_gate=True)
    if kind == "table":
        return _moe(tokens, width, inner, experts, top, weights, "clamped_swish", score="table", shared=8 * _log(rng, 8, 256))
    if kind == "identity":
        return _moe(tokens, width, inner, experts, top, weights, rng.choice(("clamped_swish", "gelu_tanh")), score="softmax",
                    correction=True, renormalize=True, identity=4)
    return _moe(tokens, width, inner, experts, top, weights, "relu2", weight_input=True)


# ------------------------------------------------------------------ 4-bit numbers, plainly

def _power(exponent):
    """2^exponent for whole numbers from -1022 to 1023, float64: the number's bits, as a power function may round."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _to_mx4(x):
    """[rows, width] -> (codes uint8 [rows, 64 G], scales uint8 [rows, 4 G]), G groups of 128 elements a row."""
    rows, width = x.shape
    groups = -(-width // GROUP)
    x = torch.nn.functional.pad(x.float(), (0, groups * GROUP - width)).view(rows, groups * 4, BLOCK)
    exponent = torch.frexp(x.abs().amax(-1)).exponent - 3                  # floor(log2 of the largest) - 2
    scales = torch.where(x.abs().amax(-1) > 0, (exponent + 127).clamp(0, 254), torch.zeros_like(exponent))
    size = x.abs().double() * _power(127 - scales).unsqueeze(-1)
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    size = (torch.round(size / step) * step).clamp(max=6.0)               # torch.round: a tie goes to the even one
    grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
    code = torch.searchsorted(grid, size) | (torch.signbit(x).long() << 3)
    code = code.to(torch.uint8).view(rows, groups, 4, 4, 4, 2).transpose(-1, -2)     # block, word, parity, place
    code = code.reshape(rows, groups, 4, 4, 4, 2)                                    # block, word, byte, half of the byte
    codes = (code[..., 0] | (code[..., 1] << 4)).transpose(2, 3).reshape(rows, groups * 64).contiguous()
    return codes, scales.to(torch.uint8).contiguous()


def _from_mx4(codes, scales, width):
    """The float32 values that codes [..., rows, 64 G] and scales [..., rows, 4 G] stand for, [..., rows, width]."""
    lead, groups = codes.shape[:-1], codes.shape[-1] // 64
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float32, device=codes.device)
    code = codes.view(*lead, groups, 4, 4, 4).transpose(-3, -2)            # word, block -> block, word
    code = torch.stack((code & 15, code >> 4), dim=-1).reshape(*lead, groups * 4, 4, 2, 4)
    code = code.transpose(-1, -2).reshape(*lead, groups * 4, BLOCK)        # parity, place -> place, parity
    value = grid[code.long()] * _power(scales.long() - 127).float().view(*lead, groups * 4, 1)
    return value.view(*lead, groups * GROUP)[..., :width]


# ------------------------------------------------------------------ what a program has in hand

def _normal(g, *shape, std=1.0, dtype=torch.float32):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * std).to(dtype)


def _weights(g, kind, *shape):
    """A stack of matrices as a checkpoint has them (a spread of sizes by output row), or its 4-bit form."""
    w = _normal(g, *shape, std=0.7 * shape[-1] ** -0.5) * torch.exp(0.3 * _normal(g, *shape[:-1], 1))
    if kind != "mx4":
        return w.to(DTYPES[kind])
    codes, scales = _to_mx4(w.view(-1, shape[-1]))
    return codes.view(*shape[:-1], -1), scales.view(*shape[:-1], -1)


def _tile(pairs, experts):
    return next((t for t in TILES if t >= 2 * pairs // experts), TILES[-1])


def _shared_by(w, width):
    """The framework's handle of a matrix, or of a stack of them."""
    if torch.is_tensor(w):
        return w
    from damendaemon_b200 import kernels
    return kernels.Mx4Matrix(w[0], w[1], width)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 17)
    c, op = case, case["op"]
    state = {"case": case}
    if op == "quantize":
        state["x"] = _weights(g, c["dtype"], c["rows"], c["width"])
    elif op == "linear":
        state["a"] = _normal(g, c["rows"], c["width"], dtype=torch.bfloat16)
        state["w"] = _weights(g, "mx4", c["out"], c["width"])
        state["bias"] = _normal(g, c["out"], std=0.1) if c["bias"] else None
        state["residual"] = _normal(g, c["rows"], c["out"]) if c["residual"] else None
    elif op == "grouped":
        pairs, experts = c["tokens"] * c["top"], c["experts"]
        tile = _tile(pairs, experts)
        # sorted by expert as a step's routing leaves them: every expert's rows start on a tile, rows of padding are zero
        chosen = torch.rand((c["tokens"], experts), generator=g, device=DEV).topk(c["top"], dim=1).indices.view(-1)
        count = torch.bincount(chosen, minlength=experts)
        tiles = (count + tile - 1) // tile
        last = torch.cumsum(tiles, 0)
        n_tiles = -(-(pairs + min(experts, pairs) * (tile - 1)) // tile)
        group = torch.searchsorted(last, torch.arange(n_tiles, device=DEV), right=True)
        state["tile"], state["tile_group"] = tile, torch.where(group < experts, group, -1).to(torch.int32)
        order = torch.argsort(chosen, stable=True)
        within = torch.arange(pairs, device=DEV) - (torch.cumsum(count, 0) - count)[chosen[order]]
        rows = (last - tiles)[chosen[order]] * tile + within
        state["a"] = torch.zeros((n_tiles * tile, c["width"]), dtype=torch.bfloat16, device=DEV)
        state["a"][rows] = _normal(g, pairs, c["width"], dtype=torch.bfloat16)
        state["row_scale"] = torch.zeros(n_tiles * tile, device=DEV) if c["row_scale"] else None
        if c["row_scale"]:
            state["row_scale"][rows] = torch.rand(pairs, generator=g, device=DEV)
        gated = c["unit"] not in ("none", "relu2")
        state["w"] = _weights(g, "mx4", experts, c["out"] * (2 if gated else 1), c["width"])
        state["out"] = torch.zeros((n_tiles * tile, c["out"]), dtype=DTYPES[c["out_dtype"]], device=DEV)
    else:
        kind, E, D, I = c["weights"], c["experts"], c["width"], c["inner"]
        dtype = torch.float32 if kind == "float32" else torch.bfloat16
        state["y"] = _normal(g, c["tokens"], D, dtype=dtype)
        state["residual"] = _normal(g, c["tokens"], D)
        halves = 1 if c["unit"] == "relu2" else 2
        state["gate_up"], state["down"] = _weights(g, kind, E, halves * I, D), _weights(g, kind, E, D, I)
        state["router"] = state["table"] = state["ids"] = state["correction"] = state["shared"] = None
        if c["score"] == "table":
            vocab = 4096
            state["table"] = torch.rand((vocab, E), generator=g, device=DEV).topk(c["top"], dim=1).indices.to(torch.int32)
            state["ids"] = torch.randint(0, vocab, (c["tokens"],), generator=g, device=DEV, dtype=torch.int32)
        else:
            state["router"] = _normal(g, E + c["identity"] + (1 if c["shared_gate"] else 0), D, std=D ** -0.5, dtype=dtype)
            if c["correction"]:
                state["correction"] = _normal(g, E + c["identity"], std=0.02)
        if c["shared"]:
            state["shared"] = (_weights(g, kind, 2 * c["shared"], D), _weights(g, kind, D, c["shared"]))
        if own:          # the handle that a model keeps beside its weights: it names the tensors above
            from damendaemon_b200 import kernels
            gated = None if c["unit"] == "relu2" else (7.0, 1.702, c["unit"])
            shared = None if not c["shared"] else (_shared_by(state["shared"][0], D), _shared_by(state["shared"][1], c["shared"]))
            state["layer"] = kernels.ExpertLayer(
                _shared_by(state["gate_up"], D), _shared_by(state["down"], I), c["top"], gated=gated,
                activation="relu2" if gated is None else None, router=state["router"], table=state["table"],
                softmax=c["score"] == "softmax", groups=c["groups"], keep=c["keep"], weight_scale=c["scale"],
                correction=state["correction"], renormalize=c["renormalize"], identity=c["identity"],
                weight_input=c["weight_input"], shared=shared, shared_gated=gated, shared_gate=c["shared_gate"])
    return state


# ------------------------------------------------------------------ one pass

def run(state):
    c = state["case"]
    return {"quantize": _run_quantize, "linear": _run_linear, "grouped": _run_grouped, "moe": _run_moe}[c["op"]](state, c)


def _act(v, name):
    if name == "gelu_new":
        return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    if name == "relu2":
        return torch.clamp(v, min=0) ** 2
    return v


def _unit(z, unit):
    """The unit's value from its product(s) along the last dimension: gate and up halves, or the up product alone."""
    if unit in ("none", "relu2"):
        return _act(z, unit)
    gate, up = z.chunk(2, dim=-1)
    if unit == "silu":
        return gate * torch.sigmoid(gate) * up
    if unit == "gelu_tanh":
        return _act(gate, "gelu_new") * up
    gate, up = torch.clamp(gate, max=7.0), torch.clamp(up, -7.0, 7.0)
    return gate * torch.sigmoid(1.702 * gate) * (up + 1)


def _run_quantize(s, c):
    if own:
        from damendaemon_b200 import kernels
        return kernels.mx4_values(kernels.mx4_quantize(s["x"]), dtype=s["x"].dtype)
    codes, scales = _to_mx4(s["x"])
    return _from_mx4(codes, scales, c["width"]).to(s["x"].dtype)


def _run_linear(s, c):
    if own:
        from damendaemon_b200 import kernels
        return kernels.gemm_mx4(s["a"], kernels.Mx4Matrix(*s["w"], c["width"]), s["bias"], s["residual"],
                                None if c["activation"] == "none" else c["activation"], DTYPES[c["out_dtype"]])
    z = s["a"].float() @ _from_mx4(*s["w"], c["width"]).t()
    if s["bias"] is not None:
        z = z + s["bias"]
    z = _act(z, c["activation"])
    if s["residual"] is not None:
        z = z + s["residual"]
    return z.to(DTYPES[c["out_dtype"]])


def _run_grouped(s, c):
    plain = c["unit"] in ("none", "relu2")
    if own:
        from damendaemon_b200 import kernels
        return kernels.gemm_grouped_mx4(s["a"], kernels.Mx4Matrix(*s["w"], c["width"]), s["tile_group"], s["tile"],
                                        gated=None if plain else (7.0, 1.702, c["unit"]), out_dtype=DTYPES[c["out_dtype"]],
                                        activation="relu2" if c["unit"] == "relu2" else None, row_scale=s["row_scale"], out=s["out"])
    group, tile = s["tile_group"].long(), s["tile"]
    w = _from_mx4(*s["w"], c["width"])[group.clamp(min=0)]
    z = torch.bmm(s["a"].float().view(-1, tile, c["width"]), w.transpose(1, 2))
    if s["row_scale"] is not None:
        z = z * s["row_scale"].view(-1, tile, 1)
    z = _unit(z, c["unit"]) * (group >= 0).view(-1, 1, 1)
    return z.view(-1, c["out"]).to(DTYPES[c["out_dtype"]])


def _route(s, c):
    """(the chosen experts [tokens, top], their weights, the shared unit's gate [tokens, 1])."""
    E = c["experts"] + c["identity"]
    if c["score"] == "table":
        return s["table"][s["ids"].long()].long(), torch.full((c["tokens"], c["top"]), 1.0 / c["top"], device=DEV), 1.0
    z = s["y"].float() @ s["router"].float().t()
    gate = torch.sigmoid(z[:, E:]) if c["shared_gate"] else 1.0
    score = torch.softmax(z[:, :E], dim=1) if c["score"] == "softmax" else torch.sigmoid(z[:, :E])
    order = score + s["correction"] if c["correction"] else (score if c["groups"] > 1 or c["score"] == "softmax" else z[:, :E])
    if c["groups"] > 1:
        runs = order.view(c["tokens"], c["groups"], -1)
        worth = runs.topk(min(2, runs.shape[2]), dim=2).values.sum(2)
        kept = torch.zeros_like(worth).scatter_(1, worth.topk(c["keep"], dim=1).indices, 1.0)
        order = torch.where(kept.unsqueeze(2) > 0, runs, -math.inf).view(c["tokens"], E)
    chosen = torch.sort(order, dim=1, descending=True, stable=True).indices[:, :c["top"]]
    weight = score.gather(1, chosen)
    if c["renormalize"]:
        weight = weight / (weight.sum(1, keepdim=True) + 1e-20)
    return chosen, weight * c["scale"], gate


def _run_moe(s, c):
    if own:
        from damendaemon_b200 import kernels
        return kernels.moe_tokens(s["layer"], s["y"], s["residual"], ids=s["ids"])
    D, I = c["width"], c["inner"]
    chosen, weight, gate = _route(s, c)
    y, real = s["y"].float(), (chosen < c["experts"]).float()
    expert = chosen.clamp(max=c["experts"] - 1)

    def pick(w, width):          # the chosen experts' matrices, float32 [tokens, top, rows, width]
        return w[expert].float() if torch.is_tensor(w) else _from_mx4(w[0][expert], w[1][expert], width)

    z = (pick(s["gate_up"], D) @ y.view(-1, 1, D, 1)).squeeze(-1)
    if c["weight_input"]:
        z = z * weight.unsqueeze(-1)
    hidden = _unit(z, c["unit"])
    out = (pick(s["down"], I) @ hidden.unsqueeze(-1)).squeeze(-1) * real.unsqueeze(-1) + y.unsqueeze(1) * (1 - real).unsqueeze(-1)
    total = s["residual"] + (out if c["weight_input"] else out * weight.unsqueeze(-1)).sum(1)
    if c["shared"]:
        up, down = ((w.float() if torch.is_tensor(w) else _from_mx4(*w, width)) for w, width in zip(s["shared"], (D, c["shared"])))
        total = total + (_unit(y @ up.t(), c["unit"]) * gate) @ down.t()
    return total


# ------------------------------------------------------------------ what a pass cannot do without

def _mx4_bytes(rows, width):
    return rows * width * 17 / 32


def work(case):
    c, op = case, case["op"]
    size = {"float32": 4, "bfloat16": 2}
    if op == "quantize":
        n = c["rows"] * c["width"]
        return {"bytes": 2 * n * size[c["dtype"]] + 2 * _mx4_bytes(c["rows"], c["width"]), "flops": 4 * n}
    if op == "linear":
        n = c["rows"] * c["out"]
        return {"bytes": _mx4_bytes(c["out"], c["width"]) + 2 * c["rows"] * c["width"] + n * size[c["out_dtype"]]
                + (4 * n if c["residual"] else 0) + (4 * c["out"] if c["bias"] else 0), "flops": 2 * n * c["width"]}
    halves = 1 if c["unit"] in ("none", "relu2") else 2
    if op == "grouped":
        pairs = c["tokens"] * c["top"]
        used = c["experts"] * (1 - (1 - c["top"] / c["experts"]) ** c["tokens"])        # experts that a token chooses, on average
        return {"bytes": used * _mx4_bytes(halves * c["out"], c["width"]) + pairs * (2 * c["width"] + c["out"] * size[c["out_dtype"]]),
                "flops": 2 * pairs * halves * c["out"] * c["width"]}
    T, D, I, E = c["tokens"], c["width"], c["inner"], c["experts"] + c["identity"]
    real = c["top"] * c["experts"] / E
    used = c["experts"] * (1 - (1 - c["top"] / E) ** T)
    element = 17 / 32 if c["weights"] == "mx4" else size[c["weights"]]
    row = size["float32" if c["weights"] == "float32" else "bfloat16"]
    per = (halves + 1) * D
    routed = 0 if c["score"] == "table" else (E + (1 if c["shared_gate"] else 0)) * D
    shared = 3 * D * c["shared"]
    return {"bytes": (used * per * I + shared) * element + routed * row + T * D * (row + 8),
            "flops": 2 * T * (real * per * I + shared + routed)}


# ------------------------------------------------------------------ the definition in 64 bits

def _exact_values(codes, scales, width):
    """Word by word: the elements of block b are words b, 4 + b, 8 + b and 12 + b of a group, eight a word."""
    rows = codes.reshape(-1, codes.shape[-1])
    words = rows.contiguous().view(torch.int32).long() & 0xffffffff
    words = words.view(rows.shape[0], -1, 16)
    out = torch.empty((rows.shape[0], words.shape[1], 4, BLOCK), dtype=torch.float64, device=codes.device)
    for b in range(4):
        for t in range(4):
            for i in range(8):
                code = (words[:, :, 4 * t + b] >> (4 * (i // 2) + 16 * (i % 2))) & 15
                e, m = (code >> 1) & 3, (code & 1).double()
                size = torch.where(e == 0, 0.5 * m, 2.0 ** (e.double() - 1) * (1 + 0.5 * m))
                out[:, :, b, 8 * t + i] = torch.where(code >= 8, -size, size)
    powers = torch.tensor([2.0 ** (k - 127) for k in range(256)], dtype=torch.float64, device=codes.device)
    out *= powers[scales.reshape(rows.shape[0], -1, 4).long()].unsqueeze(-1)
    return out.view(*codes.shape[:-1], -1)[..., :width]


def _exact_matrix(w, width):
    return w.double() if torch.is_tensor(w) else _exact_values(w[0], w[1], width)


def _exact_unit(z, unit, inner):
    if unit == "none":
        return z
    if unit == "relu2":
        return torch.relu(z).square()
    g, u = z[..., :inner], z[..., inner:]
    if unit == "silu":
        return u * g / (1 + torch.exp(-g))
    if unit == "gelu_tanh":
        return u * torch.nn.functional.gelu(g, approximate="tanh")
    g = torch.minimum(g, torch.full_like(g, 7.0))
    return g / (1 + torch.exp(-1.702 * g)) * (1 + torch.clip(u, -7.0, 7.0))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "quantize":
        x = s["x"].double()
        out = torch.empty_like(x)
        grid = torch.tensor(GRID, dtype=torch.float64, device=x.device)
        powers = torch.tensor([2.0 ** k for k in range(-160, 161)], dtype=torch.float64, device=x.device)
        for at in range(0, c["width"], BLOCK):
            block = x[:, at:at + BLOCK]
            top = block.abs().amax(1, keepdim=True)
            e = torch.searchsorted(powers, top, right=True) - 1 - 160             # the last power of two not above the largest
            by = powers[torch.clamp(e - 2, -127, 127) + 160]
            size = block.abs() / by
            # between two numbers of the grid: the nearer one, in the middle the one with an even mantissa bit
            low = torch.clamp(torch.searchsorted(grid, size, right=True) - 1, max=6)
            down, up = size - grid[low], grid[low + 1] - size
            at_up = (up < down) | ((up == down) & (low % 2 == 1))
            out[:, at:at + BLOCK] = torch.sign(block) * torch.where(at_up, grid[low + 1], grid[low]) * by
        return out
    if c["op"] == "linear":
        z = s["a"].double() @ _exact_matrix(s["w"], c["width"]).T
        z = z if s["bias"] is None else z + s["bias"].double()
        if c["activation"] == "gelu":
            z = torch.nn.functional.gelu(z)
        elif c["activation"] == "gelu_new":
            z = torch.nn.functional.gelu(z, approximate="tanh")
        elif c["activation"] == "relu2":
            z = torch.relu(z).square()
        return z if s["residual"] is None else z + s["residual"].double()
    if c["op"] == "grouped":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
        for i, e in enumerate(s["tile_group"].tolist()):
            if e >= 0:
                rows = slice(i * s["tile"], (i + 1) * s["tile"])
                z = s["a"][rows].double() @ _exact_values(s["w"][0][e], s["w"][1][e], c["width"]).T
                if s["row_scale"] is not None:
                    z = z * s["row_scale"][rows].double().unsqueeze(1)
                out[rows] = _exact_unit(z, c["unit"], c["out"])
        return out
    return _exact_moe(c, s)


def _exact_moe(c, s):
    y, out = s["y"].double(), s["residual"].double().clone()
    E, real, D, I = c["experts"] + c["identity"], c["experts"], c["width"], c["inner"]
    z = None if s["router"] is None else y @ s["router"].double().T
    for t in range(c["tokens"]):
        if z is None:
            chosen = [(e, 1.0 / c["top"]) for e in s["table"][int(s["ids"][t])].tolist()]
        else:
            logits = z[t, :E]
            score = torch.exp(logits - torch.logsumexp(logits, 0)) if c["score"] == "softmax" else 1 / (1 + torch.exp(-logits))
            order = (score + s["correction"].double() if c["correction"] else score).tolist()
            per = E // c["groups"]
            worth = [sum(sorted(order[i * per:(i + 1) * per])[-2:]) for i in range(c["groups"])]
            kept = sorted(range(c["groups"]), key=lambda i: (-worth[i], i))[:c["keep"]]
            best = sorted((e for e in range(E) if e // per in kept), key=lambda e: (-order[e], e))[:c["top"]]
            total = sum(float(score[e]) for e in best) + 1e-20 if c["renormalize"] else 1.0
            chosen = [(e, float(score[e]) / total * c["scale"]) for e in best]
        for e, weight in chosen:
            if e >= real:
                out[t] += weight * y[t]
                continue
            part = lambda w: w[e] if torch.is_tensor(w) else (w[0][e], w[1][e])  # noqa: E731
            h = _exact_matrix(part(s["gate_up"]), D) @ y[t]
            h = _exact_unit(h * weight if c["weight_input"] else h, c["unit"], I)
            out[t] += (1.0 if c["weight_input"] else weight) * (_exact_matrix(part(s["down"]), I) @ h)
    if c["shared"]:
        h = _exact_unit(y @ _exact_matrix(s["shared"][0], D).T, c["unit"], c["shared"])
        if c["shared_gate"]:
            h = h / (1 + torch.exp(-z[:, E:E + 1]))
        out += h @ _exact_matrix(s["shared"][1], c["shared"]).T
    return out
