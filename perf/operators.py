"""Microscaled 4-bit (MX4) tensors and the products over them, as cases that can be timed and compared.

An MX4 tensor holds rows of k values (k a multiple of 32) in blocks of 32 along k: `codes` uint8 [rows][k / 2], value 2i in
the low four bits of byte i, each a sign, two exponent bits and one mantissa bit (0, 0.5, 1, 1.5, 2, 3, 4, 6); `scales`
uint8 [ceil(k / 128)][rows][4], byte b of (c, r) the scale of values 128c + 32b .. of row r, 2^(byte - 127).  The scale of
a block is 2^(floor(log2(largest magnitude)) - 2), no smaller than 2^-127; values round to the nearest code, ties to
the even one, and saturate at 6.

A case is a dict of plain values with a "kind":

  roundtrip   rows to MX4 and back: what quantisation makes of them        (mx4_quantize, mx4_dequant)
  linear      y = x . w^T, w in MX4, x in 16 or 32 bits and quantised on the way         (mx4_linear)
  product     the same with x in MX4, as a layer has it that several products read       (mx4_matmul)
  feed        what a routed layer does first: the pairs in the experts' order, their rows of x gathered and quantised,
              the gate and up product by expert with the gated unit  (moe_order, mx4_quantize, mx4_matmul_grouped)
  down        the product by expert that ends it, rows scattered to their pairs            (mx4_matmul_grouped)
"""
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE_OF = {"f32": 4, "f16": 2, "bf16": 2}

_contexts = {}


def _context():
    """The library's handle: one for the device, kept for the life of the program."""
    if "ctx" not in _contexts:
        import aotx_b200
        _contexts["ctx"] = aotx_b200.Q8Context(0)
    return _contexts["ctx"]


def listed():
    return [
        # activations of one token, the smallest call
        {"name": "roundtrip_token", "kind": "roundtrip", "rows": 1, "k": 4096, "x": "bf16"},
        # a gate+up tensor when a model is laid out, from binary16
        {"name": "roundtrip_weights", "kind": "roundtrip", "rows": 28672, "k": 4096, "x": "f16"},
        # one token of one sequence against a square projection
        {"name": "linear_4096_m1", "kind": "linear", "n": 4096, "k": 4096, "m": 1, "x": "f16", "y": "f16", "gated": False},
        # gate+up of an 8B-shaped layer for eight sequences
        {"name": "linear_gate_up_m8", "kind": "linear", "n": 28672, "k": 4096, "m": 8, "x": "bf16", "y": "bf16",
         "gated": True},
        # the vocabulary projection of a decode step: the largest tensor of a model
        {"name": "linear_lm_head_m8", "kind": "linear", "n": 151936, "k": 8192, "m": 8, "x": "bf16", "y": "bf16",
         "gated": False},
        # fused QKV for a batch that fills no tile
        {"name": "product_qkv_m100", "kind": "product", "n": 6144, "k": 4096, "m": 100, "y": "f32", "gated": False},
        # a short prompt through the gate+up of a 4B-shaped layer, ragged
        {"name": "product_gate_up_m300", "kind": "product", "n": 19456, "k": 2560, "m": 300, "y": "f16", "gated": True},
        # a full prompt chunk through the 8B-shaped gate+up: the largest amount of arithmetic
        {"name": "linear_gate_up_m2048", "kind": "linear", "n": 28672, "k": 4096, "m": 2048, "x": "bf16", "y": "bf16",
         "gated": True},
        # routed experts, a decode step of eight sequences
        {"name": "feed_t8", "kind": "feed", "tokens": 8, "used": 8, "experts": 128, "hidden": 2048, "ffn": 768},
        # and a prompt chunk
        {"name": "feed_t512", "kind": "feed", "tokens": 512, "used": 8, "experts": 128, "hidden": 2048, "ffn": 768},
        {"name": "down_t512", "kind": "down", "tokens": 512, "used": 8, "experts": 128, "hidden": 2048, "ffn": 768},
        # a smaller table with widths that fill no tile
        {"name": "down_odd_t77", "kind": "down", "tokens": 77, "used": 4, "experts": 20, "hidden": 1000, "ffn": 736},
    ]


def _spread(rng, low, high):
    """An integer of [low, high], even over the logarithm."""
    return min(high, max(low, int(round(low * (high / low) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["roundtrip", "linear", "linear", "product", "product", "feed", "down"])
    if kind == "roundtrip":
        return {"kind": kind, "rows": _spread(rng, 1, 28672), "k": 32 * _spread(rng, 1, 128),
                "x": rng.choice(["f32", "f16", "bf16"])}
    if kind in ("linear", "product"):
        gated = rng.random() < 0.4
        case = {"kind": kind, "n": _spread(rng, 64, 28672), "k": 32 * _spread(rng, 4, 256),
                "m": _spread(rng, 1, 1024), "y": rng.choice(["f32", "f16", "bf16"]), "gated": gated}
        if gated:
            case["n"] += case["n"] % 2
        if kind == "linear":
            case["x"] = rng.choice(["f32", "f16", "bf16"])
        return case
    experts = _spread(rng, 4, 256)
    return {"kind": kind, "tokens": _spread(rng, 1, 1024), "used": rng.randint(1, min(8, experts)), "experts": experts,
            "hidden": 32 * _spread(rng, 8, 64), "ffn": 32 * _spread(rng, 8, 32)}


# ---------------------------------------------------------------------------------------------------
# The plain forms
# ---------------------------------------------------------------------------------------------------
def _power_of_two(exponent):
    """2^exponent as a float, by its bits: exponent from -127 to 127."""
    return torch.where(exponent > -127, (exponent + 127) << 23, torch.full_like(exponent, 1 << 22)).view(torch.float32)


def _quantize(x):
    """Codes and scales of a float tensor of [rows][k]."""
    rows, k = x.shape
    blocks = x.float().view(rows, k // 32, 32)
    _, exponent = torch.frexp(blocks.abs().amax(dim=2))
    exponent = torch.where(blocks.abs().amax(dim=2) > 0, exponent - 3, torch.full_like(exponent, -127)).clamp_min(-127)
    v = blocks * _power_of_two(-exponent).unsqueeze(2)
    a = v.abs()
    # the grid is 0.5 apart below 2, 1 apart below 4, 2 apart above; torch.round takes ties to even
    near = torch.where(a < 2, (a * 2).round() / 2, torch.where(a < 4, a.round(), (a / 2).round() * 2)).clamp_max(6)
    code = torch.where(near < 2, near * 2, torch.where(near < 4, near + 2, near / 2 + 4)).to(torch.uint8)
    code = (code + 8 * torch.signbit(v).to(torch.uint8)).view(rows, k // 2, 2)
    codes = code[:, :, 0] + 16 * code[:, :, 1]
    chunks = (k + 127) // 128
    scales = torch.zeros((rows, chunks * 4), dtype=torch.uint8, device=x.device)
    scales[:, :k // 32] = (exponent + 127).to(torch.uint8)
    return codes, scales.view(rows, chunks, 4).transpose(0, 1).contiguous()


def _values(codes, scales):
    """What an MX4 tensor stands for, as floats."""
    rows, half = codes.shape
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                         device=codes.device)
    v = torch.stack((table[(codes & 15).int()], table[(codes >> 4).int()]), dim=2).view(rows, half // 16, 32)
    exponent = scales.transpose(0, 1).reshape(rows, -1)[:, :half // 16].int() - 127
    return (v * _power_of_two(exponent).unsqueeze(2)).view(rows, 2 * half)


def _chunks(total, step):
    return [(i, min(total, i + step)) for i in range(0, total, step)]


def _product(w, x):
    """x . w^T in floats, the rows of w a piece at a time (their values take eight times the codes' bytes)."""
    codes, scales = w
    pieces = [x @ _values(codes[a:b], scales[:, a:b]).T for a, b in _chunks(codes.shape[0], 32768)]
    return pieces[0] if len(pieces) == 1 else torch.cat(pieces, dim=1)


def _gated(y):
    """silu(gate) * up of columns that take turns."""
    gate, up = y[:, 0::2], y[:, 1::2]
    return gate / (1 + torch.exp(-gate)) * up


def _by_expert(state, x, gated):
    codes, scales = state["w"]
    n = codes.shape[0] // state["experts"]
    out, at = [], 0
    for e, count in enumerate(state["counts"]):
        if count:
            part = _product((codes[e * n:e * n + n], scales[:, e * n:e * n + n]), x[at:at + count])
            out.append(_gated(part) if gated else part)
            at += count
    return torch.cat(out)


def _order(ids, experts):
    flat = ids.reshape(-1)
    order = torch.sort(flat, stable=True)[1]
    edges = torch.cumsum((flat[None, :] == torch.arange(experts, device=ids.device)[:, None]).sum(dim=1), dim=0)
    offsets = torch.cat((torch.zeros_like(edges[:1]), edges)).to(torch.int32)
    return order.to(torch.int32), torch.div(order, ids.shape[1], rounding_mode="floor").to(torch.int32), offsets


# ---------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------
def _rows(gen, rows, k, dtype):
    """Activations behind a norm: N(0, 1), a few channels ten times as large."""
    x = torch.randn((rows, k), generator=gen, device="cuda")
    loud = torch.rand((k,), generator=gen, device="cuda") < 0.01
    return torch.where(loud, x * 10, x).to(dtype)


def _weights(gen, rows, k):
    """N(0, 0.02) in MX4, a piece at a time."""
    codes = torch.empty((rows, k // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty(((k + 127) // 128, rows, 4), dtype=torch.uint8, device="cuda")
    for a, b in _chunks(rows, 16384):
        c, s = _quantize(torch.randn((b - a, k), generator=gen, device="cuda") * 0.02)
        codes[a:b] = c
        scales[:, a:b] = s
    return codes, scales


def _selections(gen, tokens, used, experts):
    """Top experts of logits that lean towards some of them."""
    lean = torch.randn((experts,), generator=gen, device="cuda") * 0.5
    logits = torch.randn((tokens, experts), generator=gen, device="cuda") + lean
    return torch.topk(logits, used, dim=1)[1].to(torch.int32)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = case["kind"]
    state = {"kind": kind}
    if kind == "roundtrip":
        # a token's activations, or weights
        x = _rows(gen, case["rows"], case["k"], torch.float32)
        state["x"] = (x if case["rows"] < 4096 else x.mul_(0.02)).to(DTYPES[case["x"]])
    elif kind in ("linear", "product"):
        state["w"] = _weights(gen, case["n"], case["k"])
        x = _rows(gen, case["m"], case["k"], DTYPES[case["x"]] if kind == "linear" else torch.float16)
        state["x"] = x if kind == "linear" else _quantize(x)
        state["y_dtype"] = DTYPES[case["y"]]
        state["gated"] = case["gated"]
    else:
        n, k = (2 * case["ffn"], case["hidden"]) if kind == "feed" else (case["hidden"], case["ffn"])
        state["experts"] = case["experts"]
        state["w"] = _weights(gen, case["experts"] * n, k)
        state["ids"] = _selections(gen, case["tokens"], case["used"], case["experts"])
        state["counts"] = torch.bincount(state["ids"].reshape(-1).long(), minlength=case["experts"]).tolist()
        if kind == "feed":
            state["x"] = _rows(gen, case["tokens"], k, torch.float16)
        else:
            state["order"], _, state["offsets"] = _order(state["ids"], case["experts"])
            # what the gated unit leaves: products of two normal values
            pairs = case["tokens"] * case["used"]
            act = _rows(gen, pairs, k, torch.float32) * torch.randn((pairs, k), generator=gen, device="cuda") * 0.3
            state["x"] = _quantize(act)
    if own:
        import aotx_b200
        state["ctx"] = _context()
        for name in ("w", "x"):
            if isinstance(state.get(name), tuple):
                state["own_" + name] = aotx_b200.Mx4Tensor(*state[name])
    return state


# ---------------------------------------------------------------------------------------------------
# A pass
# ---------------------------------------------------------------------------------------------------
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import aotx_b200
    ctx, kind = state["ctx"], state["kind"]
    if kind == "roundtrip":
        return ctx.mx4_dequant(ctx.mx4_quantize(state["x"]), dtype=state["x"].dtype)
    if kind in ("linear", "product"):
        epilogue = aotx_b200.EPILOGUE_SWIGLU if state["gated"] else aotx_b200.EPILOGUE_STORE
        if kind == "linear":
            return ctx.mx4_linear(state["own_w"], state["x"], y_dtype=state["y_dtype"], epilogue=epilogue)
        return ctx.mx4_matmul(state["own_w"], state["own_x"], y_dtype=state["y_dtype"], epilogue=epilogue)
    if kind == "feed":
        order, tokens, offsets = ctx.moe_order(state["ids"], state["experts"])
        x = ctx.mx4_quantize(state["x"], rows=tokens)
        act = ctx.mx4_matmul_grouped(state["own_w"], state["experts"], x, offsets, y_dtype=torch.float16,
                                     epilogue=aotx_b200.EPILOGUE_SWIGLU)
        return order, offsets, act
    return ctx.mx4_matmul_grouped(state["own_w"], state["experts"], state["own_x"], state["offsets"],
                                  y_rows=state["order"], y_dtype=torch.float32)


def _run_plain(state):
    kind = state["kind"]
    if kind == "roundtrip":
        return _values(*_quantize(state["x"])).to(state["x"].dtype)
    if kind in ("linear", "product"):
        x = _values(*(_quantize(state["x"]) if kind == "linear" else state["x"]))
        y = _product(state["w"], x)
        return (_gated(y) if state["gated"] else y).to(state["y_dtype"])
    if kind == "feed":
        order, tokens, offsets = _order(state["ids"], state["experts"])
        x = _values(*_quantize(state["x"][tokens.long()]))
        return order, offsets, _by_expert(state, x, True).half()
    y = _by_expert(state, _values(*state["x"]), False)
    out = torch.empty_like(y)
    out[state["order"].long()] = y
    return out


# ---------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------
def _mx4_bytes(rows, k):
    return rows * k // 2 + rows * k // 32


def work(case):
    kind = case["kind"]
    if kind == "roundtrip":
        # the values in, the values out; what lies between need not leave the chip
        values = case["rows"] * case["k"]
        return {"bytes": 2 * values * SIZE_OF[case["x"]], "flops": 0}
    if kind in ("linear", "product"):
        n, k, m = case["n"], case["k"], case["m"]
        x = m * k * SIZE_OF[case["x"]] if kind == "linear" else _mx4_bytes(m, k)
        out = m * (n // 2 if case["gated"] else n) * SIZE_OF[case["y"]]
        return {"bytes": _mx4_bytes(n, k) + x + out, "flops": 2 * m * n * k}
    pairs = case["tokens"] * case["used"]
    n, k = (2 * case["ffn"], case["hidden"]) if kind == "feed" else (case["hidden"], case["ffn"])
    # experts that are chosen at least once, for selections without a lean
    chosen = case["experts"] * (1 - (1 - case["used"] / case["experts"]) ** case["tokens"])
    weights = _mx4_bytes(int(round(chosen)) * n, k)
    if kind == "feed":
        small = 4 * pairs + 4 * pairs + 4 * (case["experts"] + 1)
        rows = case["tokens"] * k * 2 + pairs * case["ffn"] * 2
    else:
        small = 4 * pairs + 4 * (case["experts"] + 1)
        rows = _mx4_bytes(pairs, k) + pairs * n * 4
    return {"bytes": weights + rows + small, "flops": 2 * pairs * n * k}


# ---------------------------------------------------------------------------------------------------
# The definition in 64 bits
# ---------------------------------------------------------------------------------------------------
_MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _wide_power(exponent):
    """2^exponent in 64 bits (a power function may be off by a bit, which would move the borders between codes)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _exact_quantized(x):
    """The values that MX4 keeps of x: for each the nearest of eight magnitudes, found between their midpoints."""
    rows, k = x.shape
    wide = x.double().reshape(rows * (k // 32), 32)
    largest = wide.abs().max(dim=1, keepdim=True)[0]
    # the exponent by comparison with powers of two, no logarithm
    power = torch.floor(torch.log2(largest.clamp_min(2.0 ** -200)))
    power = torch.where(_wide_power(power) > largest, power - 1, power)
    power = torch.where(_wide_power(power + 1) <= largest, power + 1, power)
    scale = _wide_power((power - 2).clamp_min(-127))
    grid = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=x.device)
    middle = (grid[1:] + grid[:-1]) / 2
    ratio = wide.abs() / scale
    # up to and with a midpoint the lower one, except where the lower one is odd
    low = torch.searchsorted(middle, ratio)
    high = torch.searchsorted(middle, ratio, right=True)
    index = torch.where(low % 2 == 0, low, high)
    return (torch.sign(wide) * grid[index] * scale).view(rows, k)


def _exact_values(codes, scales):
    rows, half = codes.shape
    out = torch.empty((rows, half, 2), dtype=torch.float64, device=codes.device)
    grid = torch.tensor(_MAGNITUDES, dtype=torch.float64, device=codes.device)
    for part in range(2):
        nibble = torch.div(codes, 16 ** part, rounding_mode="floor") % 16
        out[:, :, part] = grid[(nibble % 8).long()] * (1 - 2 * (nibble >= 8).double())
    per_block = _wide_power(scales.permute(1, 0, 2).reshape(rows, -1)[:, :half // 16].long() - 127)
    return out.view(rows, half // 16, 32).mul_(per_block.unsqueeze(2)).view(rows, 2 * half)


def _exact_product(w, x, gated):
    codes, scales = w
    parts = []
    for a in range(0, codes.shape[0], 16384):
        parts.append(torch.matmul(x, _exact_values(codes[a:a + 16384], scales[:, a:a + 16384]).t()))
    y = torch.cat(parts, dim=1)
    if not gated:
        return y
    pairs = y.view(y.shape[0], -1, 2)
    return pairs[:, :, 0] * torch.sigmoid(pairs[:, :, 0]) * pairs[:, :, 1]


def exact(case, seed):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "roundtrip":
        return _exact_quantized(state["x"])
    if kind in ("linear", "product"):
        x = _exact_quantized(state["x"]) if kind == "linear" else _exact_values(*state["x"])
        return _exact_product(state["w"], x, case["gated"])
    codes, scales = state["w"]
    n = codes.shape[0] // case["experts"]
    flat = state["ids"].reshape(-1)
    # the pairs of expert 0 in their order, then those of expert 1, and so on
    lists = [torch.nonzero(flat == e).reshape(-1) for e in range(case["experts"])]
    order = torch.cat(lists)
    x = _exact_quantized(state["x"]) if kind == "feed" else _exact_values(*state["x"])
    out = torch.empty((flat.numel(), case["ffn"] if kind == "feed" else n), dtype=torch.float64, device=flat.device)
    offsets = [0]
    for e, mine in enumerate(lists):
        at = offsets[-1]
        offsets.append(at + mine.numel())
        if mine.numel():
            weights = (codes[e * n:e * n + n], scales[:, e * n:e * n + n])
            if kind == "feed":
                out[at:offsets[-1]] = _exact_product(weights, x[mine // case["used"]], True)
            else:
                out[mine] = _exact_product(weights, x[at:offsets[-1]], False)
    if kind == "feed":
        return order.to(torch.int32), torch.tensor(offsets, dtype=torch.int32, device=flat.device), out
    return out
