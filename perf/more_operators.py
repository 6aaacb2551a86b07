"""What a program whose layers choose among experts, and whose weights lie in
microscaled 4 bits, has this framework do, as cases that can be measured: rows
put into that form and read back, products with such weights, the choice of
experts, and the experts' feed-forward blocks.

Microscaled rows ("MX4").  Every 32 values of a row share a power of two, kept as
a byte b for 2^(b - 127); a value is one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 or their
negatives (e2m1: sign, two bits of exponent, one of mantissa) times it.  Codes
lie [rows][cols / 2], two a byte, low nibble first; scales [rows][cols / 32].
Written rows take 2^(floor(log2(largest magnitude)) - 2), and each value's
nearest level of it, ties to the even code, 6 at most.

Kinds:
  quant    rows into the form, and read back from it
  product  lanes of floats, or of microscaled rows, times a microscaled weight
  route    the experts a lane takes, and their weights: softmax or sigmoid scores,
           a bias for balance, groups of experts, the best of the kept groups
  experts  out = sum_j weight_j down_e(gelu(gate_e x) * up_e x) over a lane's
           experts e = pick_j, microscaled weights
"""
import math

import numpy as np
import torch

own = False

GROUP = 32
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- the cases ----------------------------------------------------------------

def listed():
    return [
        # a speculative block's activations, to be kept or sent in 4 bits
        {"name": "quant_5_lanes", "kind": "quant", "type": "f32", "rows": 5, "cols": 2048},
        # a down projection's weight, converted as a checkpoint is loaded
        {"name": "quant_sheet", "kind": "quant", "type": "f32", "rows": 6144, "cols": 12288},
        # one token's gate projection
        {"name": "product_1_lane", "kind": "product", "type": "f32", "rows": 6144, "cols": 1536, "lanes": 1},
        # the output head for a speculative block
        {"name": "product_head", "kind": "product", "type": "f32", "rows": 262144, "cols": 1536, "lanes": 5},
        # a batch of sessions, a down projection
        {"name": "product_37_lanes", "kind": "product", "type": "f32", "rows": 2048, "cols": 8192, "lanes": 37},
        # a prompt in bf16
        {"name": "product_2047_lanes", "kind": "product", "type": "bf16", "rows": 8192, "cols": 2048, "lanes": 2047},
        # a prompt whose activations are in 4 bits too
        {"name": "product_2048_mx4", "kind": "product", "type": "mx4", "rows": 8192, "cols": 2048, "lanes": 2048},
        # one token's experts of a softmax router
        {"name": "route_1_lane", "kind": "route", "experts": 128, "top": 8, "score": "softmax", "groups": 1, "kept": 1,
         "lanes": 1},
        # a long prompt's experts: sigmoid scores, a bias for balance, groups
        {"name": "route_16383_lanes", "kind": "route", "experts": 256, "top": 8, "score": "sigmoid", "groups": 8,
         "kept": 4, "lanes": 16383},
        # one token's experts
        {"name": "experts_1_lane", "kind": "experts", "type": "f32", "experts": 128, "top": 8, "hidden": 1536,
         "inner": 768, "lanes": 1},
        # a batch of sessions: most experts are taken, each by a few lanes
        {"name": "experts_37_lanes", "kind": "experts", "type": "f32", "experts": 64, "top": 6, "hidden": 1536,
         "inner": 704, "lanes": 37},
        # a prompt in bf16
        {"name": "experts_2047_lanes", "kind": "experts", "type": "bf16", "experts": 128, "top": 8, "hidden": 1536,
         "inner": 768, "lanes": 2047},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _groups(rng, low, high):
    """A number of values in whole groups."""
    return GROUP * _spread(rng, low // GROUP, high // GROUP)


def _draw_one(rng):
    kind = rng.choice(["quant", "product", "product", "route", "experts", "experts"])
    if kind == "quant":
        return {"kind": kind, "type": rng.choice(["f32", "bf16"]), "rows": _spread(rng, 1, 16384),
                "cols": _groups(rng, 64, 12288)}
    if kind == "product":
        lanes = rng.choice([1, _spread(rng, 2, 16), _spread(rng, 17, 64), _spread(rng, 65, 2048)])
        return {"kind": kind, "type": rng.choice(["f32", "bf16", "mx4"]), "rows": _spread(rng, 16, 16384),
                "cols": _groups(rng, 64, 8192), "lanes": lanes}
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        each = _spread(rng, 4, 512 // groups)
        kept = rng.randint(1, groups)
        return {"kind": kind, "experts": groups * each, "top": rng.randint(1, min(8, kept * each)),
                "score": rng.choice(["softmax", "sigmoid"]), "groups": groups, "kept": kept,
                "lanes": _spread(rng, 1, 16384)}
    count = _spread(rng, 4, 128)
    return {"kind": kind, "type": rng.choice(["f32", "bf16"]), "experts": count, "top": rng.randint(1, min(8, count)),
            "hidden": _groups(rng, 256, 2048), "inner": _groups(rng, 64, 1024),
            "lanes": rng.choice([1, _spread(rng, 2, 16), _spread(rng, 17, 2047)])}


def draw(rng):
    while True:
        case = _draw_one(rng)
        cost, most = work(case), [work(c) for c in listed() if c["kind"] == case["kind"]]
        if all(cost[key] <= max(w[key] for w in most) for key in ("bytes", "flops")):
            return case


# ---- microscaled rows -----------------------------------------------------------

def _power(exponent):
    """2^exponent, whole numbers above -127, in 32 bits."""
    return ((exponent + 127).to(torch.int32) << 23).view(torch.float32)


def _quantise(x):
    """(codes one a value, scale bytes) of rows [n, cols].  A power of two changes no digits, so 32 bits
    decide as the reals do."""
    x = x.view(x.shape[0], -1, GROUP)
    top = x.abs().amax(-1)
    power = torch.where(top > 0, torch.frexp(top)[1].to(torch.int32) - 3, -127).clamp(min=-127)
    m = (x * _power(-power).unsqueeze(-1)).abs()
    level = torch.where(m < 2, (2 * m).round(), torch.where(m < 4, 2 + m.round(), 4 + (m / 2).round())).clamp(max=7)
    code = level + 8 * (x < 0)
    return code.to(torch.uint8).view(x.shape[0], -1), (power + 127).to(torch.uint8)


def _pack(code):
    return code[:, 0::2] | (code[:, 1::2] << 4)


def _values(codes, scales):
    """What packed codes [n, cols / 2] and scale bytes [n, cols / 32] stand for, in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1, GROUP)
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), device=codes.device)
    return (table[code.long()] * _power(scales.int() - 127).unsqueeze(-1)).view(codes.shape[0], -1)


# ---- inputs ---------------------------------------------------------------------

def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rows(g, lanes, width):
    """Activations as a norm leaves them: unit variance, channels of unlike size."""
    size = torch.exp(0.4 * torch.randn((1, width), device="cuda", generator=g))
    return torch.randn((lanes, width), device="cuda", generator=g) * size


def _sheet(g, rows, cols):
    """A microscaled weight: packed codes and scale bytes."""
    codes = torch.empty((rows, cols // 2), dtype=torch.uint8, device="cuda")
    scales = torch.empty((rows, cols // GROUP), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 25) // cols)
    for at in range(0, rows, step):
        n = min(step, rows - at)
        code, scale = _quantise(torch.randn((n, cols), device="cuda", generator=g) / math.sqrt(cols))
        codes[at:at + n], scales[at:at + n] = _pack(code), scale
    return codes, scales


def _picks(g, case):
    """Experts of every lane and their weights, some experts more liked than others; the last lanes of
    a batch of several are padding, which takes none."""
    lanes, count, top = case["lanes"], case["experts"], case["top"]
    liked = 0.5 * torch.randn((1, count), device="cuda", generator=g)
    score = torch.randn((lanes, count), device="cuda", generator=g) + liked
    best, pick = torch.topk(score, top, dim=1)
    weight = torch.softmax(best, 1)
    if lanes > 32:
        pick[-(lanes // 32):] = -1
    return pick.to(torch.int32).contiguous(), weight.contiguous()


def _inputs(case, seed):
    """The tensors of a case, from the seed alone."""
    g, kind = _random(seed), case["kind"]
    if kind == "quant":
        return {"x": _rows(g, case["rows"], case["cols"]).to(TYPES[case["type"]])}
    if kind == "product":
        sheet = _sheet(g, case["rows"], case["cols"])
        x = _rows(g, case["lanes"], case["cols"])
        if case["type"] == "mx4":
            code, scale = _quantise(x)
            return {"sheet": sheet, "x": (_pack(code), scale)}
        return {"sheet": sheet, "x": x.to(TYPES[case["type"]])}
    if kind == "route":
        spread = 0.5 * torch.randn((1, case["experts"]), device="cuda", generator=g)
        logits = 1.5 * torch.randn((case["lanes"], case["experts"]), device="cuda", generator=g) + spread
        bias = 0.1 * torch.randn(case["experts"], device="cuda", generator=g) if case["score"] == "sigmoid" else None
        return {"logits": logits, "bias": bias}
    count, hidden, inner = case["experts"], case["hidden"], case["inner"]
    pick, weight = _picks(g, case)
    return {"gate_up": _sheet(g, count * 2 * inner, hidden), "down": _sheet(g, count * hidden, inner),
            "x": _rows(g, case["lanes"], hidden).to(TYPES[case["type"]]), "pick": pick, "weight": weight}


# ---- what a program holds -------------------------------------------------------

_BACKEND = None


def _backend():
    """The process's one desk."""
    global _BACKEND
    if _BACKEND is None:
        from igllm_amd.backend import Backend
        _BACKEND = Backend()
    return _BACKEND


class Buffer:
    """A torch tensor as the backend's device buffer."""

    def __init__(self, tensor):
        self.tensor = tensor
        self.ptr = tensor.data_ptr()


def _store_type(tensor):
    from igllm_amd import native
    return native.IGL_STORE_BF16 if tensor.dtype == torch.bfloat16 else native.IGL_STORE_F32


def _held(sheet, rows, cols):
    return _backend().mx4(rows, cols, Buffer(sheet[0]), Buffer(sheet[1]))


def prepare(case, seed):
    given = _inputs(case, seed)
    state = {"case": dict(case), "given": given}
    if own:
        _prepare_own(case, given, state)
    torch.cuda.synchronize()
    return state


def _prepare_own(case, given, state):
    be, kind = _backend(), case["kind"]
    if kind == "quant":
        state["store"] = be.mx4(case["rows"], case["cols"])
        state["in"] = Buffer(given["x"])
        state["out"] = Buffer(torch.empty((case["rows"], case["cols"]), device="cuda"))
    elif kind == "product":
        state["sheet"] = _held(given["sheet"], case["rows"], case["cols"])
        both = case["type"] == "mx4"
        state["in"] = _held(given["x"], case["lanes"], case["cols"]) if both else Buffer(given["x"])
        form = torch.float32 if both else given["x"].dtype
        state["out"] = Buffer(torch.empty((case["lanes"], case["rows"]), dtype=form, device="cuda"))
    elif kind == "route":
        from igllm_amd import native
        score = native.IGL_ROUTE_SOFTMAX if case["score"] == "softmax" else native.IGL_ROUTE_SIGMOID
        state["rule"] = native.Route(case["experts"], case["top"], score, case["groups"], case["kept"], 2, 1, 1.0)
        state["in"] = Buffer(given["logits"])
        state["bias"] = Buffer(given["bias"]) if given["bias"] is not None else None
        shape = (case["lanes"], case["top"])
        state["pick"] = Buffer(torch.empty(shape, dtype=torch.int32, device="cuda"))
        state["weight"] = Buffer(torch.empty(shape, device="cuda"))
    else:
        from igllm_amd import native
        count, hidden, inner = case["experts"], case["hidden"], case["inner"]
        state["experts"] = be.experts(_held(given["gate_up"], count * 2 * inner, hidden),
                                      _held(given["down"], count * hidden, inner), count, hidden, inner,
                                      native.IGL_GATE_GELU)
        state["in"], state["pick"], state["weight"] = (Buffer(given[k]) for k in ("x", "pick", "weight"))
        state["out"] = Buffer(torch.empty_like(given["x"]))


def _run_own(s):
    c, be = s["case"], _backend()
    if c["kind"] == "quant":
        out = s["out"]
        be.mx4_lay_dev(s["store"], 0, c["rows"], s["in"], _store_type(s["in"].tensor), c["cols"])
        be.mx4_read_dev(s["store"], 0, c["rows"], out, _store_type(out.tensor), c["cols"])
        return out.tensor
    if c["kind"] == "product":
        out = s["out"]
        if c["type"] == "mx4":
            be.mx4_mat_mx4_dev(s["sheet"], s["in"], 0, c["lanes"], out, _store_type(out.tensor), c["rows"])
        else:
            be.mx4_mat_mat_dev(s["sheet"], s["in"], _store_type(s["in"].tensor), c["cols"], c["lanes"], out,
                               _store_type(out.tensor), c["rows"])
        return out.tensor
    if c["kind"] == "route":
        be.route_dev(s["rule"], s["in"], c["experts"], c["lanes"], s["bias"], None, s["pick"], s["weight"])
        return s["pick"].tensor, s["weight"].tensor
    out, form = s["out"], _store_type(s["out"].tensor)
    be.experts_dev(s["experts"], s["in"], form, c["hidden"], c["lanes"], s["pick"], s["weight"], c["top"], out, form,
                   c["hidden"])
    return out.tensor


def run(state):
    if own:
        return _run_own(state)
    case, given = state["case"], state["given"]
    return {"quant": _plain_quant, "product": _plain_product, "route": _plain_route,
            "experts": _plain_experts}[case["kind"]](case, given)


def _plain_quant(case, given):
    code, scale = _quantise(given["x"].float())
    return _values(_pack(code), scale)


def _plain_product(case, given):
    x = _values(*given["x"]) if case["type"] == "mx4" else given["x"].float()
    out = x @ _values(*given["sheet"]).T
    return out if case["type"] == "mx4" else out.to(given["x"].dtype)


def _plain_route(case, given):
    # which of two scores is larger is decided in 64 bits
    x = given["logits"].double()
    if case["score"] == "softmax":
        score = torch.exp(x - x.amax(1, keepdim=True))
        score = score / score.sum(1, keepdim=True)
    else:
        score = 1 / (1 + torch.exp(-x))
    choice = score if given["bias"] is None else score + given["bias"].double()
    if case["groups"] > 1:
        parts = choice.view(case["lanes"], case["groups"], -1)
        best = torch.sort(parts, dim=-1, descending=True)[0][..., :2].sum(-1)
        kept = torch.sort(best, dim=1, descending=True, stable=True)[1][:, :case["kept"]]
        hide = torch.ones_like(best, dtype=torch.bool).scatter_(1, kept, False)
        choice = parts.masked_fill(hide.unsqueeze(-1), -math.inf).view(case["lanes"], -1)
    pick = torch.sort(choice, dim=1, descending=True, stable=True)[1][:, :case["top"]]
    weight = score.gather(1, pick)
    return pick.to(torch.int32), (weight / weight.sum(1, keepdim=True)).float()


def _gelu(x):
    return 0.5 * x * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))


def _plain_experts(case, given):
    lanes, top, hidden, inner = case["lanes"], case["top"], case["hidden"], case["inner"]
    x, pick = given["x"].float(), given["pick"]
    rows = torch.zeros((lanes * top, hidden), device="cuda")
    for e in range(case["experts"]):
        slot = (pick.view(-1) == e).nonzero().view(-1)
        if not len(slot):
            continue
        here = slice(e * 2 * inner, (e + 1) * 2 * inner), slice(e * hidden, (e + 1) * hidden)
        gate_up = _values(*(t[here[0]] for t in given["gate_up"]))
        both = x[slot // top] @ gate_up.T
        rows[slot] = (_gelu(both[:, :inner]) * both[:, inner:]) @ _values(*(t[here[1]] for t in given["down"])).T
    out = (rows.view(lanes, top, hidden) * given["weight"].unsqueeze(-1)).sum(1)
    return out.to(given["x"].dtype)


# ---- what a pass cannot do without ----------------------------------------------

def _mx4_bytes(rows, cols):
    return rows * (cols // 2 + cols // GROUP)


def work(case):
    kind = case["kind"]
    size = {"f32": 4, "bf16": 2}.get(case.get("type"))
    if kind == "quant":  # rows in, codes written and read, values out
        return {"bytes": case["rows"] * case["cols"] * (size + 4) + 2 * _mx4_bytes(case["rows"], case["cols"]),
                "flops": 0}
    if kind == "product":
        rows, cols, lanes = case["rows"], case["cols"], case["lanes"]
        x, out = (size * lanes * cols, size * lanes * rows) if size else (_mx4_bytes(lanes, cols), 4 * lanes * rows)
        return {"bytes": _mx4_bytes(rows, cols) + x + out, "flops": 2 * rows * cols * lanes}
    if kind == "route":
        return {"bytes": 4 * case["lanes"] * (case["experts"] + 2 * case["top"]) + 4 * case["experts"], "flops": 0}
    lanes, hidden, inner = case["lanes"], case["hidden"], case["inner"]
    slots = (lanes - (lanes // 32 if lanes > 32 else 0)) * case["top"]
    taken = min(case["experts"], slots)
    return {"bytes": taken * (_mx4_bytes(2 * inner, hidden) + _mx4_bytes(hidden, inner)) + 2 * size * lanes * hidden
            + 8 * lanes * case["top"], "flops": 6 * slots * hidden * inner}


# ---- the same in 64 bits --------------------------------------------------------

def _exact_values(codes, scales):
    table = torch.tensor([(-1.0) ** (c // 8) * E2M1[c % 8] for c in range(16)], dtype=torch.float64, device="cuda")
    out = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.float64, device="cuda")
    out[:, 0::2] = table[(codes % 16).long()]
    out[:, 1::2] = table[(codes // 16).long()]
    return out * torch.ldexp(torch.ones_like(scales, dtype=torch.float64),
                             scales.int() - 127).repeat_interleave(GROUP, 1)


def _exact_quant(x):
    """Every value's nearest level of its group's step, by search; halfway, the even code."""
    x = x.double().view(x.shape[0], -1, GROUP)
    top = x.abs().amax(-1, keepdim=True)
    step = torch.ldexp(torch.ones_like(top), (torch.floor(torch.log2(top.clamp(min=2.0 ** -125))) - 2).int())
    # log2 may round up to the next whole number just below it
    step = torch.where(4 * step > top.clamp(min=2.0 ** -125), step / 2, step)
    levels = torch.tensor(E2M1, dtype=torch.float64, device="cuda")
    m = (x.abs() / step).clamp(max=6.0)
    low = torch.searchsorted(levels, m.contiguous(), right=True).clamp(1, 7) - 1
    under, over = m - levels[low], levels[low + 1] - m
    low = torch.where((under > over) | ((under == over) & (low % 2 == 1)), low + 1, low)
    return (torch.copysign(levels[low], x) * step).view(x.shape[0], -1)


def _exact_route(case, given):
    x = given["logits"].double().cpu().numpy()
    if case["score"] == "softmax":
        score = np.exp(x - x.max(1, keepdims=True))
        score /= score.sum(1, keepdims=True)
    else:
        score = 1 / (1 + np.exp(-x))
    choice = score if given["bias"] is None else score + given["bias"].double().cpu().numpy()
    lanes, each = len(x), case["experts"] // case["groups"]
    if case["groups"] > 1:
        parts = np.sort(choice.reshape(lanes, case["groups"], each), -1)
        order = np.argsort(-parts[..., -2:].sum(-1), 1, kind="stable")
        shown = np.zeros((lanes, case["groups"]), bool)
        np.put_along_axis(shown, order[:, :case["kept"]], True, 1)
        choice = np.where(np.repeat(shown, each, 1), choice, -np.inf)
    pick = np.argsort(-choice, 1, kind="stable")[:, :case["top"]]
    weight = np.take_along_axis(score, pick, 1)
    return (torch.from_numpy(pick.astype(np.int32)).cuda(),
            torch.from_numpy(weight / weight.sum(1, keepdims=True)).cuda())


def _exact_experts(case, given):
    lanes, hidden, inner = case["lanes"], case["hidden"], case["inner"]
    x, out = given["x"].double(), torch.zeros((lanes, hidden), dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        at = given["pick"] == e
        taken = at.any(1).nonzero().view(-1)
        if not len(taken):
            continue
        share = (given["weight"].double() * at)[taken].sum(1, keepdim=True)
        gate, up = (_exact_values(*(t[(2 * e + i) * inner:(2 * e + i + 1) * inner] for t in given["gate_up"]))
                    for i in (0, 1))
        g = x[taken] @ gate.T
        h = g / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * (x[taken] @ up.T)
        out[taken] += share * (h @ _exact_values(*(t[e * hidden:(e + 1) * hidden] for t in given["down"])).T)
    return out


def exact(case, seed):
    given, kind = _inputs(case, seed), case["kind"]
    if kind == "quant":
        step = max(1, (1 << 24) // case["cols"])
        return torch.cat([_exact_quant(part) for part in given["x"].split(step)])
    if kind == "product":
        x = _exact_values(*given["x"]) if case["type"] == "mx4" else given["x"].double()
        step = max(1, (1 << 26) // case["cols"])
        return torch.cat([x @ _exact_values(*part).T
                          for part in zip(*(t.split(step) for t in given["sheet"]))], 1)
    return _exact_route(case, given) if kind == "route" else _exact_experts(case, given)
