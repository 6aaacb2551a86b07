"""What a program that keeps its key/value cache in 4 bits has this framework
do, as cases that can be measured: laying new rows into the ring, reading rows
back, and attention over the ring with a sliding window and first positions
that stay visible, from one decode step to a whole prompt.

The ring.  A row of a position is `kv` heads of `head` values.  Every 32 values
of a head share a gain, an e4m3 byte g, and the layer side has one scale s: a
code stands for level * g * s, its level a whole number -8 .. 7 ("int4", code =
level + 8) or one of 0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives ("e2m1").
Written rows take the e4m3 value nearest the group's largest magnitude over
top * s (top 7 or 6) as gain, and each value's nearest level of it, ties to
even.  Codes lie [span][kv * head / 2], two a byte, low nibble first; gains
[kv * head / 32][span rounded up to 64].  The first `sinks` positions keep slots
0 .. sinks - 1, position p after them slot sinks + (p - sinks) % (span - sinks).

Kinds:
  lay     rows of new positions into the ring, and read back from it
  read    rows of positions of a ring
  attend  queries of consecutive positions over a ring: position p sees the
          last `window` positions up to itself (0: all) and the first `sinks`
"""
import math

import torch

own = False

GROUP = 32
TOP = {"int4": 7, "e2m1": 6}
SCALE = 6.0 / 448.0  # calibrated: the largest magnitude of a layer's rows over e4m3's
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---- the cases ----------------------------------------------------------------

def listed():
    return [
        # a decode step's row on a sliding layer
        {"name": "lay_1_lane", "kind": "lay", "format": "int4", "kv": 1, "head": 256, "sinks": 4, "span": 516,
         "place": 700, "lanes": 1},
        # a prompt's rows on a global layer
        {"name": "lay_2047_lanes", "kind": "lay", "format": "e2m1", "kv": 1, "head": 512, "sinks": 0, "span": 4096,
         "place": 1, "lanes": 2047},
        # a long prompt's rows, eight key/value heads
        {"name": "lay_16384_lanes", "kind": "lay", "format": "int4", "kv": 8, "head": 128, "sinks": 0,
         "span": 16384, "place": 0, "lanes": 16384},
        # a sliding layer's ring read back whole, across its wrap
        {"name": "read_512", "kind": "read", "format": "int4", "kv": 1, "head": 256, "sinks": 4, "span": 516,
         "place": 900, "lanes": 512},
        # a long context read back, to be kept or moved to another form
        {"name": "read_131071", "kind": "read", "format": "e2m1", "kv": 4, "head": 128, "sinks": 0, "span": 131072,
         "place": 1, "lanes": 131071},
        # a decode step on a sliding layer that has forgotten its prompt but for four first ids
        {"name": "attend_window", "kind": "attend", "format": "int4", "kv": 1, "share": 8, "head": 256, "sinks": 4,
         "span": 516, "place": 5000, "window": 512, "lanes": 1},
        # a decode step on a global layer
        {"name": "attend_16384", "kind": "attend", "format": "int4", "kv": 1, "share": 8, "head": 256, "sinks": 0,
         "span": 16384, "place": 16383, "window": 0, "lanes": 1},
        # a decode step over the longest context, eight key/value heads
        {"name": "attend_131072", "kind": "attend", "format": "e2m1", "kv": 8, "share": 4, "head": 128, "sinks": 0,
         "span": 131072, "place": 131071, "window": 0, "lanes": 1},
        # a speculative block on a global layer
        {"name": "attend_block", "kind": "attend", "format": "e2m1", "kv": 1, "share": 8, "head": 512, "sinks": 0,
         "span": 16384, "place": 16000, "window": 0, "lanes": 5},
        # a short turn of a conversation, small heads in odd shares
        {"name": "attend_37_lanes", "kind": "attend", "format": "int4", "kv": 2, "share": 7, "head": 64, "sinks": 1,
         "span": 1100, "place": 3001, "window": 1024, "lanes": 37},
        # a prompt on a sliding layer
        {"name": "attend_2047_window", "kind": "attend", "format": "e2m1", "kv": 1, "share": 8, "head": 256,
         "sinks": 4, "span": 2600, "place": 0, "window": 512, "lanes": 2047},
        # a prompt on a global layer
        {"name": "attend_2047_lanes", "kind": "attend", "format": "int4", "kv": 1, "share": 8, "head": 512,
         "sinks": 0, "span": 2048, "place": 0, "window": 0, "lanes": 2047},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_one(rng):
    kind = rng.choice(["lay", "lay", "read", "attend", "attend", "attend"])
    case = {"kind": kind, "format": rng.choice(["int4", "e2m1"]), "kv": rng.choice([1, 1, 2, 3, 8]),
            "head": rng.choice([64, 128, 256, 512]), "sinks": rng.choice([0, 0, 1, 4, 17])}
    if kind != "attend":
        case["lanes"] = _spread(rng, 1, 16384) if kind == "lay" else _spread(rng, 1, 131072)
        case["place"] = _spread(rng, 1, 131072) - 1
        case["span"] = case["sinks"] + case["lanes"] + _spread(rng, 1, 4096) - 1
        return case
    case["share"] = rng.choice([1, 2, 4, 5, 7, 8, 8, 8, 12, 16])
    case["lanes"] = rng.choice([1, 1, _spread(rng, 2, 16), _spread(rng, 17, 2047)])
    case["window"] = rng.choice([0, 0, 512, _spread(rng, 16, 8192)])
    case["place"] = _spread(rng, 1, 131072) - 1 if case["lanes"] <= 16 else _spread(rng, 1, 8192) - 1
    last = case["place"] + case["lanes"]
    kept = min(last, case["window"] + case["lanes"] - 1) if case["window"] else last
    case["span"] = case["sinks"] + kept + _spread(rng, 1, 1024) - 1
    return case


def draw(rng):
    most = {kind: max((work(c) for c in listed() if c["kind"] == kind), key=lambda w: w["bytes"])["bytes"]
            for kind in ("lay", "read", "attend")}
    flops = max(work(c)["flops"] for c in listed() if c["kind"] == "attend")
    while True:
        case = _draw_one(rng)
        cost = work(case)
        if cost["bytes"] <= most[case["kind"]] and (case["kind"] != "attend" or cost["flops"] <= flops):
            return case


# ---- the ring -------------------------------------------------------------------

def _slots(case, places):
    """The slots of positions."""
    sinks = case["sinks"]
    return torch.where(places < sinks, places, sinks + (places - sinks) % (case["span"] - sinks))


def _seen(case):
    """The positions that some lane of an attention sees, in order."""
    last = case["place"] + case["lanes"]
    first = max(0, case["place"] + 1 - case["window"]) if case["window"] else 0
    return list(range(min(case["sinks"], first))) + list(range(first, last))


def _e4m3(x):
    """The e4m3 value nearest x >= 0, ties to even, 448 at most (64 bits)."""
    power = torch.frexp(x.clamp(min=2.0 ** -6))[1] - 1  # x in [2^power, 2^(power + 1))
    unit = torch.ldexp(torch.ones_like(x), power - 3)
    return ((x / unit).round() * unit).clamp(max=448.0)


def _quantise(x, form):
    """(codes, gains) of rows [n, width]: codes one a value, gains as e4m3 values [n, width / 32].
    Both are decisions next to borders: 64 bits."""
    x = x.double().view(x.shape[0], -1, GROUP)
    scale = float(torch.tensor(SCALE, dtype=torch.float32))
    gain = _e4m3(x.abs().amax(-1) / (TOP[form] * scale))
    step = (gain * scale).unsqueeze(-1)
    v = torch.where(step > 0, x / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(x))
    if form == "int4":
        code = v.round().clamp(-7, 7) + 8
    else:
        m = v.abs()
        level = torch.where(m < 2, (2 * m).round(), torch.where(m < 4, 2 + m.round(), 4 + (m / 2).round()))
        level = level.clamp(max=7)
        code = level + 8 * ((v < 0) & (level > 0))
    return code.to(torch.uint8).view(x.shape[0], -1), gain


def _values(codes, gains, form):
    """What packed codes [n, width / 2] and gains [n, width / 32] (e4m3 bytes) stand for, in 32 bits."""
    code = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1)
    if form == "int4":
        level = code.float() - 8
    else:
        table = torch.tensor(E2M1, device=codes.device)
        level = table[(code & 7).long()] * (1 - 2 * (code >> 3).float())
    gain = gains.contiguous().view(torch.float8_e4m3fn).float()
    return (level.view(codes.shape[0], -1, GROUP) * gain.unsqueeze(-1) * SCALE).view(codes.shape[0], -1)


def _random(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _rows(g, lanes, width):
    """Rows as a model's norms leave them: unit variance, channels of unlike size."""
    size = torch.exp(0.4 * torch.randn((1, width), device="cuda", generator=g))
    return (torch.randn((lanes, width), device="cuda", generator=g) * size).clamp_(-6, 6)


def _ring(g, case, filled):
    """One side of a ring: packed codes and gain bytes; of rows, or as allocated."""
    span, width = case["span"], case["kv"] * case["head"]
    room = (span + 63) // 64 * 64
    codes = torch.zeros((span, width // 2), dtype=torch.uint8, device="cuda")
    gains = torch.zeros((width // GROUP, room), dtype=torch.uint8, device="cuda")
    if filled:
        size = torch.exp(0.4 * torch.randn((1, width), device="cuda", generator=g))
        for at in range(0, span, 8192):
            n = min(8192, span - at)
            rows = (torch.randn((n, width), device="cuda", generator=g) * size).clamp_(-6, 6)
            code, gain = _quantise(rows, case["format"])
            codes[at:at + n] = code[:, 0::2] | (code[:, 1::2] << 4)
            gains[:, at:at + n] = gain.float().to(torch.float8_e4m3fn).view(torch.uint8).T
    return codes, gains


def _inputs(case, seed):
    """The rings and what is put to them, from the seed alone."""
    g = _random(seed)
    width, lanes = case["kv"] * case["head"], case["lanes"]
    rings = [_ring(g, case, case["kind"] != "lay") for _ in range(2)]
    if case["kind"] == "lay":
        return rings, [_rows(g, lanes, width), _rows(g, lanes, width)]
    if case["kind"] == "read":
        return rings, []
    return rings, [torch.randn((lanes, case["share"] * width), device="cuda", generator=g)]


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


def prepare(case, seed):
    rings, given = _inputs(case, seed)
    state = {"case": dict(case), "rings": rings, "given": given}
    if own:
        from igllm_amd import native
        width, lanes = case["kv"] * case["head"], case["lanes"]
        form = native.IGL_CACHE4_INT4 if case["format"] == "int4" else native.IGL_CACHE4_E2M1
        (kc, kg), (vc, vg) = rings
        state["store"] = _backend().cache4(form, case["span"], case["sinks"], case["kv"], case["head"], SCALE, SCALE,
                                           Buffer(kc), Buffer(kg), Buffer(vc), Buffer(vg))
        state["in"] = [Buffer(t) for t in given]
        shapes = [given[0].shape] if case["kind"] == "attend" else [(lanes, width)] * 2
        state["out"] = [Buffer(torch.empty(s, device="cuda")) for s in shapes]
    torch.cuda.synchronize()
    return state


def _run_own(s):
    c, be, out = s["case"], _backend(), s["out"]
    width = c["kv"] * c["head"]
    if c["kind"] == "attend":
        stride = c["share"] * width
        be.attend4_lanes_dev(s["store"], c["share"], s["in"][0], stride, c["place"], c["window"], c["lanes"],
                             1.0 / math.sqrt(c["head"]), out[0])
        return out[0].tensor
    if c["kind"] == "lay":
        be.cache4_lay_dev(s["store"], s["in"][0], s["in"][1], width, c["place"], c["lanes"])
    be.cache4_read_dev(s["store"], c["place"], c["lanes"], out[0], out[1], width)
    return out[0].tensor, out[1].tensor


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    if c["kind"] == "attend":
        return _plain_attend(c, state["rings"], state["given"][0])
    places = torch.arange(c["place"], c["place"] + c["lanes"], device="cuda")
    slots = _slots(c, places)
    out = []
    for side, (codes, gains) in enumerate(state["rings"]):
        if c["kind"] == "lay":
            code, gain = _quantise(state["given"][side], c["format"])
            codes[slots] = code[:, 0::2] | (code[:, 1::2] << 4)
            gains[:, slots] = gain.float().to(torch.float8_e4m3fn).view(torch.uint8).T
        out.append(_values(codes[slots], gains[:, slots].T, c["format"]))
    return tuple(out)


def _plain_attend(c, rings, query):
    lanes, kv, share, head = c["lanes"], c["kv"], c["share"], c["head"]
    seen = torch.tensor(_seen(c), device="cuda")
    slots = _slots(c, seen)
    key, value = (_values(codes[slots], gains[:, slots].T, c["format"]).view(-1, kv, head) for codes, gains in rings)
    lane = c["place"] + torch.arange(lanes, device="cuda")[:, None]
    show = seen[None] <= lane
    if c["window"]:
        show &= (seen[None] > lane - c["window"]) | (seen[None] < c["sinks"])
    q = query.view(lanes, kv, share, head)
    out = torch.empty_like(q)
    for h in range(kv):
        score = q[:, h].reshape(lanes * share, head) @ key[:, h].T.contiguous() / math.sqrt(head)
        score = score.view(lanes, share, -1).masked_fill(~show[:, None], -math.inf)
        weight = torch.exp(score - score.amax(-1, keepdim=True))
        weight = weight / weight.sum(-1, keepdim=True)
        out[:, h] = (weight.view(lanes * share, -1) @ value[:, h].contiguous()).view(lanes, share, head)
    return out.view(lanes, -1)


# ---- what a pass cannot do without ----------------------------------------------

def work(case):
    width, lanes = case["kv"] * case["head"], case["lanes"]
    row = 2 * (width // 2 + width // GROUP)  # a position's codes and gains, both sides
    if case["kind"] == "lay":  # rows in, the ring's rows written and read, values out
        return {"bytes": lanes * (2 * 2 * 4 * width + 2 * row), "flops": 0}
    if case["kind"] == "read":
        return {"bytes": lanes * (row + 2 * 4 * width), "flops": 0}
    sums = 0
    for p in range(case["place"], case["place"] + lanes):
        first = max(0, p + 1 - case["window"]) if case["window"] else 0
        sums += p + 1 - first + min(case["sinks"], first)
    return {"bytes": len(_seen(case)) * row + 2 * 4 * lanes * case["share"] * width,
            "flops": 4 * case["share"] * width * sums}


# ---- the same in 64 bits --------------------------------------------------------

def _nearest(x, table):
    """The index of the entry of an ascending table nearest x; halfway, the even index."""
    low = torch.searchsorted(table, x.contiguous(), right=True).clamp(1, len(table) - 1) - 1
    under, over = x - table[low], table[low + 1] - x
    return torch.where((under > over) | ((under == over) & (low % 2 == 1)), low + 1, low)


def _e4m3_table():
    """The 127 e4m3 values from 0 to 448, by code."""
    return torch.tensor([m / 512 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)][:127],
                        dtype=torch.float64, device="cuda")


def _levels(form):
    """What the sixteen codes stand for before the gain."""
    whole = [c - 8 for c in range(16)] if form == "int4" else list(E2M1) + [-v for v in E2M1]
    return torch.tensor(whole, dtype=torch.float64, device="cuda")


def _exact_lay(rows, form):
    x = rows.double().view(rows.shape[0], -1, GROUP)
    scale = float(torch.tensor(SCALE, dtype=torch.float32))
    gains = _e4m3_table()
    gain = gains[_nearest(x.abs().amax(-1) / (TOP[form] * scale), gains)]
    step = (gain * scale).unsqueeze(-1)
    half = _levels(form)[8:16] if form == "int4" else _levels(form)[:8]
    level = half[_nearest(x.abs() / step.clamp(min=1e-300), half)]
    return (torch.where(x < 0, -level, level) * step).view(rows.shape[0], -1)


def _exact_values(codes, gains, form):
    levels, table = _levels(form), _e4m3_table()
    scale = float(torch.tensor(SCALE, dtype=torch.float32))
    out = torch.empty((codes.shape[0], 2 * codes.shape[1]), dtype=torch.float64, device="cuda")
    out[:, 0::2] = levels[(codes % 16).long()]
    out[:, 1::2] = levels[(codes // 16).long()]
    return out * (table[gains.long()] * scale).repeat_interleave(GROUP, 1)


def exact(case, seed):
    rings, given = _inputs(case, seed)
    if case["kind"] == "lay":
        return tuple(_exact_lay(rows, case["format"]) for rows in given)
    sinks, back = case["sinks"], case["span"] - case["sinks"]
    places = _seen(case) if case["kind"] == "attend" else range(case["place"], case["place"] + case["lanes"])
    at = torch.tensor([p if p < sinks else sinks + (p - sinks) % back for p in places], device="cuda")
    if case["kind"] == "read":
        return tuple(_exact_values(codes[at], gains[:, at].T, case["format"]) for codes, gains in rings)
    kv, share, head, lanes = case["kv"], case["share"], case["head"], case["lanes"]
    places = torch.tensor(list(places), device="cuda")
    lane = torch.arange(case["place"], case["place"] + lanes, device="cuda").unsqueeze(1)
    hide = places > lane
    if case["window"]:
        hide = hide | ((places <= lane - case["window"]) & (places >= sinks))
    out = torch.empty((lanes, kv * share * head), dtype=torch.float64, device="cuda")
    for k in range(kv):
        dims, packed = slice(k * head // GROUP, (k + 1) * head // GROUP), slice(k * head // 2, (k + 1) * head // 2)
        key, value = (_exact_values(codes[at][:, packed], gains[dims][:, at].T, case["format"])
                      for codes, gains in rings)
        for h in range(k * share, (k + 1) * share):
            cols = slice(h * head, (h + 1) * head)
            score = given[0][:, cols].double() @ key.T / math.sqrt(head)
            out[:, cols] = torch.softmax(score.masked_fill(hide, -math.inf), -1) @ value
    return out
