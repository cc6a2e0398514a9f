"""Workloads of the token operators: quantize_rows, linear and linear_grouped.

Each case is one call a serving program makes on device tensors.  `run` makes it with the
framework's operators where `own` is true, and with elementary torch operations in 32 bits
where it is false.  `exact` computes the same from the definition in 64 bits.

Codes that `quantize_rows` returns are whole numbers by definition (the exact quotient
rounded half away from zero), so they are returned as such.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_ops = None


def _handle():
    """The program's one operator handle (error word, launch attributes), made at its first use."""
    global _ops
    if _ops is None:
        from ptq_int8_lab_b200.ops import Int8Ops
        _ops = Int8Ops(0)
    return _ops


# ------------------------------------------------------------------------------ cases

def listed():
    q = dict(kind="quantize", top=0)
    lin = dict(kind="linear", bits=8, gated=False, bias=False, out_type="bf16")
    exp = dict(kind="experts", bits=8, gated=False, bias=False, out_type="bf16", skew=0.3)
    return [
        # one generated token's hidden state, between two layers: launch latency
        dict(q, name="quantize 1 token", tokens=1, width=4096, type="bf16"),
        # a long prompt's hidden states: memory bandwidth
        dict(q, name="quantize 8192 tokens", tokens=8192, width=4096, type="bf16"),
        # an odd width, so that rows start at any 4-byte boundary; 32-bit states
        dict(q, name="quantize odd width", tokens=2047, width=1001, type="f32"),
        # dispatch of a prompt to experts: each token's codes written once per chosen expert
        dict(q, name="quantize to experts", tokens=4096, width=2048, type="f16", top=4),
        # a projection for one generated token: the weights are read once
        dict(lin, name="linear 1 token", tokens=1, inp=4096, out=4096),
        # first half of an MLP for a batch of 16 generating sequences, packed 4-bit weights
        dict(lin, name="linear 16 tokens int4 gated", tokens=16, inp=4096, out=8192, bits=4, gated=True),
        # a short ragged prompt through a narrow projection with bias, kept in 32 bits
        dict(lin, name="linear 333 tokens ragged", tokens=333, inp=2000, out=1270, bias=True, out_type="f32"),
        # first half of an MLP for a prompt, packed 4-bit weights
        dict(lin, name="linear 4096 tokens int4 gated", tokens=4096, inp=4096, out=8192, bits=4, gated=True),
        # the largest: a batch of long prompts through a wide projection
        dict(lin, name="linear 16384 tokens", tokens=16384, inp=8192, out=8192),
        # a few generating sequences spread over many experts: most experts idle, the others have a row or two
        dict(exp, name="experts 8 tokens", tokens=8, top=2, experts=32, inp=2048, out=1024, gated=True),
        # a prompt over many experts, gated, unevenly loaded
        dict(exp, name="experts 4096 tokens gated", tokens=4096, top=4, experts=32, inp=2048, out=1024, gated=True),
        # second half of the experts' MLP with packed 4-bit weights and ragged sizes
        dict(exp, name="experts 1000 tokens int4", tokens=1000, top=2, experts=8, inp=1408, out=2050, bits=4, out_type="f16"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature count: a power of two, an odd multiple of 16, or any odd number."""
    how, v = rng.random(), _spread(rng, lo, hi)
    if how < 0.35:
        v = 1 << round(math.log2(v))
    elif how < 0.8:
        v = 16 * (v // 32 * 2 + 1)
    else:
        v |= 1
    return min(max(v, lo), hi)


_MOST = 2 * 16384 * 8192 * 8192   # operations of the largest listed case


def draw(rng):
    while True:
        kind = rng.choice(["quantize", "linear", "linear", "experts"])
        if kind == "quantize":
            return dict(kind=kind, tokens=_spread(rng, 1, 16384), width=_width(rng, 64, 8192),
                        type=rng.choice(["bf16", "bf16", "f16", "f32"]), top=rng.choice([0, 0, 1, 2, 4]))
        gated = rng.random() < 0.4
        case = dict(kind=kind, tokens=_spread(rng, 1, 16384), inp=_width(rng, 256, 16384), out=_width(rng, 64, 16384),
                    bits=rng.choice([8, 8, 4]), gated=gated, bias=rng.random() < 0.3,
                    out_type=rng.choice(["bf16", "bf16", "f16", "f32"]))
        if kind == "experts":
            case.update(tokens=_spread(rng, 1, 8192), inp=_width(rng, 256, 4096), out=_width(rng, 256, 4096),
                        top=rng.choice([1, 2, 4, 8]), experts=rng.choice([8, 16, 17, 32, 64]),
                        skew=rng.choice([0.0, 0.3, 1.0]))
        if work(case)["flops"] <= _MOST and work(case)["bytes"] <= 1 << 30:
            return case


def work(case):
    if case["kind"] == "quantize":
        rows = case["tokens"] * max(1, case["top"])
        read = case["tokens"] * case["width"] * _SIZE[case["type"]] + (4 * rows if case["top"] else 0)
        return {"bytes": read + rows * case["width"] + 4 * rows, "flops": 3 * rows * case["width"]}
    channels = case["out"] * (2 if case["gated"] else 1)
    rows, sets = case["tokens"], 1.0
    if case["kind"] == "experts":
        rows = case["tokens"] * case["top"]
        # experts that get a row at all, each token's choices being distinct and spread evenly
        sets = case["experts"] * (1.0 - (1.0 - case["top"] / case["experts"]) ** case["tokens"])
    weights = sets * channels * ((case["inp"] + 1) // 2 if case["bits"] == 4 else case["inp"])
    scales = 4 * rows + 4 * sets * channels * (2 if case["bias"] else 1)
    return {"bytes": rows * case["inp"] + weights + scales + rows * case["out"] * _SIZE[case["out_type"]],
            "flops": 2.0 * rows * channels * case["inp"]}


# ------------------------------------------------------------------------------ inputs

def _pitched(rows, width, dtype=torch.int8):
    """[..., width] bytes whose rows start at multiples of 16: how codes and weights are laid out once."""
    pitch = (width + 15) // 16 * 16
    return torch.zeros(*rows, pitch, dtype=dtype, device="cuda")[..., :width]


def _weights(g, lead, channels, inp, bits):
    """Codes of normally distributed weights, and their scales: one per channel."""
    shape = (*lead, channels, inp)
    if bits == 8:
        w = _pitched((*lead, channels), inp)
        for part in (w if lead else [w]):
            part.copy_(torch.randn((channels, inp), generator=g, device="cuda", dtype=torch.float16).mul_(34).round_().clamp_(-127, 127))
    else:
        half = (inp + 1) // 2
        w = _pitched((*lead, channels), half, torch.uint8)
        for part in (w if lead else [w]):
            c = torch.randn((channels, 2 * half), generator=g, device="cuda", dtype=torch.float16).mul_(2.4).round_().clamp_(-8, 7)
            if inp % 2:
                c[:, -1] = 0
            c = c.to(torch.int8)
            part.copy_((c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4))
    top = 127.0 if bits == 8 else 7.0
    scale = torch.rand(shape[:-1], generator=g, device="cuda") * (0.06 / top) + 0.05 / top
    return w, scale


def _hidden(g, rows, width, dtype):
    """Hidden states: normal, a few channels an order of magnitude larger, tokens of differing size."""
    x = torch.randn((rows, width), generator=g, device="cuda")
    x[:, torch.randint(0, width, (max(1, width // 256),), generator=g, device="cuda")] *= 12.0
    x *= torch.rand((rows, 1), generator=g, device="cuda") * 2 + 0.1
    return x.to(dtype)


def _routing(g, case):
    """(rows in order of their expert, offsets, the fullest expert's rows) of a router's choices."""
    logits = torch.randn((case["tokens"], case["experts"]), generator=g, device="cuda")
    logits += case["skew"] * torch.randn((case["experts"],), generator=g, device="cuda")
    ids = logits.topk(case["top"], dim=1).indices.reshape(-1)
    order = torch.argsort(ids, stable=True)
    counts = torch.bincount(ids, minlength=case["experts"])
    offsets = torch.zeros(case["experts"] + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = counts.cumsum(0)
    return (order // case["top"]).to(torch.int32), offsets, int(counts.max())


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    state = dict(case)
    if case["kind"] == "quantize":
        state["x"] = _hidden(g, case["tokens"], case["width"], _DT[case["type"]])
        rows, state["rows"] = case["tokens"], None
        if case["top"]:
            state["rows"] = _routing(g, dict(case, experts=16, skew=1.0))[0]
            rows = state["rows"].numel()
        state["codes"] = _pitched((rows,), case["width"])
        state["scale"] = torch.zeros(rows, device="cuda")
        return state
    rows, lead = case["tokens"], ()
    if case["kind"] == "experts":
        _, state["offsets"], state["most"] = _routing(g, case)
        rows, lead = case["tokens"] * case["top"], (case["experts"],)
    x = torch.randn((rows, case["inp"]), generator=g, device="cuda")
    x[:, ::97] *= 4.0
    top = x.abs().amax(1, keepdim=True)
    state["x"] = _pitched((rows,), case["inp"])
    state["x"].copy_((x * (127.0 / top)).round_())
    state["x_scale"] = (top[:, 0] / 127.0).contiguous()
    channels = case["out"] * (2 if case["gated"] else 1)
    state["w"], state["w_scale"] = _weights(g, lead, channels, case["inp"], case["bits"])
    state["bias"] = torch.randn((*lead, channels), generator=g, device="cuda") if case["bias"] else None
    state["y"] = torch.zeros((rows, case["out"]), dtype=_DT[case["out_type"]], device="cuda")
    return state


# ------------------------------------------------------------------------------ the plain forms

def _quantize_plain(x, rows):
    x = x.float()
    if rows is not None:
        x = x[rows.long()]
    top = x.abs().amax(1)
    scale = (top / torch.full_like(top, 127.0)).clamp_min(1e-8)
    s = scale[:, None]
    q = x / s
    # Half away from zero.  A quotient that reads k + 1/2 may have been rounded onto it: the sign of
    # the remainder x - q s tells, exactly, with s in two halves whose products with q are exact.
    t = q.trunc()
    s_hi = (s.contiguous().view(torch.int32) & -4096).view(torch.float32)
    rest = (x - q * s_hi) - q * (s - s_hi)
    sign = q.sign()
    half = torch.where(rest * sign >= 0, t + sign, t)
    codes = torch.where((q - t).abs() == 0.5, half, q.round())
    return codes.clamp(-128, 127).to(torch.int8), scale


def _values(w, bits, inp):
    """Weights' codes as 32-bit floats; int4 codes lie two per byte, the even one in the low half."""
    if bits == 8:
        return w.float()
    low, high = w & 15, w >> 4
    c = torch.stack((low, high), dim=-1).reshape(*w.shape[:-1], 2 * w.shape[-1])[..., :inp].float()
    return torch.where(c >= 8, c - 16, c)


def _finish_plain(acc, x_scale, w_scale, bias, gated, dtype):
    y = acc * (x_scale[:, None] * w_scale)
    if bias is not None:
        y = y + bias
    if gated:
        gate, up = y.chunk(2, dim=1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(dtype)


def _linear_plain(s):
    acc = s["x"].float() @ _values(s["w"], s["bits"], s["inp"]).t()
    return _finish_plain(acc, s["x_scale"], s["w_scale"], s["bias"], s["gated"], _DT[s["out_type"]])


def _experts_plain(s):
    rows = torch.arange(s["x"].shape[0], device="cuda")
    e = torch.searchsorted(s["offsets"][1:].long(), rows, right=True)
    slot = rows - s["offsets"].long()[e]
    padded = torch.zeros((s["experts"], s["most"], s["inp"]), device="cuda")
    padded[e, slot] = s["x"].float()
    acc = torch.bmm(padded, _values(s["w"], s["bits"], s["inp"]).transpose(1, 2))[e, slot]
    bias = None if s["bias"] is None else s["bias"][e]
    return _finish_plain(acc, s["x_scale"], s["w_scale"][e], bias, s["gated"], _DT[s["out_type"]])


def run(state):
    s = state
    if not own:
        if s["kind"] == "quantize":
            codes, scale = _quantize_plain(s["x"], s["rows"])
            return {"codes": codes, "scale": scale}
        return {"y": _linear_plain(s) if s["kind"] == "linear" else _experts_plain(s)}
    ops = _handle()
    if s["kind"] == "quantize":
        codes, scale = ops.quantize_rows(s["x"], rows=s["rows"], out=(s["codes"], s["scale"]))
        return {"codes": codes, "scale": scale}
    act = 1 if s["gated"] else 0   # EPI_SWIGLU, EPI_NONE
    if s["kind"] == "linear":
        return {"y": ops.linear(s["x"], s["x_scale"], s["w"], s["w_scale"], bias=s["bias"], bits=s["bits"], act=act,
                                out=s["y"])}
    return {"y": ops.linear_grouped(s["x"], s["x_scale"], s["offsets"], s["w"], s["w_scale"], bias=s["bias"],
                                    bits=s["bits"], act=act, out=s["y"])}


# ------------------------------------------------------------------------------ the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "quantize":
        x = s["x"].double()
        if s["rows"] is not None:
            x = x.index_select(0, s["rows"].long())
        scale = torch.clamp_min(x.abs().max(dim=1).values / 127.0, float(torch.tensor(1e-8)))
        # the scale is a 32-bit number, and the codes are those of that number
        q = x / scale.float().double()[:, None]
        codes = (q.abs() + 0.5).floor() * q.sign()
        return {"codes": codes.clamp(-128, 127).to(torch.int8), "scale": scale}
    y = torch.empty((s["x"].shape[0], s["out"]), dtype=torch.float64, device="cuda")
    experts = case.get("experts", 1)
    ends = s["offsets"].tolist() if experts > 1 else [0, s["x"].shape[0]]
    for e in range(experts):
        w, scale, bias = ((s[k][e] if experts > 1 else s[k]) if s[k] is not None else None for k in ("w", "w_scale", "bias"))
        if s["bits"] == 4:
            c = torch.empty((w.shape[0], 2 * w.shape[1]), dtype=torch.float64, device="cuda")
            c[:, 0::2], c[:, 1::2] = torch.remainder(w.double(), 16), torch.floor(w.double() / 16)
            w = (c - 16 * (c > 7))[:, :s["inp"]]
        w = w.double() * scale.double()[:, None]
        for a in range(ends[e], ends[e + 1], 4096):
            b = min(ends[e + 1], a + 4096)
            z = s["x"][a:b].double() @ w.t() * s["x_scale"][a:b].double()[:, None]
            if bias is not None:
                z += bias.double()
            if s["gated"]:
                z = torch.nn.functional.silu(z[:, :s["out"]]) * z[:, s["out"]:]
            y[a:b] = z
    return {"y": y}
