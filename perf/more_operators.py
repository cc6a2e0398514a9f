"""Workloads of the 4-bit operators of generation: the cache of keys and values (cache_write, cache_read,
cache_attention) and the product of float activations with 4-bit weights that have a scale per group (linear_w4).

Each case is one call a serving program makes on device tensors.  `run` makes it with the
framework's operators where `own` is true, and with elementary torch operations in 32 bits
where it is false.  `exact` computes the same from the definition in 64 bits.

A cache holds pages of a power of two tokens.  A token's key (and value) of a head is head_dim codes of 4 bits, two per
byte, the even one low, and a pair (step, least) of bf16: a code c stands for least + step * c.
A sequence's table names its pages, its length counts the tokens it has, the new ones among them.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZE = {"f32": 4, "bf16": 2, "f16": 2}
_ops = None


def _handle():
    """The program's one operator handle, made at its first use."""
    global _ops
    if _ops is None:
        from ptq_int8_lab_b200.ops import Int8Ops
        _ops = Int8Ops(0)
    return _ops


# ------------------------------------------------------------------------------ cases

def listed():
    cache = dict(type="bf16", dim=128, kv_heads=8, page=64, seqs=1, shortest=1, longest=1, fresh=1)
    att = dict(cache, kind="attention", heads=32)
    lin = dict(kind="linear", type="bf16", out_type="bf16", group=128, gated=False, bias=False, scale_type="f16")
    return [
        # one generated token each of a batch of sequences: launch latency
        dict(cache, kind="write", name="write 32 sequences", seqs=32, shortest=100, longest=4000),
        # a batch of prompts of differing lengths goes into the cache: memory bandwidth
        dict(cache, kind="write", name="write 4 prompts", seqs=4, shortest=2000, longest=8000, fresh=8000),
        # short ragged pieces of prompts, 32-bit states, small pages, an odd number of heads
        dict(cache, kind="write", name="write ragged f32", type="f32", dim=64, kv_heads=5, page=16, seqs=9, shortest=40, longest=500, fresh=301),
        # the last 100 tokens of a few sequences read back (a prefix handed to another server)
        dict(cache, kind="read", name="read 100 tokens", type="f16", page=16, seqs=6, shortest=300, longest=900, fresh=100),
        # a long context read back whole
        dict(cache, kind="read", name="read 32768 tokens", longest=32768, shortest=32768, fresh=32768),
        # one user's generated token over a short context: latency
        dict(att, name="attend 1 token", longest=2000, shortest=2000),
        # a batch of generating sequences whose lengths differ widely: the cache is read once
        dict(att, name="attend batch of 32", seqs=32, shortest=200, longest=8192),
        # one user with a very long context, all heads on one key: the work of few rows split over a long axis
        dict(att, name="attend 131072 tokens", type="f16", kv_heads=2, heads=32, longest=131072, shortest=131072, page=256),
        # pieces of prompts over what is cached, causal
        dict(att, name="attend prompt piece", seqs=2, shortest=4500, longest=8192, fresh=512),
        # a projection for one generated token: the weights are read once
        dict(lin, name="linear w4 1 token", tokens=1, inp=4096, out=4096),
        # first half of an MLP for a batch of 8 generating sequences, small groups
        dict(lin, name="linear w4 8 tokens gated", tokens=8, inp=4096, out=8192, group=64, gated=True),
        # a batch of generating sequences through a ragged projection with bias, kept in 32 bits
        dict(lin, name="linear w4 45 tokens ragged", type="f32", out_type="f32", tokens=45, inp=2000, out=1270, group=32, bias=True, scale_type="f32"),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi):
    """A feature count: a power of two, an odd multiple of 32, or any even number."""
    how, v = rng.random(), _spread(rng, lo, hi)
    if how < 0.4:
        v = 1 << round(math.log2(v))
    elif how < 0.8:
        v = 32 * (v // 64 * 2 + 1)
    else:
        v += v % 2
    return min(max(v, lo), hi)


def draw(rng):
    most = max(max(work(c).values()) for c in listed())
    while True:
        kind = rng.choice(["write", "read", "attention", "attention", "linear", "linear"])
        if kind == "linear":
            return dict(kind=kind, type=rng.choice(["bf16", "bf16", "f16", "f32"]), out_type=rng.choice(["bf16", "bf16", "f16", "f32"]),
                        tokens=_spread(rng, 1, 64), inp=_width(rng, 256, 8192), out=_width(rng, 64, 8192), group=rng.choice([32, 64, 128]),
                        gated=rng.random() < 0.4, bias=rng.random() < 0.3, scale_type=rng.choice(["f16", "bf16", "f32"]))
        case = dict(kind=kind, dim=rng.choice([64, 128, 128, 256]), kv_heads=rng.choice([1, 2, 3, 4, 8, 8, 16]), page=rng.choice([16, 32, 64, 128, 256]),
                    seqs=_spread(rng, 1, 64), longest=_spread(rng, 1, 65536))
        case["shortest"] = max(1, int(case["longest"] * rng.choice([1.0, 0.5, 0.1, 0.02])))
        case["fresh"] = rng.choice([1, 1, _spread(rng, 1, case["longest"])])
        case["type"] = rng.choice(["bf16", "bf16", "f16"] + ([] if kind == "attention" else ["f32"]))
        if kind == "attention":
            case["heads"] = case["kv_heads"] * rng.choice([1, 2, 4, 4, 6, 8, 16])
            # what the plain form holds, in 32-bit values: keys and values as floats, and all scores
            padded = case["seqs"] * case["longest"]
            held = 2 * padded * case["kv_heads"] * case["dim"] + 2 * padded * case["heads"] * min(case["fresh"], case["longest"])
            if held > 3 << 29 or work(case)["flops"] > most:
                continue
        lengths, _ = _lengths(case)
        if max(sum(lengths) * case["kv_heads"] * case["dim"], work(case)["bytes"]) <= 1 << 28:
            return case


def _lengths(case):
    """(lengths, new tokens) of the sequences, in order of their lengths; the new ones are a length at most."""
    n, a, b = case["seqs"], case["shortest"], case["longest"]
    lengths = [int(round(a * (b / a) ** (i / max(1, n - 1)))) if n > 1 else b for i in range(n)]
    return lengths, [min(case["fresh"], v) for v in lengths]


def work(case):
    if case["kind"] == "linear":
        channels = case["out"] * (2 if case["gated"] else 1)
        groups = -(-case["inp"] // case["group"])
        weights = channels * (case["inp"] // 2 + groups * _SIZE[case["scale_type"]] + (4 if case["bias"] else 0))
        return {"bytes": weights + case["tokens"] * (case["inp"] * _SIZE[case["type"]] + case["out"] * _SIZE[case["out_type"]]),
                "flops": 2.0 * case["tokens"] * channels * case["inp"]}
    lengths, fresh = _lengths(case)
    held = 2 * case["kv_heads"] * (case["dim"] // 2 + 4)   # bytes of a token
    rows = sum(fresh)
    if case["kind"] != "attention":
        floats = 2 * case["kv_heads"] * case["dim"] * _SIZE[case["type"]]
        # a written piece is read back too
        return {"bytes": rows * ((held + floats) if case["kind"] == "read" else (2 * held + floats + 2 * case["kv_heads"] * case["dim"] * 4)),
                "flops": rows * 2 * case["kv_heads"] * case["dim"] * 4}
    pairs = sum(n * v - n * (n - 1) // 2 for v, n in zip(lengths, fresh))   # (query, key) pairs that a head sees
    return {"bytes": sum(lengths) * held + 2 * rows * case["heads"] * case["dim"] * _SIZE[case["type"]],
            "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ------------------------------------------------------------------------------ inputs

def _keys(g, rows, heads, dim):
    """Keys: normal, with a few dimensions that are large and off zero in every token."""
    x = torch.randn((rows, heads, dim), generator=g, device="cuda")
    strong = torch.randint(0, dim, (max(1, dim // 32),), generator=g, device="cuda")
    x[..., strong] = x[..., strong] * 2.0 + 3.0
    return x


def _values(g, rows, heads, dim):
    """Values: normal, tokens of differing size."""
    x = torch.randn((rows, heads, dim), generator=g, device="cuda")
    return x * (torch.rand((rows, heads, 1), generator=g, device="cuda") + 0.2)


def _filled(g, case, pages):
    """Codes and (step, least) pairs of `pages` pages of keys, and of values."""
    shape = (pages, case["kv_heads"], case["page"])
    out = []
    for make in (_keys, _values):
        codes = torch.empty((*shape, case["dim"] // 2), dtype=torch.uint8, device="cuda")
        scale = torch.empty((*shape, 2), dtype=torch.bfloat16, device="cuda")
        at = max(1, (1 << 25) // (case["kv_heads"] * case["page"] * case["dim"]))
        for a in range(0, pages, at):
            b = min(pages, a + at)
            rows = (b - a) * case["page"]
            c, s = _quantize_plain(make(g, rows, case["kv_heads"], case["dim"]))
            c = c.view(b - a, case["page"], case["kv_heads"], case["dim"]).transpose(1, 2)
            codes[a:b] = c[..., 0::2] | (c[..., 1::2] << 4)
            scale[a:b] = s.view(b - a, case["page"], case["kv_heads"], 2).transpose(1, 2).to(torch.bfloat16)
        out += [codes, scale]
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = dict(case)
    if case["kind"] == "linear":
        groups = -(-case["inp"] // case["group"])
        channels = case["out"] * (2 if case["gated"] else 1)
        x = torch.randn((case["tokens"], case["inp"]), generator=g, device="cuda")
        x[:, torch.randint(0, case["inp"], (max(1, case["inp"] // 256),), generator=g, device="cuda")] *= 12.0
        s["x"] = (x * (torch.rand((case["tokens"], 1), generator=g, device="cuda") * 2 + 0.1)).to(_DT[case["type"]])
        # rows at multiples of 16 bytes, as weights are laid once
        pitch = (case["inp"] // 2 + 15) // 16 * 16
        s["w"] = torch.zeros((channels, pitch), dtype=torch.uint8, device="cuda")[:, :case["inp"] // 2]
        c = torch.randn((channels, case["inp"]), generator=g, device="cuda", dtype=torch.float16).mul_(2.8).round_().clamp_(-8, 7).to(torch.int8)
        s["w"].copy_((c[:, 0::2] & 15) | ((c[:, 1::2] & 15) << 4))
        s["w_scale"] = (torch.rand((channels, groups), generator=g, device="cuda") * 0.01 + 0.003).to(_DT[case["scale_type"]])
        s["bias"] = torch.randn(channels, generator=g, device="cuda") if case["bias"] else None
        s["y"] = torch.zeros((case["tokens"], case["out"]), dtype=_DT[case["out_type"]], device="cuda")
        return s
    lengths, fresh = _lengths(case)
    order = torch.randperm(case["seqs"], generator=g, device="cuda").tolist()
    lengths, fresh = [lengths[i] for i in order], [fresh[i] for i in order]
    wide = -(-max(lengths) // case["page"])
    need = [-(-n // case["page"]) for n in lengths]
    pages = sum(need) + 3
    # a sequence's pages lie anywhere; behind its last one the table holds what it held before
    names = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.randint(0, pages, (case["seqs"], wide), generator=g, device="cuda").to(torch.int32)
    ends = torch.tensor([0] + need).cumsum(0).tolist()
    for b in range(case["seqs"]):
        table[b, :need[b]] = names[ends[b]:ends[b + 1]]
    s["table"], s["lengths"] = table, torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["rows"], s["most"] = sum(fresh), max(fresh)
    s["starts"] = torch.tensor([0] + fresh).cumsum(0).to(device="cuda", dtype=torch.int32)
    kv = (s["rows"], case["kv_heads"], case["dim"])
    if case["kind"] == "write":
        s["cache"] = [torch.zeros((pages, case["kv_heads"], case["page"], n), dtype=t, device="cuda")
                      for n, t in ((case["dim"] // 2, torch.uint8), (2, torch.bfloat16)) * 2]
        # as a projection leaves them: keys and values of a token beside each other
        both = torch.empty((s["rows"], 2 * case["kv_heads"], case["dim"]), dtype=_DT[case["type"]], device="cuda")
        both[:, :case["kv_heads"]] = _keys(g, *kv)
        both[:, case["kv_heads"]:] = _values(g, *kv)
        s["k"], s["v"] = both[:, :case["kv_heads"]], both[:, case["kv_heads"]:]
        s["out"] = [torch.zeros(kv, device="cuda") for _ in range(2)]
        return s
    s["cache"] = _filled(g, case, pages)
    if case["kind"] == "read":
        s["out"] = [torch.zeros(kv, dtype=_DT[case["type"]], device="cuda") for _ in range(2)]
    else:
        s["q"] = (torch.randn((s["rows"], case["heads"], case["dim"]), generator=g, device="cuda") * 1.3).to(_DT[case["type"]])
        s["out"] = torch.zeros_like(s["q"])
    return s


# ------------------------------------------------------------------------------ the plain forms

def _bf16_down(x):
    """The largest bf16 number that is not above x, as f32; x is finite."""
    b = x.contiguous().view(torch.int32)
    cut = b & -65536
    return torch.where((b < 0) & (cut != b), cut + 65536, cut).view(torch.float32)


def _quantize_plain(x):
    """(codes uint8, (step, least) f32) of rows x: f32 steps as defined, each one rounding."""
    x = x.float()
    low = _bf16_down(x.amin(-1, keepdim=True))
    step = -_bf16_down(-((x.amax(-1, keepdim=True) - low).double() / 15.0).float())
    step = step.clamp_min(2.0 ** -100)
    inverse = (1.0 / step.double()).float()
    codes = ((x - low) * inverse).round().clamp(0, 15).to(torch.uint8)
    return codes, torch.cat((step, low), dim=-1)


def _where(s):
    """(page, place in it, head's index) of the new tokens, to index caches [page, head, place]."""
    rows = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    at = s["lengths"].long()[b] - s["starts"].long()[b + 1] + rows
    page = s["table"].long()[b, at // s["page"]]
    return page[:, None], torch.arange(s["kv_heads"], device="cuda")[None], (at % s["page"])[:, None]


def _stands_for(codes, scale):
    """The values that codes (two per byte) and pairs stand for, f32."""
    c = torch.stack((codes & 15, codes >> 4), dim=-1).reshape(*codes.shape[:-1], 2 * codes.shape[-1]).float()
    return c * scale[..., :1].float() + scale[..., 1:].float()


def _write_plain(s):
    where = _where(s)
    for x, codes, scale in ((s["k"], *s["cache"][:2]), (s["v"], *s["cache"][2:])):
        c, pair = _quantize_plain(x)
        codes[where] = c[..., 0::2] | (c[..., 1::2] << 4)
        scale[where] = pair.to(torch.bfloat16)


def _read_plain(s, dtype):
    where, (k, ks, v, vs) = _where(s), s["cache"]
    return {"k": _stands_for(k[where], ks[where]).to(dtype), "v": _stands_for(v[where], vs[where]).to(dtype)}


def _attend_plain(s):
    n, h, d, most = s["seqs"], s["kv_heads"], s["dim"], s["most"]
    per = s["heads"] // h
    # all sequences padded to the longest: keys and values [seqs, head, position, dim], queries [seqs, head, query x per, dim]
    k, ks, v, vs = (t[s["table"].long()].transpose(1, 2).flatten(2, 3) for t in s["cache"])
    rows = torch.arange(s["rows"], device="cuda")
    b = torch.searchsorted(s["starts"][1:].long(), rows, right=True)
    count = (s["starts"][1:] - s["starts"][:-1]).long()
    place = rows - s["starts"].long()[b]
    q = torch.zeros((n, most, h, per, d), device="cuda")
    q[b, place] = s["q"].float().view(-1, h, per, d)
    q = q.permute(0, 2, 1, 3, 4).reshape(n, h, most * per, d)
    scores = (q @ _stands_for(k, ks).transpose(2, 3)) * (1.0 / math.sqrt(d))
    # query i of a sequence sees the positions up to its own
    last = s["lengths"].long()[:, None] - count[:, None] + torch.arange(most, device="cuda")
    seen = torch.arange(k.shape[2], device="cuda") <= last.repeat_interleave(per, dim=1)[:, :, None]
    scores.masked_fill_(~seen[:, None], -math.inf)
    scores -= scores.amax(-1, keepdim=True)
    scores.exp_()
    scores /= scores.sum(-1, keepdim=True)
    y = scores @ _stands_for(v, vs)
    y = y.view(n, h, most, per, d).permute(0, 2, 1, 3, 4)[b, place]
    return y.reshape(s["q"].shape).to(s["q"].dtype)


def _linear_plain(s):
    c = torch.stack((s["w"] & 15, s["w"] >> 4), dim=-1).reshape(s["w"].shape[0], s["inp"]).float()
    w = torch.where(c >= 8, c - 16, c)
    w *= s["w_scale"].float().repeat_interleave(s["group"], dim=1)[:, :s["inp"]]
    y = s["x"].float() @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["gated"]:
        gate, up = y.chunk(2, dim=1)
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(_DT[s["out_type"]])


def run(state):
    s = state
    if not own:
        if s["kind"] == "linear":
            return {"y": _linear_plain(s)}
        if s["kind"] == "attention":
            return {"y": _attend_plain(s)}
        if s["kind"] == "write":
            _write_plain(s)
            return _read_plain(s, torch.float32)
        return _read_plain(s, _DT[s["type"]])
    ops = _handle()
    if s["kind"] == "linear":
        act = 1 if s["gated"] else 0   # EPI_SWIGLU, EPI_NONE
        return {"y": ops.linear_w4(s["x"], s["w"], s["w_scale"], s["group"], bias=s["bias"], act=act, out=s["y"])}
    starts = s["starts"] if s["most"] > 1 else None   # one new token each needs none
    if s["kind"] == "attention":
        return {"y": ops.cache_attention(s["q"], s["cache"], s["table"], s["lengths"], starts=starts, out=s["out"])}
    if s["kind"] == "write":
        ops.cache_write(s["cache"], s["k"], s["v"], s["table"], s["lengths"], starts=starts)
    k, v = ops.cache_read(s["cache"], s["table"], s["lengths"], starts=starts, out=s["out"])
    return {"k": k, "v": v}


# ------------------------------------------------------------------------------ the definition in 64 bits

def _f64_of(codes, scale):
    out = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device="cuda")
    out[..., 0::2], out[..., 1::2] = torch.remainder(codes.double(), 16), torch.floor(codes.double() / 16)
    return out.mul_(scale[..., :1].double()).add_(scale[..., 1:].double())


def _next_bf16(x, up):
    """The nearest bf16 number, moved on by one where it is on the other side of x."""
    r = x.to(torch.bfloat16)
    to = torch.full_like(r, math.inf if up else -math.inf)
    return torch.where((r.double() < x) if up else (r.double() > x), torch.nextafter(r, to), r)


def _written(x):
    """What a row of a cache stands for once x is written."""
    x = x.double()
    least = _next_bf16(x.min(-1, keepdim=True).values, False).double()
    step = _next_bf16(((x.max(-1, keepdim=True).values - least).float().double() / 15).float().double(), True).double()
    step = torch.clamp_min(step, 2.0 ** -100)
    # the code is defined by 32-bit steps: a difference and a product with 1 / step
    code = torch.round(((x - least).float().double() * (1 / step).float().double()).float().double())
    return least + step * torch.clamp(code, 0, 15)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "linear":
        codes = torch.empty((s["w"].shape[0], s["inp"]), dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = torch.remainder(s["w"].double(), 16), torch.floor(s["w"].double() / 16)
        codes -= 16 * (codes > 7)
        y = torch.zeros((s["tokens"], codes.shape[0]), dtype=torch.float64, device="cuda")
        for i, a in enumerate(range(0, s["inp"], s["group"])):
            b = min(a + s["group"], s["inp"])
            y += (s["x"][:, a:b].double() @ codes[:, a:b].t()) * s["w_scale"][:, i].double()
        if s["bias"] is not None:
            y += s["bias"].double()
        if s["gated"]:
            y = torch.nn.functional.silu(y[:, :s["out"]]) * y[:, s["out"]:]
        return {"y": y}
    if case["kind"] == "write":
        return {"k": _written(s["k"]), "v": _written(s["v"])}
    lengths, starts, table = s["lengths"].tolist(), s["starts"].tolist(), s["table"].long()
    k_out, v_out, y = [], [], []
    for b, n in enumerate(lengths):
        new = starts[b + 1] - starts[b]
        mine = table[b, :-(-n // s["page"])]
        if case["kind"] == "read":
            mine = mine[(n - new) // s["page"]:]
        k, v = (_f64_of(s["cache"][i][mine], s["cache"][i + 1][mine]).transpose(1, 2).flatten(0, 1) for i in (0, 2))
        if case["kind"] == "read":
            first = (n - new) % s["page"]
            k_out.append(k[first:first + new]), v_out.append(v[first:first + new])
            continue
        for h in range(s["kv_heads"]):
            per = s["heads"] // s["kv_heads"]
            q = s["q"][starts[b]:starts[b + 1], h * per:(h + 1) * per].double()
            z = torch.einsum("ipd,jd->pij", q, k[:n, h]) / math.sqrt(s["dim"])
            z = z.masked_fill(torch.ones((new, n), device="cuda").tril(n - new) == 0, -math.inf)
            y.append((b, h, torch.einsum("pij,jd->ipd", torch.softmax(z, dim=-1), v[:n, h])))
    if case["kind"] == "read":
        return {"k": torch.cat(k_out), "v": torch.cat(v_out)}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, h, part in y:
        per = s["heads"] // s["kv_heads"]
        out[starts[b]:starts[b + 1], h * per:(h + 1) * per] = part
    return {"y": out}
