"""Measured cases of the operators for 4-bit weights and expert layers (smelter_amd.ops: mx4_quantize / mx4_dequantize,
mx4_linear, moe_route, expert_linear, moe_combine).

`run` computes a case in plain torch (fp32, rounded once at the end) or, where `own` is set, with the framework's operators.
An MX4 tensor is two byte arrays: `codes` [rows, 16 * ceil(K / 32)] (two e2m1 elements per byte, the even column in the low
nibble; columns behind K hold zero) and `scales` [rows, ceil(K / 32)] (e8m0: 2^(byte - 127); 255 = NaN)."""
import math

import torch

own = False

F16, BF16, F32 = "float16", "bfloat16", "float32"


def listed():
    return [
        # the weights of a 2048 -> 1000 image classifier, packed and read back when a model is loaded
        dict(name="quantize classifier fp16", op="quantize", rows=1000, k=2048, x=F16),
        # the expert weights of one large layer (16 experts of 4096 x 4096), packed when a model is loaded
        dict(name="quantize experts bf16", op="quantize", rows=65536, k=4096, x=BF16),
        # that classifier on one image: the smallest call, latency counts
        dict(name="linear classifier 1 row", op="linear", m=1, n=1000, k=2048, x=F16, bias=True, act="none", gated=False),
        # a gated hidden layer for five tokens that are decoded together: bound by the weights' bytes
        dict(name="linear gated 5 rows bf16", op="linear", m=5, n=8192, k=8192, x=BF16, bias=False, act="none", gated=True),
        # a prompt of odd length through a 16-bit x 4-bit layer
        dict(name="linear 4001 rows bf16", op="linear", m=4001, n=8192, k=4096, x=BF16, bias=True, act="relu", gated=False),
        # a long prompt with both sides in 4 bits, the rows packed in the call: bound by the matrix cores
        dict(name="linear 4 bit 8192 rows", op="linear", m=8192, n=8192, k=8192, x="mx4", bias=False, act="none", gated=False),
        # routing of a decode batch
        dict(name="route 7 tokens", op="route", t=7, e=64, k=6, x=F32, renorm=True),
        # routing of a long prompt; 16-bit scores hold many ties
        dict(name="route 16384 tokens", op="route", t=16384, e=128, k=8, x=BF16, renorm=False),
        # 32 tokens over 64 experts with 4-bit weights: a few rows for each, some experts empty
        dict(name="experts 4 bit decode", op="experts", t=32, top=4, e=64, n=4096, k=2048, x=BF16, w="mx4", gated=True, gather=True),
        # a long prompt over 16 experts with 16-bit weights, ragged groups
        dict(name="experts fp16 prompt", op="experts", t=8191, top=2, e=16, n=4096, k=4096, x=F16, w=F16, gated=False, gather=True),
        # the experts' answers of a long prompt, weighted and added for each token
        dict(name="combine 16384 tokens", op="combine", t=16384, top=8, e=128, n=2048, x=BF16),
        # a whole expert layer for a decode batch: route, gated hidden product, output product, combine
        dict(name="layer decode", op="layer", t=48, top=4, e=32, k=2048, f=1024, x=BF16, w="mx4"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "linear", "linear", "linear", "route", "experts", "experts", "experts", "combine", "layer"])
    t16 = rng.choice([F16, BF16])
    if op == "quantize":
        k = _log(rng, 33, 8192)
        return dict(op=op, rows=_log(rng, 1, min(65536, (1 << 28) // k)), k=k, x=rng.choice([F16, BF16, F32]))
    if op == "linear":
        # inner sizes are multiples of 8 as model widths are, or odd; row counts are anything
        n, k = _log(rng, 64, 8192), _log(rng, 64, 8192)
        if rng.random() < 0.75:
            n, k = -(-n // 8) * 8, -(-k // 8) * 8
        return dict(op=op, m=_log(rng, 1, 8192), n=n, k=k, x=rng.choice([F16, BF16, "mx4"]), bias=rng.random() < 0.5,
                    act=rng.choice(["none", "relu"]), gated=rng.random() < 0.3)
    if op == "route":
        e = rng.randint(4, 256)
        return dict(op=op, t=_log(rng, 1, 16384), e=e, k=rng.randint(1, min(8, e)), x=rng.choice([F16, BF16, F32]), renorm=rng.random() < 0.5)
    if op == "experts":
        e, top = rng.randint(2, 64), rng.randint(1, 2)
        n, k = _log(rng, 64, 4096), _log(rng, 64, 4096)
        if rng.random() < 0.75:
            n, k = -(-n // 8) * 8, -(-k // 8) * 8
        most = max(1, min(8191, (1 << 38) // (n * k * top)))
        return dict(op=op, t=_log(rng, 1, most), top=top, e=e, n=n, k=k, x=t16, w=rng.choice(["mx4", t16]), gated=rng.random() < 0.3, gather=rng.random() < 0.7)
    if op == "combine":
        top = rng.randint(1, 8)
        return dict(op=op, t=_log(rng, 1, 16384), top=top, e=rng.randint(8, 128), n=_log(rng, 64, 2048), x=t16)
    return dict(op=op, t=_log(rng, 1, 256), top=rng.randint(1, 4), e=rng.randint(4, 32), k=8 * _log(rng, 8, 256), f=8 * _log(rng, 8, 128), x=t16, w=rng.choice(["mx4", t16]))


# ---- inputs ----------------------------------------------------------------------------------------------------------------


def _dtype(name):
    return getattr(torch, name)


def _blocks(k):
    return -(-k // 32)


def _pack(w):
    """(codes, scales) of a float tensor [..., K] (the layout of the module's docstring)"""
    k = w.shape[-1]
    v = torch.nn.functional.pad(w.float(), (0, 32 * _blocks(k) - k)).unflatten(-1, (-1, 32))
    amax = v.abs().amax(-1)
    bits = amax.view(torch.int32)
    byte = ((bits >> 23) - 2).clamp_(min=0)                               # floor(log2 amax) - 2, biased by 127
    bad = (bits >> 23) == 255                                             # an infinity or a NaN in the block
    byte = torch.where(bad, torch.full_like(byte, 255), byte)
    a = torch.ldexp(v.abs(), 127 - byte.unsqueeze(-1))
    c = (a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
    c = torch.where(torch.signbit(v), c + 8, c)
    c = torch.where(bad.unsqueeze(-1), torch.zeros_like(c), c).flatten(-2)
    return c[..., 0::2] | (c[..., 1::2] << 4), byte.to(torch.uint8)


def _unpack(codes, scales, k):
    """the fp32 values of an MX4 tensor"""
    table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float32, device=codes.device)
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    s = torch.ldexp(torch.ones((), device=codes.device), scales.int() - 127)
    s = torch.where(scales == 255, torch.full_like(s, float("nan")), s)
    return (table[c.int()].unflatten(-1, (-1, 32)) * s.unsqueeze(-1)).flatten(-2)[..., :k]


def _gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def _rows(g, m, k, t):
    """activations: normal, some channels ten times larger than the others"""
    x = torch.randn((m, k), generator=g, device="cuda")
    loud = torch.rand((k,), generator=g, device="cuda") < 0.01
    return torch.where(loud, x * 10, x).to(t)


def _weights(g, shape):
    return torch.randn(shape, generator=g, device="cuda") * shape[-1] ** -0.5


def _held(w, kind):
    """a weight tensor as a program keeps it"""
    return _pack(w) if kind == "mx4" else (w.to(_dtype(kind)),)


def _assign(seed, t, top, e):
    """a routing of t tokens: distinct experts for each, some experts popular and some never chosen"""
    g = torch.Generator().manual_seed(seed)
    top = min(top, e)
    score = torch.randn((t, e), generator=g) + torch.randn((e,), generator=g)
    experts = score.topk(top, -1).indices
    flat = experts.flatten()
    order = torch.sort(flat, stable=True).indices                          # slot -> assignment
    counts = torch.bincount(flat, minlength=e)
    offsets = torch.zeros(e + 1, dtype=torch.int32)
    offsets[1:] = counts.cumsum(0)
    slots = torch.empty_like(order)
    slots[order] = torch.arange(t * top)
    return dict(offsets=offsets.cuda(), rows=(order // top).int().cuda(), slots=slots.view(t, top).int().cuda(), most=int(counts.max()))


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(c)
    if c["op"] == "quantize":
        s["data"] = (_weights(g, (c["rows"], c["k"]))).to(_dtype(c["x"]))
    elif c["op"] == "linear":
        n = 2 * c["n"] if c["gated"] else c["n"]
        s["data"] = _rows(g, c["m"], c["k"], torch.bfloat16 if c["x"] == "mx4" else _dtype(c["x"]))
        s["weight"] = _held(_weights(g, (n, c["k"])), "mx4")
        s["shift"] = torch.randn((n,), generator=g, device="cuda") if c["bias"] else None
    elif c["op"] == "route":
        s["data"] = (torch.randn((c["t"], c["e"]), generator=g, device="cuda") + torch.randn((c["e"],), generator=g, device="cuda")).to(_dtype(c["x"]))
    elif c["op"] == "experts":
        s["plan"] = _assign(seed, c["t"], c["top"], c["e"])
        m = s["plan"]["rows"].numel()
        n = 2 * c["n"] if c["gated"] else c["n"]
        s["data"] = _rows(g, c["t"] if c["gather"] else m, c["k"], _dtype(c["x"]))
        s["weight"] = _held(_weights(g, (c["e"], n, c["k"])), c["w"])
    elif c["op"] == "combine":
        s["plan"] = _assign(seed, c["t"], c["top"], c["e"])
        s["data"] = _rows(g, s["plan"]["rows"].numel(), c["n"], _dtype(c["x"]))
        s["part"] = torch.softmax(torch.randn(s["plan"]["slots"].shape, generator=g, device="cuda"), -1)
    else:
        s["top"] = min(c["top"], c["e"])
        s["data"] = _rows(g, c["t"], c["k"], _dtype(c["x"]))
        s["score"] = torch.randn((c["t"], c["e"]), generator=g, device="cuda")
        s["hidden"] = _held(_weights(g, (c["e"], 2 * c["f"], c["k"])), c["w"])
        s["answer"] = _held(_weights(g, (c["e"], c["k"], c["f"])), c["w"])
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------


def _float(held, k):
    return _unpack(*held, k) if len(held) == 2 else held[0].float()


def _after(y, act, gated):
    """activation or gate of a product's last axis: the first half of the columns gates the second"""
    if gated:
        a, b = y.chunk(2, -1)
        return a / (1 + torch.exp(-a)) * b
    return torch.where(y < 0, torch.zeros_like(y), y) if act == "relu" else y


def _plain_route(score, k, renorm):
    """top-k (ties: the lowest index), softmax weights and the order by expert"""
    t, e = score.shape
    z = score.float()
    index = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    p = torch.exp(z - z.amax(-1, keepdim=True))
    chosen = p.gather(1, index)
    weights = chosen / (chosen if renorm else p).sum(-1, keepdim=True)
    flat = index.flatten()
    order = torch.sort(flat, stable=True).indices
    slots = torch.empty_like(order)
    slots[order] = torch.arange(order.numel(), device=order.device)
    offsets = torch.searchsorted(flat[order], torch.arange(e + 1, device=order.device))
    return dict(weights=weights, experts=index.int(), offsets=offsets.int(), rows=(order // k).int(), slots=slots.view(t, k).int())


def _plain_experts(x, w, offsets, most, gated):
    """products of the groups, each padded to the largest group's rows"""
    e = w.shape[0]
    at = offsets[:-1, None].long() + torch.arange(most, device=x.device)
    held = at < offsets[1:, None]
    y = torch.bmm(x.float()[torch.where(held, at, torch.zeros_like(at))], w.transpose(1, 2).contiguous())
    return _after(y, "none", gated)[held]


def _plain(s):
    if s["op"] == "quantize":
        x = s["data"]
        return _unpack(*_pack(x), x.shape[-1]).to(x.dtype)
    if s["op"] == "linear":
        x = s["data"]
        v = _unpack(*_pack(x), s["k"]) if s["x"] == "mx4" else x.float()
        y = v @ _float(s["weight"], s["k"]).t()
        return _after(y if s["shift"] is None else y + s["shift"], s["act"], s["gated"]).to(x.dtype)
    if s["op"] == "route":
        return _plain_route(s["data"], s["k"], s["renorm"])
    if s["op"] == "experts":
        x, plan = s["data"], s["plan"]
        v = x[plan["rows"]] if s["gather"] else x
        return _plain_experts(v, _float(s["weight"], s["k"]), plan["offsets"], plan["most"], s["gated"]).to(x.dtype)
    if s["op"] == "combine":
        y = s["data"].float()[s["plan"]["slots"]]
        return (y * s["part"].unsqueeze(-1)).sum(1).to(s["data"].dtype)
    # the layer: every token through every expert, weighted with zero where the expert is not chosen
    r = _plain_route(s["score"], s["top"], True)
    part = torch.zeros_like(s["score"]).scatter_(1, r["experts"].long(), r["weights"])
    x, e, f = s["data"].float(), s["e"], s["f"]
    h = _after((x @ _float(s["hidden"], s["k"]).flatten(0, 1).t()).unflatten(1, (e, 2 * f)), "none", True)
    return ((h * part.unsqueeze(-1)).flatten(1) @ _float(s["answer"], f).transpose(1, 2).flatten(0, 1)).to(s["data"].dtype)


# ---- the framework's operators -----------------------------------------------------------------------------------------------


def _own_weight(ops, held, k):
    return ops.Mx4(held[0], held[1], k) if len(held) == 2 else held[0]


def _own(s):
    from smelter_amd import ops

    if s["op"] == "quantize":
        return ops.mx4_dequantize(ops.mx4_quantize(s["data"]), s["data"].dtype)
    if s["op"] == "linear":
        x = ops.mx4_quantize(s["data"]) if s["x"] == "mx4" else s["data"]
        act = ops.ACT_RELU if s["act"] == "relu" and not s["gated"] else ops.ACT_NONE
        return ops.mx4_linear(x, _own_weight(ops, s["weight"], s["k"]), s["shift"], act=act, gated=s["gated"], dtype=s["data"].dtype)
    if s["op"] == "route":
        r = ops.moe_route(s["data"], s["k"], renormalize=s["renorm"])
        return dict(weights=r.weights, experts=r.experts, offsets=r.offsets, rows=r.rows, slots=r.slots)
    if s["op"] == "experts":
        plan = s["plan"]
        return ops.expert_linear(s["data"], _own_weight(ops, s["weight"], s["k"]), plan["offsets"], rows=plan["rows"] if s["gather"] else None, gated=s["gated"])
    if s["op"] == "combine":
        return ops.moe_combine(s["data"], s["plan"]["slots"], s["part"])
    r = ops.moe_route(s["score"], s["top"])
    # fp32 between the products: rounded like the answer, the hidden values would double what it is off by, and a product of two unbounded values fits no 16-bit type with more bits than bf16
    h = ops.expert_linear(s["data"], _own_weight(ops, s["hidden"], s["k"]), r.offsets, rows=r.rows, gated=True, dtype=torch.float32)
    y = ops.expert_linear(h, _own_weight(ops, s["answer"], s["f"]), r.offsets, dtype=torch.float32)
    return ops.moe_combine(y, r.slots, r.weights, dtype=s["data"].dtype)


def run(state):
    return _own(state) if own else _plain(state)


# ---- work and the answers in 64 bits -----------------------------------------------------------------------------------------

_SIZE = {F16: 2, BF16: 2, F32: 4, "mx4": 0.5 + 1 / 32}


def work(case):
    c = case
    if c["op"] == "quantize":                                             # read, pack, read the packed form back, write the values
        n = c["rows"] * c["k"]
        return dict(bytes=n * (2 * _SIZE[c["x"]] + 2 * _SIZE["mx4"]), flops=4 * n)
    if c["op"] == "linear":
        n = c["n"] * (2 if c["gated"] else 1)
        return dict(bytes=c["m"] * c["k"] * 2 + n * c["k"] * _SIZE["mx4"] + c["m"] * c["n"] * 2, flops=2 * c["m"] * n * c["k"])
    if c["op"] == "route":
        return dict(bytes=c["t"] * c["e"] * _SIZE[c["x"]] + c["t"] * c["k"] * 16 + 4 * c["e"], flops=c["t"] * c["e"] * 4)
    m = c["t"] * min(c["top"], c["e"])
    used = min(c["e"], m)
    if c["op"] == "experts":
        n = c["n"] * (2 if c["gated"] else 1)
        x = (c["t"] if c["gather"] else m) * c["k"] * 2
        return dict(bytes=x + used * n * c["k"] * _SIZE[c["w"]] + m * c["n"] * 2, flops=2 * m * n * c["k"])
    if c["op"] == "combine":
        return dict(bytes=m * c["n"] * 2 + m * 8 + c["t"] * c["n"] * 2, flops=2 * m * c["n"])
    return dict(bytes=2 * c["t"] * c["k"] * 2 + c["t"] * c["e"] * 4 + used * 3 * c["f"] * c["k"] * _SIZE[c["w"]], flops=6 * m * c["f"] * c["k"])


def _exact_mx4(v):
    """the values that MX4 stands for, in 64 bits: scale 2^(floor(log2 amax) - 2), elements rounded to the nearest of the e2m1 grid, ties to even"""
    k = v.shape[-1]
    b = torch.nn.functional.pad(v.double(), (0, -k % 32)).unflatten(-1, (-1, 32))
    top = torch.frexp(b.abs().amax(-1, keepdim=True)).exponent - 1        # amax in [2^top, 2^(top + 1))
    scale = torch.exp2((top - 2).clamp(min=-127).double())
    q = b / scale
    step = torch.exp2((torch.frexp(q).exponent - 2).clamp(0 - 1, 1).double())
    q = (torch.round(q / step) * step).clamp(-6, 6)
    return (q * scale).flatten(-2)[..., :k]


def _exact_held(held, k):
    if len(held) == 1:
        return held[0].double()
    code = torch.empty(held[0].shape[:-1] + (2 * held[0].shape[-1],), dtype=torch.int64, device=held[0].device)
    code[..., 0::2], code[..., 1::2] = held[0] % 16, held[0] // 16
    mag, ex, man = code % 8, code % 8 // 2, code % 2
    v = torch.where(ex == 0, 0.5 * man, (1 + 0.5 * man) * torch.exp2((ex - 1).double()))
    v = torch.where(code >= 8, -v, v) * torch.exp2(held[1].double() - 127).repeat_interleave(32, -1)
    return v[..., :k]


def _exact_gate(y):
    n = y.shape[-1] // 2
    return y[..., :n] * torch.sigmoid(y[..., :n]) * y[..., n:]


def _exact_route(score, k, renorm):
    z = score.double().cpu()
    t, e = z.shape
    # one key per (token, expert): the rank of the score, ties by index
    index = torch.argsort(-z, dim=-1, stable=True)[:, :k]
    p = torch.softmax(z, -1)
    w = p.gather(1, index)
    if renorm:
        w = w / w.sum(-1, keepdim=True)
    groups = [[] for _ in range(e)]
    for a, x in enumerate(index.flatten().tolist()):
        groups[x].append(a)
    order = [a for v in groups for a in v]
    offsets = [0]
    for v in groups:
        offsets.append(offsets[-1] + len(v))
    slots = [0] * len(order)
    for i, a in enumerate(order):
        slots[a] = i
    return dict(weights=w, experts=index.int(), offsets=torch.tensor(offsets, dtype=torch.int32), rows=torch.tensor([a // k for a in order], dtype=torch.int32),
                slots=torch.tensor(slots, dtype=torch.int32).view(t, k))


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] == "quantize":
        return _exact_mx4(s["data"])
    if s["op"] == "linear":
        x = _exact_mx4(s["data"]) if s["x"] == "mx4" else s["data"].double()
        y = x @ _exact_held(s["weight"], s["k"]).t()
        if s["shift"] is not None:
            y = y + s["shift"].double()
        return _exact_gate(y) if s["gated"] else y.clamp(min=0) if s["act"] == "relu" else y
    if s["op"] == "route":
        return _exact_route(s["data"], s["k"], s["renorm"])
    if s["op"] == "combine":
        y, at, part = s["data"].double(), s["plan"]["slots"].long(), s["part"].double()
        out = torch.zeros((s["t"], s["n"]), dtype=torch.float64, device="cuda")
        for j in range(at.shape[1]):
            out += part[:, j, None] * y[at[:, j]]
        return out
    if s["op"] == "experts":
        plan = s["plan"]
        edge = plan["offsets"].tolist()
        out = []
        for i in range(s["e"]):
            at = torch.arange(edge[i], edge[i + 1], device="cuda")
            x = s["data"][plan["rows"][at].long() if s["gather"] else at].double()
            y = x @ _exact_held([h[i] for h in s["weight"]], s["k"]).t()
            out.append(_exact_gate(y) if s["gated"] else y)
        return torch.cat(out)
    r = _exact_route(s["score"], s["top"], True)
    out = torch.zeros((s["t"], s["k"]), dtype=torch.float64, device="cuda")
    part = r["weights"].cuda()
    chosen = r["experts"].cuda()
    for i in range(s["e"]):
        tok, j = (chosen == i).nonzero(as_tuple=True)
        h = _exact_gate(s["data"][tok].double() @ _exact_held([v[i] for v in s["hidden"]], s["k"]).t())
        out[tok] += part[tok, j, None] * (h @ _exact_held([v[i] for v in s["answer"]], s["f"]).t())
    return out
