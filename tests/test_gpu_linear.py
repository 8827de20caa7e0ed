"""4-bit (MX4) tensors, linear layers on them, expert layers and their routing, against plain 64-bit forms (tests/mx4ref.py)."""
import pytest
import torch

import mx4ref
from smelter_amd import _native as N
from smelter_amd import ops

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, scale=1.0):
    return torch.randn(shape, generator=g) * scale


def mx4(w):
    c, s = mx4ref.pack(w)
    return ops.Mx4(c.cuda(), s.cuda(), w.shape[-1])


def val(q):
    return mx4ref.unpack(q.codes, q.scales, q.k)


# ---- packing ------------------------------------------------------------------------------------------------------------------------------


def same_pack(x):
    q = ops.mx4_quantize(x.cuda())
    c, s = mx4ref.pack(x)
    assert torch.equal(q.scales.cpu(), s) and torch.equal(q.codes.cpu(), c) and q.k == x.shape[-1] and q.shape == tuple(x.shape)
    return q


@pytest.mark.parametrize("t", [F16, BF16, F32])
@pytest.mark.parametrize("rows, k", [(1, 1), (1, 31), (3, 32), (2, 33), (5, 100), (1, 2048), (257, 72), (0, 64), (4, 0)])
def test_quantize_sizes(t, rows, k):
    same_pack(randn(gen(rows + k), rows, k).to(t))


@pytest.mark.parametrize("t", [F16, BF16])
def test_quantize_every_pattern(t):
    """every 16-bit pattern once as the largest of its block (beside smaller ones), and among neighbours in value"""
    x = torch.arange(-32768, 32768, dtype=torch.int32).to(torch.int16).view(t)
    same_pack(x.view(-1, 32))
    fine = x[torch.isfinite(x.float())]
    f = fine.double()
    block = torch.stack([(f * m).to(t) for m in (1, 0.5, -0.25, 0.3125, 0.4375, -0.625, 0.875, 0.03125)], 1)
    same_pack(torch.where(torch.isfinite(block.float()), block, torch.zeros_like(block)))


def test_quantize_fp32_extremes():
    x = torch.tensor([[0.0, -0.0, 1e-45, -1e-45], [1e-38, 1.1754944e-38, -5e-39, 3e-39], [3.4028235e38, -3.4028235e38, 1e30, 2.0], [INF, 1, 2, 3], [-INF, 0, 0, 0], [NAN, INF, 1, 0], [6.0, 5.0, 3.5, 2.5]])
    same_pack(x)


@pytest.mark.parametrize("t", [F16, F32])
def test_quantize_strides_and_leading_axes(t):
    big = randn(gen(3), 6, 4, 130).to(t)
    same_pack(big)
    g = big.cuda()
    for v in (g[..., :70], g[:, 1], g[..., 3:40], g[:2, :1, 5:6]):
        q = ops.mx4_quantize(v)
        c, s = mx4ref.pack(v.cpu())
        assert torch.equal(q.codes.cpu(), c) and torch.equal(q.scales.cpu(), s)
    with pytest.raises(N.SmelterError):
        ops.mx4_quantize(g.transpose(0, 2))


@pytest.mark.parametrize("t", [F16, BF16, F32])
@pytest.mark.parametrize("rows, k", [(1, 1), (3, 33), (9, 70), (2, 256), (300, 40)])
def test_dequantize(t, rows, k):
    """exact: every value of these scales is representable in all three types"""
    g = gen(k)
    q = mx4(randn(g, rows, k))
    assert torch.equal(ops.mx4_dequantize(q, t).cpu().double(), val(q))
    wide = torch.full((rows, k + 9), 7.0, dtype=t, device="cuda")
    ops.mx4_dequantize(q, out=wide[:, 1:k + 1])
    assert torch.equal(wide[:, 1:k + 1].cpu().double(), val(q)) and wide[:, 0].eq(7).all() and wide[:, k + 1:].eq(7).all()


@pytest.mark.parametrize("t", [F16, BF16, F32])
def test_dequantize_every_scale(t):
    codes = torch.arange(256, dtype=torch.uint8).view(1, 16, 16).repeat(256, 1, 1).reshape(256, 256)
    scales = torch.arange(256).to(torch.uint8).view(256, 1).repeat(1, 16)
    got = ops.mx4_dequantize(ops.Mx4(codes.cuda(), scales.cuda(), 512), t).cpu()
    want = mx4ref.unpack(codes, scales, 512).to(t)                      # one rounding: to nearest even, to an infinity above the range
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[:255], want[:255])


# ---- products -----------------------------------------------------------------------------------------------------------------------------

KINDS = ["f16", "bf16", "f16-mx4", "bf16-mx4", "mx4-mx4"]


def operands(kind, g, t, k, wshape, spread=False):
    """(x as handed over, its fp64 values, w as handed over, its fp64 values, type of the output)"""
    dt = BF16 if kind.startswith("bf16") else F16
    x = randn(g, t, k).to(dt)
    w = randn(g, *wshape, scale=max(k, 1) ** -0.5)
    if kind == "mx4-mx4":
        qx, qw = mx4(x), mx4(w)
        return qx, val(qx), qw, val(qw), dt
    if kind.endswith("mx4"):
        qw = mx4(w)
        return x.cuda(), x.double(), qw, val(qw), dt
    w = w.to(dt)
    return x.cuda(), x.double(), w.cuda(), w.double(), dt


@pytest.mark.parametrize("kind", ["f16-mx4", "bf16-mx4", "mx4-mx4"])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 33, 64, 65, 129, 260, 530])
@pytest.mark.parametrize("n, k", [(1, 1), (33, 40), (100, 129), (256, 512), (72, 1000), (300, 2088)])
def test_mx4_linear(kind, m, n, k):
    g = gen(m * 1000 + n + k)
    x, xv, w, wv, dt = operands(kind, g, m, k, (n, k))
    bias = randn(g, n)
    want, err = mx4ref.linear(xv, wv, bias)
    mx4ref.close(ops.mx4_linear(x, w, bias.cuda(), dtype=dt), want, err)
    mx4ref.close(ops.mx4_linear(x, w, dtype=F32), *mx4ref.linear(xv, wv))


@pytest.mark.parametrize("kind", ["f16-mx4", "bf16-mx4", "mx4-mx4"])
@pytest.mark.parametrize("m, n, k", [(1, 1, 32), (3, 17, 64), (70, 40, 100), (150, 128, 256), (300, 264, 328)])
def test_mx4_linear_gated(kind, m, n, k):
    g = gen(m + n + k)
    x, xv, w, wv, dt = operands(kind, g, m, k, (2 * n, k))
    bias = randn(g, 2 * n)
    mx4ref.close(ops.mx4_linear(x, w, bias.cuda(), gated=True, dtype=dt), *mx4ref.linear(xv, wv, bias, gated=True))


@pytest.mark.parametrize("act, slope, f", [(ops.ACT_RELU, 0.0, lambda z: z.clamp(min=0)), (ops.ACT_PRELU, 0.25, lambda z: torch.where(z < 0, 0.25 * z, z)),
                                           (ops.ACT_CLIP, 0.5, lambda z: z.clamp(0, 0.5)), (ops.ACT_CODES["sigmoid"], 0.0, torch.sigmoid)])
@pytest.mark.parametrize("m", [3, 200])
def test_mx4_linear_activations(act, slope, f, m):
    """all four have slopes of at most 1 and are computed in fp32 with a relative error below 2^-20 of values of at most 1 (sigmoid), or exactly"""
    x, xv, w, wv, dt = operands("f16-mx4", gen(m), m, 96, (136, 96))
    want, err = mx4ref.linear(xv, wv, act=f)
    mx4ref.close(ops.mx4_linear(x, w, act=act, slope=slope), want, err + 2.0 ** -20)


@pytest.mark.parametrize("kind", ["f16-mx4", "bf16-mx4"])
@pytest.mark.parametrize("m", [4, 200])
def test_mx4_linear_wide_scales(kind, m):
    """block scales over 2^60 of each other, rows of tiny weights, a row of zeros, one NaN block"""
    g = gen(5)
    k = 640
    w = randn(g, 70, k)
    w = w * torch.exp2(torch.randint(-30, 30, (70, k // 32), generator=g).float()).repeat_interleave(32, 1)
    w[1] *= 2.0 ** -60
    w[2] = 0
    w[3] = randn(g, k) * 2.0 ** -100
    w[4, 33] = NAN
    q = mx4(w)
    x = randn(g, m, k).to(F16 if kind == "f16-mx4" else BF16)
    got = ops.mx4_linear(x.cuda(), q, dtype=F32).cpu()
    mx4ref.close(got, *mx4ref.linear(x, val(q)))
    assert got[:, 4].isnan().all() and got[:, 2].eq(0).all() and got[:, 3].ne(0).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m", [5, 150])
def test_memory_beside_the_operands(kind, m):
    """NaN behind every row of x, an output with a stride and neighbours that stay, an x that is aligned to its element only"""
    g = gen(m)
    n, k = 45, 88
    x, xv, w, wv, dt = operands(kind, g, m, k, (1, n, k))
    if kind != "mx4-mx4":
        wide = torch.full((m, k + 13), NAN, dtype=dt, device="cuda")
        wide[:, 3:k + 3] = x
        x = wide[:, 3:k + 3]
    out = torch.full((m + 2, n + 7), 7.0, dtype=dt, device="cuda")
    off = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    ops.expert_linear(x, w, off, out=out[1:m + 1, 2:n + 2])
    mx4ref.close(out[1:m + 1, 2:n + 2], *mx4ref.linear(xv, wv[0]))
    out[1:m + 1, 2:n + 2] = 7
    assert out.eq(7).all()


def grouped(xv, wv, offsets, rows, bias=None, gated=False, m=None):
    m = len(rows) if rows is not None else xv.shape[0]
    n = wv.shape[1] // (2 if gated else 1)
    want, err = torch.full((m, n), 7.0, dtype=torch.float64), torch.zeros(m, n, dtype=torch.float64)
    for e in range(len(offsets) - 1):
        s = torch.arange(offsets[e], offsets[e + 1])
        at = torch.as_tensor(rows)[s].long() if rows is not None else s
        ok = (at >= 0) & (at < xv.shape[0])
        x = torch.where(ok[:, None], xv[at.clamp(0, max(xv.shape[0] - 1, 0))], torch.zeros(1, dtype=torch.float64))
        want[s], err[s] = mx4ref.linear(x, wv[e], None if bias is None else bias[e], gated=gated)
    return want, err


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes, n, k, gather", [([1], 24, 32, False), ([0, 3, 0, 1, 17, 0], 40, 64, True), ([5] * 70 + [0, 16, 40], 19, 96, True), ([130, 0, 1, 300, 64], 136, 136, True),
                                                 ([0, 0], 8, 32, False), ([257, 255, 256, 1], 264, 200, False), ([33, 31, 700], 64, 77, True)])
def test_expert_linear(kind, gated, sizes, n, k, gather):
    g = gen(sum(sizes) + n + k + gated)
    m, e = sum(sizes), len(sizes)
    t = m // 2 + 1 if gather else m
    x, xv, w, wv, dt = operands(kind, g, t, k, (e, 2 * n if gated else n, k))
    off = torch.tensor([0] + sizes).cumsum(0).tolist()
    rows = torch.randint(0, t, (m,), generator=g).tolist() if gather else None
    bias = randn(g, e, 2 * n if gated else n)
    out = torch.full((m + 3, n), 7.0, dtype=dt, device="cuda")
    if gather:                                                         # slots behind the last group stay as they were
        got = ops.expert_linear(x, w, torch.tensor(off, dtype=torch.int32, device="cuda"), torch.tensor(rows + [0, -1, t], dtype=torch.int32, device="cuda"), bias.cuda(), gated=gated, out=out)
        assert got is out and out[m:].eq(7).all()
        got = out[:m]
    else:
        got = ops.expert_linear(x, w, torch.tensor(off, dtype=torch.int32, device="cuda"), bias=bias.cuda(), gated=gated)
    want, err = grouped(xv, wv, off, rows, bias, gated)
    mx4ref.close(got, want, err)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("scale", [1, 40])
def test_expert_linear_odd_lists(kind, scale):
    """the same row for many slots; indices outside x (rows of zeros); slots before the first and behind the last group; offsets outside the slots are clamped"""
    g = gen(9)
    x, xv, w, wv, dt = operands(kind, g, 6, 72, (3, 56, 72))
    rows = [0, 0, 0, 5, -1, 6, 3, 3, 1 << 30, -(1 << 31), 2, 2] * scale
    m = len(rows)
    r = torch.tensor(rows, dtype=torch.int32, device="cuda")
    a, b = 2 * scale, 7 * scale
    off = [a, a, b, m - 1]
    out = torch.full((m, 56), 7.0, dtype=dt, device="cuda")
    ops.expert_linear(x, w, torch.tensor(off, dtype=torch.int32, device="cuda"), r, out=out)
    mx4ref.close(out, *grouped(xv, wv, off, rows))
    assert out[:a].eq(7).all() and out[m - 1].eq(7).all()
    out.fill_(7)
    ops.expert_linear(x, w, torch.tensor([-5, a, b, m + 1000], dtype=torch.int32, device="cuda"), r, out=out)
    mx4ref.close(out, *grouped(xv, wv, [0, a, b, m], rows))


@pytest.mark.parametrize("kind", KINDS)
def test_expert_linear_of_nothing(kind):
    x, xv, w, wv, dt = operands(kind, gen(1), 0, 64, (2, 24, 64))
    off = torch.zeros(3, dtype=torch.int32, device="cuda")
    assert ops.expert_linear(x, w, off).shape == (0, 24)
    bias = torch.ones(2, 24, device="cuda")
    got = ops.expert_linear(x, w, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), bias)
    assert got.eq(1).all()                                             # no row of x at all: rows of zeros
    x, xv, w, wv, dt = operands(kind, gen(1), 2, 0, (2, 24, 0))
    assert ops.expert_linear(x, w, torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda"), None, bias).eq(1).all()


@pytest.mark.parametrize("m", [3, 200])
def test_linear_infinities_and_nan(m):
    """a NaN or an infinity of x reaches its own row only"""
    x, xv, w, wv, dt = operands("f16-mx4", gen(2), m, 96, (40, 96))
    bad = x.clone()
    bad[1, 5], bad[2, 95] = NAN, INF
    got, fine = ops.mx4_linear(bad, w), ops.mx4_linear(x, w)
    keep = [i for i in range(m) if i not in (1, 2)]
    assert torch.equal(got[keep], fine[keep]) and got[1].isnan().all() and (~torch.isfinite(got[2])).all()


def test_python_refusals():
    x, xv, w, wv, dt = operands("f16-mx4", gen(2), 4, 64, (8, 64))
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    w3 = ops.Mx4(w.codes[None], w.scales[None], 64)
    for f in (lambda: ops.mx4_linear(x[:, :32], w), lambda: ops.mx4_linear(x.double(), w), lambda: ops.mx4_linear(x, w3), lambda: ops.mx4_linear(x, w, torch.zeros(7, device="cuda")),
              lambda: ops.mx4_linear(x, w, torch.zeros(8, device="cuda", dtype=F16)), lambda: ops.mx4_linear(x, w, dtype=BF16), lambda: ops.mx4_linear(x, w, out=torch.empty(4, 9, device="cuda", dtype=F16)),
              lambda: ops.mx4_linear(x, ops.Mx4(w.codes, w.scales, 40)), lambda: ops.mx4_linear(x, ops.Mx4(w.codes[:, ::2], w.scales, 64)), lambda: ops.mx4_linear(x, w, act=99),
              lambda: ops.expert_linear(x, w3, off.long()), lambda: ops.expert_linear(x, w3, off[:1]), lambda: ops.expert_linear(x, w3, off, torch.zeros(4, device="cuda")),
              lambda: ops.expert_linear(x, torch.zeros(1, 8, 64, device="cuda", dtype=BF16), off), lambda: ops.expert_linear(x, torch.zeros(1, 64, 8, device="cuda", dtype=F16).transpose(1, 2), off),
              lambda: ops.expert_linear(x, ops.Mx4(w.codes[None, :7], w.scales[None, :7], 64), off, gated=True), lambda: ops.moe_route(x, 65), lambda: ops.moe_route(x, 0),
              lambda: ops.moe_combine(x, off.view(1, 2), torch.zeros(1, 3, device="cuda")), lambda: ops.moe_combine(x.double(), off.view(1, 2), torch.zeros(1, 2, device="cuda")),
              lambda: ops.moe_combine(x, off.view(1, 2), torch.zeros(1, 2, device="cuda"), dtype=torch.int32)):
        with pytest.raises(N.SmelterError) as e:
            f()
        assert e.value.kind == "invalidArgument"


# ---- routing ------------------------------------------------------------------------------------------------------------------------------


def same_route(scores, k, renorm):
    got = ops.moe_route(scores.cuda() if not scores.is_cuda else scores, k, renormalize=renorm)
    want = mx4ref.route(scores.cpu(), k, renorm)
    for name in ("experts", "offsets", "rows", "slots"):
        assert torch.equal(getattr(got, name).cpu(), want[name]), name
    # one exponential (within 2 ulp), a sum of E of them in a tree or a chain, a division
    e = scores.shape[1]
    assert ((got.weights.cpu().double() - want["weights"]).abs() <= (e + 8) * 2.0 ** -24 * want["weights"] + 2.0 ** -126).all()
    return got


@pytest.mark.parametrize("t", [F32, F16, BF16])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("tokens, e, k", [(0, 4, 2), (1, 1, 1), (1, 8, 8), (7, 64, 6), (63, 65, 3), (64, 128, 32), (65, 60, 4), (130, 256, 8), (1000, 5, 2), (700, 1000, 8)])
def test_route(t, renorm, tokens, e, k):
    g = gen(tokens + e + k)
    same_route((randn(g, tokens, e) + 2 * randn(g, e)).to(t), k, renorm)


@pytest.mark.parametrize("tokens", [40, 300])
@pytest.mark.parametrize("renorm", [True, False])
def test_route_masks_and_ties(tokens, renorm):
    g = gen(tokens)
    z = torch.randint(-2, 3, (tokens, 70), generator=g).float()         # ties everywhere
    z[z == 0] *= torch.where(torch.rand(int((z == 0).sum()), generator=g) < 0.5, -1.0, 1.0)   # zeros of either sign are equal
    z[3] = -INF                                                         # nothing left
    z[4] = NAN
    z[5, 2:] = -INF                                                     # fewer than k left
    z[6, 1:] = NAN
    z[7] = torch.finfo(F32).min                                         # the lowest value is a score like any other
    z[8, 5] = INF
    z[9, [3, 60]] = INF
    z[10, ::2] = -INF
    z[11] = torch.finfo(F32).max
    z[12, 0], z[12, 1:] = torch.finfo(F32).max, torch.finfo(F32).min
    z[20:30] = -INF                                                     # padding
    same_route(z, 6, renorm)


def test_route_strided_and_many_tokens():
    g = gen(1)
    z = randn(g, 5000, 40).cuda()
    same_route(z[:, 3:20], 3, True)
    same_route(z[::7, :16], 3, False)
    same_route(torch.zeros(3000, 64), 2, True)                          # everything to two experts


@pytest.mark.parametrize("t", [F16, BF16, F32])
@pytest.mark.parametrize("tokens, k, n", [(1, 1, 1), (7, 6, 40), (50, 8, 131), (300, 2, 264), (3, 0, 8)])
def test_combine(t, tokens, k, n):
    g = gen(tokens + n)
    m = max(1, tokens * k)
    y, w = randn(g, m, n).to(t), torch.rand(tokens, k, generator=g)
    slots = torch.randint(-1, m + 1, (tokens, k), generator=g).int()    # nothing, repeated ones, one outside
    ok = ((slots >= 0) & (slots < m)).double() * w.double()
    rows = y.double()[slots.clamp(0, m - 1).long()]
    want, mag = (rows * ok[..., None]).sum(1), (rows.abs() * ok[..., None]).sum(1)
    mx4ref.close(ops.moe_combine(y.cuda(), slots.cuda(), w.cuda()), want, (k + 1) * 2.0 ** -23 * mag)
    for d in (F16, BF16, F32):
        mx4ref.close(ops.moe_combine(y.cuda(), slots.cuda(), w.cuda(), dtype=d), want, (k + 1) * 2.0 ** -23 * mag)
    wide = torch.full((tokens, n + 5), 7.0, dtype=t, device="cuda")
    yw = torch.full((m, n + 3), NAN, dtype=t, device="cuda")
    yw[:, 1:n + 1] = y.cuda()
    ops.moe_combine(yw[:, 1:n + 1], slots.cuda(), w.cuda(), out=wide[:, 2:n + 2])
    mx4ref.close(wide[:, 2:n + 2], want, (k + 1) * 2.0 ** -23 * mag)
    assert wide[:, :2].eq(7).all() and wide[:, n + 2:].eq(7).all()


# ---- together -----------------------------------------------------------------------------------------------------------------------------


def layer(x, scores, hidden, answer, k):
    r = ops.moe_route(scores, k)
    h = ops.expert_linear(x, hidden, r.offsets, rows=r.rows, gated=True)
    return ops.moe_combine(ops.expert_linear(h, answer, r.offsets), r.slots, r.weights)


def layer_case(seed, tokens, kind, e=6, k=2, d=64, f=96):
    g = gen(seed)
    dt = BF16 if kind.startswith("bf16") else F16
    x = randn(g, tokens, d).to(dt)
    z = randn(g, tokens, e)
    hidden, answer = randn(g, e, 2 * f, d, scale=d ** -0.5), randn(g, e, d, f, scale=f ** -0.5)
    if kind.endswith("mx4"):
        hidden, answer = mx4(hidden), mx4(answer)
        hv, av = val(hidden), val(answer)
    else:
        hidden, answer = hidden.to(dt).cuda(), answer.to(dt).cuda()
        hv, av = hidden.cpu().double(), answer.cpu().double()
    return x, z, hidden, answer, hv, av


def layer_want(x, z, hv, av, k):
    r = mx4ref.route(z, k, True)
    want, err = torch.zeros(x.shape[0], av.shape[1], dtype=torch.float64), torch.zeros(x.shape[0], av.shape[1], dtype=torch.float64)
    step = mx4ref.half_step(x.dtype)
    for i in range(x.shape[0]):
        for j in range(k):
            e = int(r["experts"][i, j])
            if e < 0:
                continue
            h, he = mx4ref.linear(x[i:i + 1], hv[e], gated=True)
            he = he + step * (h.abs() + he)                             # the hidden row is rounded once
            y, ye = mx4ref.linear(h, av[e])
            ye = ye * 1.01 + he @ av[e].abs().t()
            ye = ye + step * (y.abs() + ye)                             # and the answer
            w = float(r["weights"][i, j])
            want[i] += w * y[0]
            err[i] += w * (ye[0] + 2.0 ** -20 * y[0].abs())
    return want, err


@pytest.mark.parametrize("kind", ["f16", "bf16", "f16-mx4", "bf16-mx4"])
@pytest.mark.parametrize("tokens", [1, 9, 80, 400])
def test_layer(kind, tokens):
    x, z, hidden, answer, hv, av = layer_case(tokens, tokens, kind)
    mx4ref.close(layer(x.cuda(), z.cuda(), hidden, answer, 2), *layer_want(x, z, hv, av, 2))


@pytest.mark.parametrize("tokens", [40, 200])
def test_layer_padded_batch(tokens):
    """padded tokens (all scores -inf, NaN rows of x) cost no slot, give zeros and touch nobody else"""
    x, z, hidden, answer, hv, av = layer_case(7, tokens, "bf16-mx4")
    full = layer(x.cuda(), z.cuda(), hidden, answer, 2)
    pad = torch.zeros(tokens, dtype=torch.bool)
    pad[5::3] = True
    x2, z2 = x.clone(), z.clone()
    x2[pad], z2[pad] = NAN, -INF
    got = layer(x2.cuda(), z2.cuda(), hidden, answer, 2)
    assert got[pad].eq(0).all() and torch.equal(got[~pad], full[~pad])


@pytest.mark.parametrize("tokens", [9, 300])
def test_layer_in_a_graph_and_on_a_stream(tokens):
    """captured once, replayed on changing inputs with eager work between; two graphs of the same shapes share nothing"""
    x, z, hidden, answer, hv, av = layer_case(3, tokens, "bf16-mx4")
    xs, zs = [x.cuda(), x.cuda() * 2], [z.cuda(), -z.cuda()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = layer(xs[0], zs[0], hidden, answer, 2)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, layer(xs[0], zs[0], hidden, answer, 2))
    graphs, outs, ins = [], [], []
    for i in range(2):
        xi, zi = xs[i].clone(), zs[i].clone()
        gr = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr):
            out = layer(xi, zi, hidden, answer, 2)
        graphs.append(gr), outs.append(out), ins.append((xi, zi))
    for turn in range(4):
        for i in range(2):
            ins[i][0].copy_(xs[(turn + i) % 2] + turn)
            ins[i][1].copy_(zs[(turn + i) % 2])
        graphs[0].replay()
        graphs[1].replay()
        for i in range(2):
            assert torch.equal(outs[i], layer(*ins[i], hidden, answer, 2)), (turn, i)
        torch.cuda.synchronize()


def test_same_answer_every_time():
    x, z, hidden, answer, hv, av = layer_case(3, 700, "f16-mx4")
    a = (x.cuda(), z.cuda(), hidden, answer, 2)
    first = layer(*a)
    for _ in range(5):
        assert torch.equal(layer(*a), first)


def test_packed_by_the_gpu_and_used_at_once():
    """weights and activations packed on the GPU, and the product of the packed pair"""
    g = gen(4)
    x, w = randn(g, 130, 200).to(BF16), randn(g, 90, 200, scale=0.07).to(BF16)
    qx, qw = ops.mx4_quantize(x.cuda()), ops.mx4_quantize(w.cuda())
    mx4ref.close(ops.mx4_linear(qx, qw, dtype=BF16), *mx4ref.linear(mx4ref.unpack(*mx4ref.pack(x), 200), mx4ref.unpack(*mx4ref.pack(w), 200)))


# ---- sizes behind 32 bits -----------------------------------------------------------------------------------------------------------------


def test_gather_from_more_than_4_gb():
    """rows of x behind 2^32 bytes, for few and for many slots"""
    g = gen(1)
    t, k, n = 270000, 8192, 40
    x = torch.empty((t, k), dtype=F16, device="cuda")                   # 4.4 GB; only the rows that are read are written
    w = randn(g, 2, n, k, scale=k ** -0.5).to(F16)
    for m in (7, 90):
        at = torch.randint(t - 9000, t, (m,), generator=g)
        at[0], at[-1] = t - 1, 0
        v = randn(g, m, k).to(F16)
        x[at.cuda()] = v.cuda()
        v = x[at.cuda()].cpu()                                          # (a row drawn twice)
        off = [0, m // 3, m]
        got = ops.expert_linear(x, w.cuda(), torch.tensor(off, dtype=torch.int32, device="cuda"), at.int().cuda())
        mx4ref.close(got, *grouped(v.double(), w.double(), off, list(range(m))))


@pytest.mark.parametrize("m", [3, 20, 300])
def test_weights_of_more_than_2_gb(m):
    """one matrix of 2.6 GB: the last rows' offsets need all 32 bits"""
    g = gen(2)
    n, k = 40000, 32768
    w = torch.zeros((1, n, k), dtype=BF16, device="cuda")
    rows = [0, 1, 20000, n - 2, n - 1]
    v = randn(g, len(rows), k, scale=k ** -0.5).to(BF16)
    w[0, rows] = v.cuda()
    x = randn(g, m, k).to(BF16)
    got = ops.expert_linear(x.cuda(), w, torch.tensor([0, m], dtype=torch.int32, device="cuda")).cpu()
    mx4ref.close(got[:, rows], *mx4ref.linear(x, v))
    rest = torch.ones(n, dtype=torch.bool)
    rest[rows] = False
    assert got[:, rest].eq(0).all()


@pytest.mark.parametrize("kind", ["f16", "bf16-mx4"])
def test_experts_behind_4_gb(kind):
    """the last of many experts lies behind 2^32 bytes (fp16) of the first"""
    g = gen(3)
    e, n, k = 80, 4096, 8192
    last = randn(g, n, k, scale=k ** -0.5)
    if kind == "f16":
        w = torch.empty((e, n, k), dtype=F16, device="cuda")
        w[-1] = last.to(F16).cuda()
        wv, dt = last.to(F16).double(), F16
    else:
        c, s = mx4ref.pack(last)
        w = ops.Mx4(torch.empty((e, n, k // 2), dtype=torch.uint8, device="cuda"), torch.empty((e, n, k // 32), dtype=torch.uint8, device="cuda"), k)
        w.codes[-1], w.scales[-1] = c.cuda(), s.cuda()
        wv, dt = mx4ref.unpack(c, s, k), BF16
    for m in (5, 40):
        x = randn(g, m, k).to(dt)
        off = torch.zeros(e + 1, dtype=torch.int32)
        off[-1] = m
        mx4ref.close(ops.expert_linear(x.cuda(), w, off.cuda()), *mx4ref.linear(x, wv))


def test_outputs_of_more_than_2_31_elements():
    g = gen(4)
    m, n, k = 300000, 8192, 32
    w = randn(g, n, k, scale=0.2)
    q = mx4(w)
    x = randn(g, m, k).to(BF16)
    got = ops.mx4_linear(x.cuda(), q)
    some = torch.cat((torch.arange(40), torch.arange(262100, 262200), torch.arange(m - 40, m)))
    mx4ref.close(got[some.cuda()], *mx4ref.linear(x[some], val(q)))
    # ... as the operand of the weighted sum, of the packing and of the reading back
    slots = torch.stack((some, some.flip(0)), 1).int()
    wt = torch.rand(slots.shape, generator=g)
    y = got[slots.flatten().long().cuda()].cpu().double().view(*slots.shape, n)
    mx4ref.close(ops.moe_combine(got, slots.cuda(), wt.cuda()), (y * wt.double()[..., None]).sum(1), 2.0 ** -21 * (y.abs() * wt.double()[..., None]).sum(1))
    p = ops.mx4_quantize(got)
    c, s = mx4ref.pack(got[some.cuda()].cpu())
    assert torch.equal(p.codes[some.cuda()].cpu(), c) and torch.equal(p.scales[some.cuda()].cpu(), s)
    back = ops.mx4_dequantize(p, BF16)
    assert torch.equal(back[some.cuda()].cpu().double(), mx4ref.unpack(c, s, n))


@pytest.mark.parametrize("tokens, e, k", [(70, 300, 5), (33, 600, 17), (200, 1024, 32), (100000, 16, 2)])
def test_route_wide_and_long(tokens, e, k):
    z = randn(gen(e), tokens, e)
    if tokens < 1000:
        same_route(z, k, True)
        same_route(z.to(BF16), k, False)                                # many ties
        return
    got = ops.moe_route(z.cuda(), k)
    ex = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :k]
    order = torch.sort(ex.flatten(), stable=True).indices
    assert torch.equal(got.experts.cpu().long(), ex) and torch.equal(got.rows.cpu().long(), order // k)
    assert torch.equal(got.slots.cpu().flatten()[order].long(), torch.arange(tokens * k)) and got.offsets.cpu().tolist() == [0] + torch.bincount(ex.flatten(), minlength=e).cumsum(0).tolist()


# ---- every kernel behind the products ------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind, aligned", [(k, True) for k in KINDS] + [(k, False) for k in KINDS if k != "mx4-mx4"])
@pytest.mark.parametrize("m, n, k", [(17, 256, 4096), (40, 130, 8192), (129, 1000, 2048), (1000, 1100, 264), (700, 4096, 72), (2500, 3300, 136), (2048, 4096, 1000), (3100, 4100, 200), (4096, 4096, 1032)])
def test_products_of_all_shapes(kind, m, n, k, aligned):
    """split and whole K, the three tile shapes, whole and ragged rows; every output against fp64 on the GPU"""
    g = torch.Generator("cuda").manual_seed(m + n + k)
    k -= 0 if aligned else 3
    dt = BF16 if kind.startswith("bf16") else F16
    x = torch.randn((m, k), generator=g, device="cuda").to(dt)
    w = torch.randn((n, k), generator=g, device="cuda") * k ** -0.5
    xv = x.double()
    if kind == "mx4-mx4":
        x = ops.mx4_quantize(x)
        xv = ops.mx4_dequantize(x, F32).double()                        # (exact: tested above)
    if kind.endswith("mx4"):
        w = ops.mx4_quantize(w)
        wv = ops.mx4_dequantize(w, F32).double()
        got = ops.mx4_linear(x, w, dtype=F32)
    else:
        w = w.to(dt)[None]
        wv = w[0].double()
        got = ops.expert_linear(x, w, torch.tensor([0, m], dtype=torch.int32, device="cuda"), dtype=F32)
    want, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    lim = (k / 8 + 64) * 2.0 ** -23 * mag + 2.0 ** -23 * xv.abs().sum(1, keepdim=True) * wv.abs().amax(1)
    assert ((got.double() - want).abs() <= lim).all()


@pytest.mark.parametrize("kind, k", [(k, 264) for k in KINDS] + [(k, 261) for k in KINDS if k != "mx4-mx4"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes, n", [([0, 700, 1, 2500, 256, 130, 900], 2100), ([40, 90, 33, 64, 0, 17], 520), ([20] * 20, 100)])
def test_groups_of_all_shapes(kind, k, gated, sizes, n):
    """ragged groups with gathered rows and a bias on the tile kernels; every output against fp64 on the GPU"""
    g = torch.Generator("cuda").manual_seed(n + k + gated)
    dt = BF16 if kind.startswith("bf16") else F16
    m, e, wn = sum(sizes), len(sizes), 2 * n if gated else n
    x = torch.randn((m, k), generator=g, device="cuda").to(dt)
    w = torch.randn((e, wn, k), generator=g, device="cuda") * k ** -0.5
    rows = torch.randint(-1, m, (m,), generator=g, device="cuda").int()      # -1: a row of zeros
    bias = torch.randn((e, wn), generator=g, device="cuda")
    xv = x.double()
    if kind == "mx4-mx4":
        x = ops.mx4_quantize(x)
        xv = ops.mx4_dequantize(x, F32).double()
    if kind.endswith("mx4"):
        w = ops.mx4_quantize(w)
        wv = ops.mx4_dequantize(w, F32).double()
    else:
        w = w.to(dt)
        wv = w.double()
    off = [0] + torch.tensor(sizes).cumsum(0).tolist()
    got = ops.expert_linear(x, w, torch.tensor(off, dtype=torch.int32, device="cuda"), rows, bias, gated=gated, dtype=F32).double()
    for i in range(e):
        r = rows[off[i]:off[i + 1]].long()
        v = torch.where(r[:, None] >= 0, xv[r.clamp(min=0)], torch.zeros((), dtype=torch.float64, device="cuda"))
        z, mag = v @ wv[i].t() + bias[i].double(), v.abs() @ wv[i].abs().t()
        lim = (k / 8 + 64) * 2.0 ** -23 * mag + 2.0 ** -23 * v.abs().sum(1, keepdim=True) * wv[i].abs().amax(1) + 2.0 ** -23 * z.abs()
        if gated:                                                       # |silu'| < 1.1; the exponential, the division and the products below 2^-19 of the result
            a, b, la, lb = z[:, :n], z[:, n:], lim[:, :n], lim[:, n:]
            s = a * torch.sigmoid(a)
            z, lim = s * b, 1.1 * la * b.abs() + s.abs() * lb + 1.1 * la * lb + 2.0 ** -19 * (s * b).abs()
        assert ((got[off[i]:off[i + 1]] - z).abs() <= lim).all(), i


# ---- what a caller may also do --------------------------------------------------------------------------------------------------------------

WAYS = [(6, 40, 96), (90, 256, 512), (90, 256, 4096), (1500, 2048, 512), (4000, 4096, 256), (7000, 2048, 256)]     # slots, columns, K: streamed, few tiles, K split, the three tiles


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m, n, k", WAYS)
def test_weights_that_are_not_finite(kind, m, n, k):
    """a weight row with an infinity or a NaN reaches its own column only, and no slot without a row of x (its product is zero, whatever the weights hold)"""
    g = gen(m)
    x, xv, w, wv, dt = operands(kind, g, m, k, (2, n, k))
    rows = torch.arange(m, dtype=torch.int32)
    rows[2::3] = -1
    off = torch.tensor([0, m // 2 + 1, m], dtype=torch.int32, device="cuda")
    bias = randn(g, 2, n)
    fine = ops.expert_linear(x, w, off, rows.cuda(), bias.cuda())
    if isinstance(w, ops.Mx4):
        s = w.scales.clone()
        s[:, 3, 0], s[:, 9, -1] = 255, 255
        bad = ops.Mx4(w.codes, s, k)
    else:
        bad = w.clone()
        bad[:, 3, 1], bad[:, 9, k - 1] = NAN, INF
    got = ops.expert_linear(x, bad, off, rows.cuda(), bias.cuda())
    cols = [j for j in range(n) if j not in (3, 9)]
    assert torch.equal(got[:, cols], fine[:, cols])
    none = rows.cuda() < 0
    assert not torch.isfinite(got[~none][:, [3, 9]]).any()
    want = bias.to(dt)[torch.bucketize(torch.arange(m), off.cpu()[1:], right=True)]
    assert torch.equal(got[none].cpu(), want[rows < 0])


@pytest.mark.parametrize("kind", ["bf16", "f16-mx4", "mx4-mx4"])
@pytest.mark.parametrize("m, n, k", WAYS[1:4])
def test_two_calls_at_once(kind, m, n, k):
    """the same layer on two streams at the same time, each with scratch of its own"""
    g = gen(5)
    x, xv, w, wv, dt = operands(kind, g, m, k, (1, n, k))
    y, yv, _, _, _ = operands(kind, g, m, k, (1, 1, k))
    off = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    want = [ops.expert_linear(v, w, off) for v in (x, y)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, v in enumerate((x, y)):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.expert_linear(v, w, off))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i]) for i in range(2) for a in got[i])


@pytest.mark.parametrize("kind", ["f16", "bf16-mx4", "mx4-mx4"])
@pytest.mark.parametrize("m, n, k", WAYS[:5])
def test_groups_that_overlap_or_descend(kind, m, n, k):
    """offsets are meant to ascend; others cost nothing but the slots they name: nothing beside the slots is written"""
    x, xv, w, wv, dt = operands(kind, gen(6), m, k, (4, n, k))
    out = torch.full((m + 2, n), 7.0, dtype=dt, device="cuda")
    for off in ([m, 0, m, 0, m], [0, m, 0, m, 0], [m, m, 0, 0, 0], [-(1 << 31), (1 << 31) - 1, -5, 3, 1 << 30]):
        ops.expert_linear(x, w, torch.tensor(off, dtype=torch.int32, device="cuda"), out=out[1:m + 1])
    assert out[0].eq(7).all() and out[m + 1].eq(7).all()


def test_masked_scores_of_the_lowest_value():
    """a mask of the type's lowest finite value is a score like any other: chosen last, with weight 0"""
    for t in (F16, BF16, F32):
        z = torch.full((70, 8), torch.finfo(t).min, dtype=t)
        z[:, 5] = 1
        p = ops.moe_route(z.cuda(), 2)
        assert p.experts.cpu().eq(torch.tensor([5, 0])).all() and p.weights.cpu().eq(torch.tensor([1.0, 0.0])).all()
        assert p.offsets.cpu().tolist() == [0, 70, 70, 70, 70, 70, 140, 140, 140]
        p = ops.moe_route(torch.full((3, 8), torch.finfo(t).min, dtype=t).cuda(), 2)
        assert p.experts.cpu().eq(torch.tensor([0, 1])).all() and p.weights.eq(0.5).all()


@pytest.mark.parametrize("kind, aligned", [(k, True) for k in KINDS] + [(k, False) for k in KINDS if k != "mx4-mx4"])
@pytest.mark.parametrize("m, n, k", [(4400, 4096, 264), (1400, 4000, 200), (1100, 4000, 136), (2000, 4040, 72)])
def test_products_between_whole_rounds(kind, aligned, m, n, k):
    """numbers of tiles a little above what the card holds at once (the last ones are cut in half), one tile of 128 x 128 to some CUs and two to others"""
    test_products_of_all_shapes(kind, m, n, k, aligned)


@pytest.mark.parametrize("kind, k", [(k, 136) for k in KINDS] + [(k, 133) for k in KINDS if k != "mx4-mx4"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("sizes, n", [([1100, 0, 130, 90], 3900), ([257, 385, 128, 1, 640, 900, 300, 1500], 4000)])
def test_groups_between_whole_rounds(kind, k, gated, sizes, n):
    test_groups_of_all_shapes(kind, k, gated, sizes, n)


@pytest.mark.parametrize("kind", ["bf16", "bf16-mx4"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m, n, k", WAYS + [(300, 1004, 520)])
def test_fp16_answers_of_bf16_rows(kind, gated, m, n, k):
    """a bf16 layer that hands fp16 to the next one: rounded once, to eleven bits"""
    g = torch.Generator("cuda").manual_seed(m + n)
    x = torch.randn((m, k), generator=g, device="cuda").to(BF16)
    w = torch.randn((2 * n if gated else n, k), generator=g, device="cuda") * k ** -0.5
    if kind == "bf16":
        w = w.to(BF16)
        got, wv = ops.expert_linear(x, w[None], torch.tensor([0, m], dtype=torch.int32, device="cuda"), gated=gated, dtype=F16), w.double()
    else:
        w = ops.mx4_quantize(w)
        got, wv = ops.mx4_linear(x, w, gated=gated, dtype=F16), ops.mx4_dequantize(w, F32).double()
    assert got.dtype == F16
    z, mag = x.double() @ wv.t(), x.double().abs() @ wv.abs().t()
    err = (k / 8 + 64) * 2.0 ** -23 * mag + 2.0 ** -23 * x.double().abs().sum(1, keepdim=True) * wv.abs().amax(1)
    if gated:                                                            # as mx4ref.linear: |silu'| < 1.1; the exponential, division and products: below 2^-19 of the result
        a, b, ea, eb = z[:, :n], z[:, n:], err[:, :n], err[:, n:]
        s = a * torch.sigmoid(a)
        z, err = s * b, 1.1 * ea * b.abs() + s.abs() * eb + 1.1 * ea * eb + 2.0 ** -19 * (s * b).abs()
    lim = err + 2.0 ** -11 * (z.abs() + err) + 2.0 ** -25
    assert ((got.double() - z).abs() <= lim).all()


@pytest.mark.parametrize("weights", [F16, BF16, "mx4"])
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("m, n, k", [(1, 24, 1), (7, 40, 96), (33, 130, 261), (90, 256, 4096), (1500, 1000, 72)])
def test_fp32_rows(weights, gated, m, n, k):
    """fp32 rows in two parts: right to 2^-16 of the products' magnitudes (bf16 parts: what two roundings of half a step 2^-8 leave), 2^-22 under fp16 weights (2^-11 each)"""
    g = torch.Generator("cuda").manual_seed(m + n + k)
    t = m // 2 + 1
    x = torch.randn((t, k + 3), generator=g, device="cuda")[:, 2:k + 2]
    rows = torch.randint(-1, t + 1, (m,), generator=g, device="cuda").int()             # -1, t: no row of x
    off = torch.tensor([0, m // 3, m // 3, m], dtype=torch.int32, device="cuda")
    wn = 2 * n if gated else n
    w = torch.randn((3, wn, k), generator=g, device="cuda") * k ** -0.5
    bias = torch.randn((3, wn), generator=g, device="cuda")
    if weights == "mx4":
        w = ops.mx4_quantize(w)
        wv = ops.mx4_dequantize(w, F32).double()
    else:
        w = w.to(weights)
        wv = w.double()
    got = ops.expert_linear(x, w, off, rows, bias, gated=gated)
    assert got.dtype == F32 and got.shape == (m, n)
    ok = ((rows >= 0) & (rows < t))[:, None]
    xv = torch.where(ok, x.double()[rows.clamp(0, t - 1).long()], torch.zeros((), dtype=torch.float64, device="cuda"))
    part = 2.0 ** -22 if weights == F16 else 2.0 ** -16
    for e in range(3):
        s = slice(int(off[e]), int(off[e + 1]))
        z, mag = xv[s] @ wv[e].t(), xv[s].abs() @ wv[e].abs().t()
        err = (k / 8 + 64) * 2.0 ** -22 * mag + 2.0 ** -22 * xv[s].abs().sum(1, keepdim=True) * wv[e].abs().amax(1) + part * mag + 2.0 ** -24 * wv[e].abs().sum(1)
        z = z + bias[e].double()
        err = err + 2.0 ** -23 * z.abs()
        if gated:
            a, b, ea, eb = z[:, :n], z[:, n:], err[:, :n], err[:, n:]
            q = a * torch.sigmoid(a)
            z, err = q * b, 1.1 * ea * b.abs() + q.abs() * eb + 1.1 * ea * eb + 2.0 ** -19 * (q * b).abs()
        assert ((got[s].double() - z).abs() <= err + 2.0 ** -24 * z.abs()).all(), e
    out = torch.full((m + 1, n + 8), 7.0, dtype=BF16, device="cuda")
    ops.expert_linear(x, w, off, rows, bias, gated=gated, out=out[:m, :n])
    assert torch.equal(out[:m, :n], got.to(BF16)) and out[m].eq(7).all() and out[:, n:].eq(7).all()


def test_fp32_rows_of_nothing_and_infinities():
    off = torch.tensor([0, 0, 2], dtype=torch.int32, device="cuda")
    w = torch.ones((2, 8, 40), dtype=BF16, device="cuda")
    bias = torch.full((2, 8), 3.0, device="cuda")
    x = torch.ones((3, 40), device="cuda")
    x[0, 4], x[1, 5] = INF, NAN
    got = ops.expert_linear(x, w, off, torch.tensor([0, 2], dtype=torch.int32, device="cuda"), bias)
    assert got[0].eq(INF).all() and got[1].eq(43).all()
    assert ops.expert_linear(x, w, off, torch.tensor([1, 2], dtype=torch.int32, device="cuda"), bias)[0].isnan().all()
    w[1, 3] = INF
    got = ops.expert_linear(x, w, off, torch.tensor([-1, 2], dtype=torch.int32, device="cuda"), bias)
    assert got[0].eq(3).all() and got[1, 3].eq(INF) and got[1, 2].eq(43)
    assert ops.expert_linear(x[:0], w, off, torch.tensor([0, 0], dtype=torch.int32, device="cuda"), bias).eq(3).all()
    assert ops.expert_linear(x[:, :0], w[:, :, :0], torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda"), bias=bias).eq(3).all()
    out = torch.full((4, 8), 7.0, device="cuda")
    ops.expert_linear(torch.ones((4, 40), device="cuda"), w, torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), out=out)
    assert out[0].eq(7).all() and out[3].eq(7).all() and out[1].eq(40).all()


def test_fp32_rows_in_a_graph():
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn((70, 256), generator=g, device="cuda")
    w = ops.mx4_quantize(torch.randn((2, 96, 256), generator=g, device="cuda"))
    off = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    ops.expert_linear(x, w, off)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = ops.expert_linear(x, w, off)
    for turn in range(4):
        x.mul_(1.5)
        off.copy_(torch.tensor([0, 10 * turn + 5, 70], dtype=torch.int32))
        gr.replay()
        assert torch.equal(y, ops.expert_linear(x, w, off)), turn
        torch.cuda.synchronize()
