"""Linear and expert layers over the whole range of their operands: rows of very large, very small and mixed values, weights whose scales lie far apart.
Every limit here is relative to the sum of the products' own magnitudes: nothing is allowed for values that a product does not hold."""
import ctypes as C

import pytest
import torch

from smelter_amd import _native as N
from smelter_amd import ops

pytestmark = pytest.mark.gpu
F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
INF, NAN = float("inf"), float("nan")


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def chain(k):
    """An fp32 sum of k exact products, in any order: at most k + 16 additions (16: partial sums of waves, lane groups, runs and parts) that round by half a step, 2^-24, or are cut, 2^-23"""
    return (k + 16) * 2.0 ** -23


def inside(got, want, lim, what=""):
    """|got - want| <= lim + half a step of got's type (its smallest value's half below its range); the same infinities and NaN"""
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = torch.isinf(want)
    assert torch.equal(got.double()[inf], want[inf]), what
    info = torch.finfo(got.dtype)
    fine = torch.isfinite(want) & (want.abs() + lim < info.max)         # (near the end of the range a value may round to an infinity)
    off = (got.double() - want).abs() - lim - info.eps / 2 * (want.abs() + lim) - info.smallest_normal * info.eps / 2
    bad = fine & ~(off <= 0)
    assert not bad.any(), "%s: off by %.3g of %.3g where %.3g is allowed, at %s" % (what, (got.double() - want).abs()[bad][0], want[bad][0], lim.expand_as(want)[bad][0], bad.nonzero()[0].tolist())


def gate(z, lim, n):
    """silu(a) * b of the halves: |silu'| < 1.1; the exponential, the reciprocal and the products below 2^-19 of the result"""
    a, b, la, lb = z[:, :n], z[:, n:], lim[:, :n], lim[:, n:]
    s = a * torch.sigmoid(a)
    return s * b, 1.1 * la * b.abs() + s.abs() * lb + 1.1 * la * lb + 2.0 ** -19 * (s * b).abs()


def fp32_rows(g, m, k):
    """rows whose magnitudes differ: all near 1e5, 1e-5, 1e-8, 1e30, 1e-30, of one magnitude for each element, with loud columns, behind a loud first column"""
    x = randn(g, m, k)
    scale = torch.tensor([1e5, 1e-5, 1e-8, 1e30, 1e-30, 1.0, 1.0, 1e-8], device="cuda")[torch.arange(m, device="cuda") % 8]
    x = x * scale[:, None]
    mixed = torch.arange(m, device="cuda") % 8 == 5
    x = torch.where(mixed[:, None], x * 10.0 ** torch.randint(-9, 6, (m, k), generator=g, device="cuda").float(), x)
    loud = torch.arange(m, device="cuda") % 8 >= 6
    x[:, 0] = torch.where(loud, torch.full_like(x[:, 0], 7e4), x[:, 0])
    return x


def same_as_fp64(x, w, wv, off, rows, bias, gated, dtype, more=0.0):
    """fp32 rows on weights [2, N, K]; `more`: of the products' magnitudes, allowed beside the sum's own error"""
    got = ops.expert_linear(x, w, off, rows, bias, gated=gated, dtype=dtype)
    t, k = x.shape
    n = wv.shape[1] // (2 if gated else 1)
    ok = ((rows >= 0) & (rows < t))[:, None]
    xv = torch.where(ok, x.double()[rows.clamp(0, t - 1).long()], torch.zeros((), dtype=F64, device="cuda"))
    for e in range(2):
        s = slice(int(off[e]), int(off[e + 1]))
        z, mag = xv[s] @ wv[e].t() + bias[e].double(), xv[s].abs() @ wv[e].abs().t()
        lim = (chain(k) + more) * mag + 2.0 ** -23 * z.abs() + 2.0 ** -126
        if gated:
            z, lim = gate(z, lim, n)
        inside(got[s], z, lim, "group %d" % e)
    return got


@pytest.mark.parametrize("gated, dtype", [(False, F32), (True, F32), (False, BF16), (True, F16)])
@pytest.mark.parametrize("m, n, k", [(1, 24, 1), (8, 40, 96), (40, 130, 261), (96, 256, 4096), (64, 2048, 2048), (1500, 1000, 72)])
def test_fp32_rows_on_fp16_weights(gated, dtype, m, n, k):
    """no row is too large, too small or too mixed (some are multiplied in other ways than others).  Some weight rows are zero where the loud column is"""
    g = gen(m + n + k)
    x = torch.full((m, k + 3), NAN, device="cuda")[:, 2:k + 2]
    x.copy_(fp32_rows(g, m, k))
    w = (randn(g, 2, 2 * n if gated else n, k) * k ** -0.5).to(F16)
    w[:, ::3, 0] = 0
    rows = torch.randint(-1, m + 1, (m + 5,), generator=g, device="cuda").int()          # -1, m: no row of x
    off = torch.tensor([0, m // 3 + 1, m + 5], dtype=torch.int32, device="cuda")
    same_as_fp64(x, w, w.double(), off, rows, randn(g, 2, w.shape[1]) * 1e-8, gated, dtype)


@pytest.mark.parametrize("weights", [BF16, "mx4"])
@pytest.mark.parametrize("gated, dtype", [(False, F32), (True, F32), (False, BF16)])
@pytest.mark.parametrize("m, n, k", [(1, 24, 1), (8, 40, 96), (40, 130, 261), (96, 256, 4096), (64, 2048, 2048), (1500, 1000, 72)])
def test_fp32_rows_keep_their_bits(weights, gated, dtype, m, n, k):
    """under bf16 and MX4 weights an fp32 row is not rounded to 16 bits on its way"""
    g = gen(m + n + k)
    x = torch.full((m, k + 3), NAN, device="cuda")[:, 2:k + 2]
    x.copy_(fp32_rows(g, m, k))
    w = randn(g, 2, 2 * n if gated else n, k) * k ** -0.5
    w[:, ::3, 0] = 0
    if weights == "mx4":
        w = ops.mx4_quantize(w)
        wv = ops.mx4_dequantize(w, F32).double()
    else:
        w = w.to(weights)
        wv = w.double()
    rows = torch.randint(-1, m + 1, (m + 5,), generator=g, device="cuda").int()
    off = torch.tensor([0, m // 3 + 1, m + 5], dtype=torch.int32, device="cuda")
    same_as_fp64(x, w, wv, off, rows, randn(g, 2, wv.shape[1]) * 1e-8, gated, dtype)


def test_fp32_rows_at_the_end_of_the_range():
    """values that bf16 would round to an infinity, under weights of 1, and each of them under an infinite weight"""
    off = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    x = torch.tensor([[3.4028235e38], [-3.4e38], [1.1754944e-38], [1 + 2.0 ** -23]], device="cuda")
    for w in (torch.ones((1, 8, 1), dtype=BF16, device="cuda"), ops.mx4_quantize(torch.ones((1, 8, 1), device="cuda")), torch.ones((1, 8, 1), dtype=F16, device="cuda")):
        assert torch.equal(ops.expert_linear(x, w, off), x.expand(4, 8))
    for t in (BF16, F16):
        got = ops.expert_linear(x, torch.full((1, 8, 1), INF, dtype=t, device="cuda"), off)
        assert torch.equal(got, torch.tensor([[INF], [-INF], [INF], [INF]], device="cuda").expand(4, 8))


@pytest.mark.parametrize("reach", [20, 37, 38, 39, 60])
@pytest.mark.parametrize("m, n, k", [(6, 40, 96), (90, 256, 520), (700, 1000, 264)])
def test_fp32_rows_at_the_edge_of_fp16_parts(reach, m, n, k):
    """elements down to 2^-reach of the first, which meets weights of zero: each is there with all its bits"""
    g = gen(reach)
    x = (1 + torch.rand((m, k), generator=g, device="cuda")) * torch.exp2(-torch.randint(0, reach + 1, (m, k), generator=g, device="cuda").float())
    x = x * torch.exp2(torch.randint(-60, 60, (m, 1), generator=g, device="cuda").float())
    x[::3] *= 2.0 ** -(reach - 1)
    x[:, 0] = x[:, 1:].amax(1) * (2.0 ** reach if reach < 38 else 1.0)
    w = (randn(g, 1, n, k) / 8).to(F16)
    w[..., 0] = 0
    w[:, ::2, 1:] *= (x[0, 1:] < x[0, 1:].amax() * 2.0 ** -(reach // 2)).half()       # rows of weights that meet small elements only
    off = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    xv, wv = x.double(), w[0].double()
    inside(ops.expert_linear(x, w, off), xv @ wv.t(), chain(3 * k) * (xv.abs() @ wv.abs().t()) + 2.0 ** -126)


def test_fp32_rows_on_fp16_weights_one_by_one():
    """values whose fp16 form is an infinity, coarse or zero"""
    off = torch.tensor([0, 5], dtype=torch.int32, device="cuda")
    x = torch.tensor([[7e4], [3e-5], [1e-6], [2e-8], [1e-9]], device="cuda")
    w = torch.tensor([[[0.1], [1.0]]], device="cuda").to(F16)
    want = x.double() * w[0, :, 0].double()
    inside(ops.expert_linear(x, w, off), want, 2.0 ** -23 * want.abs())
    w[0, 1] = INF
    got = ops.expert_linear(x, w, off)
    assert got[:, 1].eq(INF).all() and torch.isfinite(got[:, 0]).all()
    assert torch.equal(ops.expert_linear(-x, w, off), -got)
    # two large terms of opposite signs
    pair = torch.tensor([[7e4, -7e4]] * 5, device="cuda")
    assert ops.expert_linear(pair, torch.ones((1, 8, 2), dtype=F16, device="cuda"), off).eq(0).all()
    # an infinity and a NaN beside small values
    odd = torch.tensor([[INF, 1e-9], [-INF, 1e-9], [NAN, 1.0], [INF, -INF], [1e-9, 1.0]], device="cuda")
    got = ops.expert_linear(odd, torch.ones((1, 8, 2), dtype=F16, device="cuda"), off)
    assert got[0].eq(INF).all() and got[1].eq(-INF).all() and got[2:4].isnan().all() and got[4].eq(1).all()


@pytest.mark.parametrize("weights", [F16, "mx4"])
@pytest.mark.parametrize("act, slope, f", [(ops.ACT_RELU, 0.0, lambda z: z.clamp(min=0)), (ops.ACT_PRELU, 0.25, lambda z: torch.where(z < 0, 0.25 * z, z)), (ops.ACT_CLIP, 0.5, lambda z: z.clamp(0, 0.5))])
@pytest.mark.parametrize("m", [5, 200])
def test_fp32_rows_without_groups(weights, act, slope, f, m):
    """one layer without offsets, with activations (their slopes are at most 1): from Python, and through the C interface for fp16 weights"""
    g = gen(m)
    n, k = 72, 200
    x, w, bias = fp32_rows(g, m, k), randn(g, n, k) * k ** -0.5, randn(g, n)
    if weights == "mx4":
        w = ops.mx4_quantize(w)
        wv = ops.mx4_dequantize(w, F32).double()
        got = ops.mx4_linear(x, w, bias, act=act, slope=slope)
    else:
        w = w.to(weights)
        wv, got = w.double(), torch.empty((m, n), device="cuda")
        d = N.LinearDesc(m, m, n, k, 1, 2, 0, 2, act, slope, 0, 0, 0)
        size = N.lib().sm_linear_workspace_bytes(C.byref(d), 0, 0)
        work = torch.empty(size, dtype=torch.uint8, device="cuda")
        N.check(N.lib().sm_linear_fwd(C.byref(d), x.data_ptr(), None, w.data_ptr(), None, bias.data_ptr(), None, None, got.data_ptr(), work.data_ptr(), size, torch.cuda.current_stream().cuda_stream))
    z, mag = x.double() @ wv.t() + bias.double(), x.double().abs() @ wv.abs().t()
    inside(got, f(z), chain(3 * k) * mag + 2.0 ** -23 * z.abs() + 2.0 ** -126)


@pytest.mark.parametrize("weights", [F16, BF16])
def test_fp32_rows_more_than_blocks(weights):
    """a block takes several slots, ordinary and odd ones after one another"""
    g = gen(8)
    m, n, k = 40000, 24, 72
    x, w = fp32_rows(g, m, k), (randn(g, 2, n, k) / 8).to(weights)
    rows = torch.randperm(m, generator=g, device="cuda").int()
    rows[5::7] = -1
    off = torch.tensor([0, 15000, m], dtype=torch.int32, device="cuda")
    same_as_fp64(x, w, w.double(), off, rows, randn(g, 2, n), False, F32)


@pytest.mark.parametrize("weights", [F16, BF16])
@pytest.mark.parametrize("m", [4, 700])
def test_fp32_rows_beside_their_outputs(weights, m):
    """slots that no group covers, and what lies beside the outputs, stay as they were, whichever way a row is multiplied"""
    g = gen(9)
    n, k = 40, 96
    x, w = fp32_rows(g, m, k), (randn(g, 2, n, k) / 8).to(weights)
    for dtype in (F32, F16):
        out = torch.full((m + 2, n + 7), 7.0, dtype=dtype, device="cuda")
        off = torch.tensor([1, m // 2, m - 1], dtype=torch.int32, device="cuda")
        ops.expert_linear(x, w, off, out=out[1:m + 1, 2:n + 2])
        whole = ops.expert_linear(x, w, torch.tensor([0, m // 2, m], dtype=torch.int32, device="cuda"), dtype=dtype)
        assert torch.equal(out[2:m, 2:n + 2], whole[1:m - 1])
        out[2:m, 2:n + 2] = 7
        assert out.eq(7).all()


def test_fp32_rows_on_two_streams():
    """two calls at once, each with scratch of its own"""
    g = gen(10)
    xs, w = [fp32_rows(g, 300, 520) for _ in range(2)], (randn(g, 1, 264, 520) / 16).to(F16)
    off = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    want = [ops.expert_linear(x, w, off) for x in xs]
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    torch.cuda.synchronize()
    for _ in range(8):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(ops.expert_linear(xs[i], w, off))
    torch.cuda.synchronize()
    assert all(torch.equal(a, want[i]) for i in range(2) for a in got[i])


def test_fp32_rows_on_fp16_weights_in_a_graph():
    """which rows are multiplied in another way is decided on the device: a replay goes by the present rows"""
    g = gen(3)
    fine, odd = randn(g, 70, 256), fp32_rows(g, 70, 256)
    x, w = fine.clone(), (randn(g, 2, 96, 256) / 16).to(F16)
    off = torch.tensor([0, 30, 70], dtype=torch.int32, device="cuda")
    ops.expert_linear(x, w, off)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = ops.expert_linear(x, w, off)
    for turn in range(4):
        x.copy_(odd.roll(turn, 0) if turn % 2 else fine)
        gr.replay()
        assert torch.equal(y, ops.expert_linear(x, w, off)), turn
        torch.cuda.synchronize()


# ---- MX4 weights whose scales lie far apart ----------------------------------------------------------------------------------------------------

KINDS = [F16, BF16, "mx4"]
WAYS = [(1, 40, 96), (6, 1000, 1500), (16, 200, 2088), (90, 256, 512), (90, 256, 4096), (90, 300, 264), (90, 300, 261), (300, 1000, 333), (1500, 2048, 512), (2304, 4096, 256), (2304, 4096, 251)]


def wide_weights(g, n, k):
    """rows of blocks up to 2^80 apart; ordinary rows; rows with one huge value in a block that is zero otherwise, with blocks of zeros, with a block just inside and just outside fp16's reach"""
    nb = -(-k // 32)
    blocks = lambda v: v.repeat_interleave(32, -1)[:, :k]  # noqa: E731
    w = randn(g, n, k)
    kind = torch.arange(n, device="cuda") % 6
    far = torch.exp2(torch.randint(-40, 41, (n, nb), generator=g, device="cuda").float())
    w = torch.where((kind == 0)[:, None], w * blocks(far), w)
    w = torch.where((kind == 2)[:, None] & blocks(torch.rand((n, nb), generator=g, device="cuda") < 0.3), torch.zeros_like(w), w)
    edge = torch.exp2(-torch.randint(33, 41, (n, nb), generator=g, device="cuda").float())
    w = torch.where((kind == 3)[:, None], w * blocks(edge), w)
    huge = (kind == 1) | (kind == 3)
    w[:, :32] = torch.where(huge[:, None], torch.zeros_like(w[:, :32]), w[:, :32])
    w[:, 0] = torch.where(huge, torch.where(kind == 1, 2.0 ** 60, 1.0), w[:, 0])
    return w


def mx4ref_values(q):
    """the values of an MX4 tensor in 64 bits (fp32 does not hold the largest)"""
    low = q.scales.clamp(max=200)
    up = torch.exp2((q.scales - low).double()).repeat_interleave(32, -1)[..., :q.k]
    return ops.mx4_dequantize(ops.Mx4(q.codes, low, q.k), F32).double() * up


def rows_of(kind, x):
    """(x as handed over, its values in 64 bits, type of the output)"""
    if kind == "mx4":
        q = ops.mx4_quantize(x)
        return q, ops.mx4_dequantize(q, F32).double(), F16
    return x.to(kind), x.to(kind).double(), kind


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("loud", [False, True])
@pytest.mark.parametrize("m, n, k", WAYS)
def test_scales_far_apart(kind, loud, m, n, k):
    """a block of weights counts for what it is, however large the others of its row are: every other row of x is zero where they are"""
    g = gen(m + n + k)
    w = ops.mx4_quantize(wide_weights(g, n, k))
    wv = ops.mx4_dequantize(w, F32).double()
    x = randn(g, m, k) * (3e4 if loud else 1.0) / (4 if loud else 1)
    x[::2, 0] = 0
    if loud:
        x[1::4, 32:] = 0
    x, xv, dt = rows_of(kind, x)
    z, mag = xv @ wv.t(), xv.abs() @ wv.abs().t()
    inside(ops.mx4_linear(x, w, dtype=F32), z, chain(2 * k) * mag + 2.0 ** -126)
    rows = torch.randint(-1, m + 1, (m + 5,), generator=g, device="cuda").int()
    off = torch.tensor([0, m // 3 + 1, m + 5], dtype=torch.int32, device="cuda")
    both = ops.Mx4(torch.stack((w.codes, w.codes.flip(0))), torch.stack((w.scales, w.scales.flip(0))), k)
    ok = ((rows >= 0) & (rows < m))[:, None]
    got = ops.expert_linear(x, both, off, rows, dtype=F32)
    for e in range(2):
        s = slice(int(off[e]), int(off[e + 1]))
        zero, at = torch.zeros((), dtype=F64, device="cuda"), rows[s].clamp(0, m - 1).long()
        want, lim = torch.where(ok[s], z[at], zero), torch.where(ok[s], mag[at], zero)
        if e:
            want, lim = want.flip(1), lim.flip(1)
        inside(got[s], want, chain(2 * k) * lim + 2.0 ** -126, "group %d" % e)


@pytest.mark.parametrize("kind", [F16, BF16])
@pytest.mark.parametrize("m, n, k", WAYS)
def test_16_bit_weights_of_mixed_magnitudes(kind, m, n, k):
    """a product's limit is its own sum of magnitudes, not the largest weight of its row"""
    g = gen(m + n + k)
    w = randn(g, 2, n, k) * torch.exp2(torch.randint(-14, 9, (2, n, k), generator=g, device="cuda").float())
    w[:, ::3, :32] = 0
    w[:, 1::3, 0] = 6e4
    w = w.to(kind)
    x = randn(g, m, k) * torch.exp2(torch.randint(-14, 9, (m, k), generator=g, device="cuda").float())
    x[::2, 0] = 0
    x = x.to(kind)
    off = torch.tensor([0, m // 3 + 1, m], dtype=torch.int32, device="cuda")
    got = ops.expert_linear(x, w, off, dtype=F32)
    for e in range(2):
        s = slice(int(off[e]), int(off[e + 1]))
        xv, wv = x[s].double(), w[e].double()
        inside(got[s], xv @ wv.t(), chain(k) * (xv.abs() @ wv.abs().t()) + 2.0 ** -126, "group %d" % e)


@pytest.mark.parametrize("m", [1, 16, 17, 90, 1500])
def test_one_far_block(m):
    """two blocks, 2^30 apart and further, x zero in the larger one"""
    for apart in (0, 22, 24, 30, 36, 37, 60, 126):
        scales = torch.tensor([[127, 127 - apart]], dtype=torch.uint8, device="cuda").repeat(24, 1)
        w = ops.Mx4(torch.full((24, 32), 0x22, dtype=torch.uint8, device="cuda"), scales, 64)        # every code 1
        x = torch.zeros((m, 64), dtype=F16, device="cuda")
        x[:, 40] = 30000
        got = ops.mx4_linear(x, w, dtype=F32)
        assert got.eq(30000 * 2.0 ** -apart).all(), apart
        x[:, 41] = INF
        assert ops.mx4_linear(x, w, dtype=F32).eq(INF).all(), apart


@pytest.mark.parametrize("m, n, k", [(1, 40, 96), (17, 40, 96), (90, 256, 4128), (300, 1000, 64), (1500, 2048, 288), (2304, 4096, 288), (2304, 4096, 261)])
def test_both_ends_of_the_scales(m, n, k):
    """blocks of the largest scales beside the smallest ones, x zero where they are or not: as in 64 bits (an infinity behind fp32's range)"""
    g = gen(k)
    q = ops.mx4_quantize(randn(g, n, k))
    q.scales[1::2] = torch.randint(200, 255, q.scales[1::2].shape, generator=g, device="cuda").byte()
    q.scales[1::2, ::2] = torch.randint(0, 60, q.scales[1::2, ::2].shape, generator=g, device="cuda").byte()
    x = (randn(g, m, k) * 2.0 ** -12).to(F16)
    cols = torch.arange(k, device="cuda") // 32 % 2 == 1
    x[::3, cols] = 0
    x[1::3, ~cols] = 0
    w = mx4ref_values(q)
    z, mag = x.double() @ w.t(), x.double().abs() @ w.abs().t()
    got = ops.mx4_linear(x, q, dtype=F32)
    big = z.abs() > 3.3e38
    assert (got.isinf() == (z.abs() > 3.4028235e38))[~big | (z.abs() > 3.5e38)].all() and not got.isnan().any()
    inside(torch.where(big, 0, got), torch.where(big, 0, z), chain(2 * k) * torch.where(mag > 3.3e38, 1e300, mag) + 2.0 ** -126)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("m, n, k", [(1, 40, 96), (17, 40, 96), (90, 256, 4128), (300, 1000, 32), (1500, 2048, 288), (2304, 4096, 288), (2304, 4096, 260)])
def test_largest_scales_in_the_last_block(kind, m, n, k):
    """weights behind fp32's range in the last block of an odd number of blocks: infinities, not NaN"""
    q = ops.mx4_quantize(randn(gen(k), n, k))
    q.scales[1, -1], q.scales[2, -1] = 254, 254
    last = slice(-16, (k - 1) % 32 // 2 - 15 or None)                    # (columns behind the end hold code 0)
    q.codes[1, last], q.codes[2, last] = 0x77, 0xff
    x, xv, _ = rows_of(kind, torch.ones((m, k), device="cuda"))
    got = ops.mx4_linear(x, q, dtype=F32)
    assert got[:, 1].eq(INF).all() and got[:, 2].eq(-INF).all()
    got[:, 1:3] = 0
    wv = ops.mx4_dequantize(q, F32).double()
    wv[1:3] = 0
    inside(got, xv @ wv.t(), chain(2 * k) * (xv.abs() @ wv.abs().t()))


@pytest.mark.parametrize("m", [5, 90])
def test_scales_that_change_between_replays(m):
    """which weights are multiplied in another way is decided on the device"""
    g = gen(2)
    fine, far = ops.mx4_quantize(randn(g, 200, 1024)), ops.mx4_quantize(wide_weights(g, 200, 1024))
    w = ops.Mx4(fine.codes.clone(), fine.scales.clone(), 1024)
    x = randn(g, m, 1024).to(F16)
    ops.mx4_linear(x, w)
    torch.cuda.synchronize()
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        y = ops.mx4_linear(x, w, dtype=F32)
    for turn in range(4):
        now = far if turn % 2 else fine
        w.codes.copy_(now.codes), w.scales.copy_(now.scales)
        gr.replay()
        assert torch.equal(y, ops.mx4_linear(x, now, dtype=F32)), turn
        torch.cuda.synchronize()


# ---- a layer whose hidden values fit no 16-bit type ----------------------------------------------------------------------------------------------


@pytest.mark.parametrize("kind", ["f16", "bf16", "f16-mx4", "bf16-mx4"])
@pytest.mark.parametrize("tokens", [1, 48, 500])
@pytest.mark.parametrize("size", [2.0 ** 6, 2.0 ** -8])
def test_layer_hands_fp32_over(kind, tokens, size):
    """gated hidden values beyond 65504 in some rows (size 2^6: silu(gate) * up of about 2^6 * 2^6 * 2^6) and below 2^-17 in others, handed over in fp32: only the answer's own rounding is left"""
    g = gen(tokens)
    e, k, f, top = 6, 128, 96, 2
    dt = BF16 if kind.startswith("bf16") else F16
    x = (randn(g, tokens, k) * size).to(dt)
    hidden, answer = randn(g, e, 2 * f, k) * k ** -0.5, randn(g, e, k, f) * f ** -0.5
    hidden[:, f:] *= size
    answer *= size ** -3 if size > 1 else 1
    if kind.endswith("mx4"):
        hidden, answer = ops.mx4_quantize(hidden), ops.mx4_quantize(answer)
        hv, av = ops.mx4_dequantize(hidden, F32).double(), ops.mx4_dequantize(answer, F32).double()
    else:
        hidden, answer = hidden.to(dt), answer.to(dt)
        hv, av = hidden.double(), answer.double()
    scores = randn(g, tokens, e)
    plan = ops.moe_route(scores, top)
    h = ops.expert_linear(x, hidden, plan.offsets, plan.rows, gated=True, dtype=F32)
    got = ops.moe_combine(ops.expert_linear(h, answer, plan.offsets, dtype=F32), plan.slots, plan.weights, dtype=dt)
    want, err = torch.zeros((2, tokens, k), dtype=F64, device="cuda")
    reach = 0.0
    for i in range(e):
        tok, j = (plan.experts == i).nonzero(as_tuple=True)
        v = x[tok].double()
        hh, he = gate(v @ hv[i].t(), chain(k) * (v.abs() @ hv[i].abs().t()) + 2.0 ** -126, f)
        he = he + 2.0 ** -24 * hh.abs()
        y, ye = hh @ av[i].t(), chain(3 * f) * ((hh.abs() + he) @ av[i].abs().t()) + he @ av[i].abs().t() + 2.0 ** -126
        part = plan.weights[tok, j].double()[:, None]
        want.index_add_(0, tok, part * y)
        err.index_add_(0, tok, part * (ye + 2.0 ** -21 * (y.abs() + ye)))
        reach = max(reach, hh.abs().max().item() if len(tok) else 0.0)
    if tokens > 1:
        assert reach > 65504 if size > 1 else reach < 2.0 ** -10
    inside(got, want, err)


# ---- sizes that the C interface does not hold ----------------------------------------------------------------------------------------------------


def test_columns_behind_32_bits_are_refused():
    """not cut to their low 32 bits"""
    k = (1 << 32) + 32
    x = torch.empty((1, k), dtype=F16, device="cuda")
    w = torch.empty((1, k // 2), dtype=torch.uint8, device="cuda")
    q = ops.Mx4(w, torch.empty((1, k // 32), dtype=torch.uint8, device="cuda"), k)
    one = torch.zeros((1, 1), device="cuda")
    for f in (lambda: ops.mx4_quantize(x), lambda: ops.mx4_dequantize(q), lambda: ops.mx4_linear(x, q), lambda: ops.moe_combine(x, one.int(), one)):
        with pytest.raises(N.SmelterError) as e:
            f()
        assert e.value.kind == "invalidArgument"
