"""Plain 64-bit forms of the 4-bit and expert-layer operators, from their definitions, on the CPU."""
import numpy as np
import torch

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def pack(x):
    """(codes, scales) of an array [..., K]: e2m1 blocks of 32 with e8m0 scales"""
    x = torch.as_tensor(x).double().numpy()
    k = x.shape[-1]
    nb = -(-k // 32)
    v = np.zeros(x.shape[:-1] + (32 * nb,))
    v[..., :k] = x
    v = v.reshape(x.shape[:-1] + (nb, 32))
    amax = np.abs(v).max(-1, initial=0)
    bad = ~np.isfinite(amax)
    with np.errstate(all="ignore"):
        e = np.where(bad | (amax == 0), -127, np.frexp(amax)[1] - 1 - 2)
    e = np.maximum(e, -127)
    q = np.abs(np.where(bad[..., None], 0, v)) / np.exp2(e.astype(np.float64))[..., None]
    # nearest grid value; of two equally near ones the even code
    d = np.abs(q[..., None] - GRID)
    near = d == d.min(-1, keepdims=True)
    even = near & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
    code = code + np.where(np.signbit(v) & ~bad[..., None], 8, 0)
    code = code.reshape(x.shape[:-1] + (32 * nb,)).astype(np.uint8)
    scale = np.where(bad, 255, e + 127).astype(np.uint8)
    return torch.from_numpy(code[..., 0::2] | (code[..., 1::2] << 4)), torch.from_numpy(scale)


def unpack(codes, scales, k):
    """the fp64 values"""
    c = codes.cpu().numpy()
    v = np.stack((c & 15, c >> 4), -1).reshape(c.shape[:-1] + (2 * c.shape[-1],))
    val = np.where(v >= 8, -1.0, 1.0) * GRID[v & 7]
    s = scales.cpu().numpy().astype(np.float64)
    s = np.where(s == 255, np.nan, np.exp2(s - 127))
    return torch.from_numpy((val * np.repeat(s, 32, -1))[..., :k].copy())


def half_step(t):
    return torch.finfo(t).eps / 2


def linear(x, w, bias=None, act=None, gated=False, k_err=None):
    """(result, bound of an fp32-accumulated kernel's distance before the output rounding) of x [M, K] . w [N, K]^T in fp64.
    The kernels add K products in chains of at least 32 / 8 products per matrix instruction plus a join of at most 16 partial sums; an fp32 sum of that depth with either rounding of its
    additions is off by less than depth * 2^-23 of the sum of the magnitudes."""
    x, w = x.double(), w.double()
    z, mag = x @ w.t(), x.abs() @ w.abs().t()
    kk = x.shape[1]
    err = (kk / 8 + 64) * 2.0 ** -23 * mag + 2.0 ** -23 * x.abs().sum(1, keepdim=True) * (w.abs().amax(1) if kk else torch.zeros(w.shape[0], dtype=torch.float64))
    if bias is not None:
        z = z + bias.double()
        err = err + 2.0 ** -23 * z.abs()
    if gated:
        n = z.shape[1] // 2
        a, b, ea, eb = z[:, :n], z[:, n:], err[:, :n], err[:, n:]
        s = a * torch.sigmoid(a)
        # |silu'| < 1.1; the exponential, division and products: below 2^-19 of the result
        return s * b, 1.1 * ea * b.abs() + s.abs() * eb + 1.1 * ea * eb + 2.0 ** -19 * (s * b).abs()
    if act is not None:
        z = act(z)
    return z, err


def close(got, want, err, name=""):
    """|got - want| <= half a step of got's type (relative, plus the smallest subnormal) + err; NaN and infinities where wanted"""
    got = got.cpu()
    step = half_step(got.dtype)
    g = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(g), torch.isnan(want)), name
    lim = err + step * (want.abs() + err) + torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    over = want.abs() + lim >= torch.finfo(got.dtype).max            # may round to an infinity
    ok = ((g - want).abs() <= lim) | ~fin | over
    assert ok.all(), "%s: off by %.3g where %.3g is allowed, at %s" % (name, (g - want)[~ok][0], lim[~ok][0], (~ok).nonzero()[0].tolist())


def route(scores, k, renorm):
    """dict of the plan for scores [T, E], by loops"""
    z = torch.as_tensor(scores).double().tolist()
    t, e = scores.shape
    w, ex = torch.zeros(t, k, dtype=torch.float64), torch.full((t, k), -1, dtype=torch.int32)
    for i, row in enumerate(z):
        ok = [j for j in range(e) if row[j] > -float("inf")]
        top = sorted(ok, key=lambda j: (-row[j], j))[:k]
        if not top:
            continue
        m = row[top[0]]
        p = lambda j: 1.0 if row[j] == m else float(np.exp(row[j] - m))  # noqa: E731
        s = sum(p(j) for j in (top if renorm else ok))
        for r, j in enumerate(top):
            ex[i, r], w[i, r] = j, p(j) / s
    flat = ex.flatten().tolist()
    order = [a for j in range(e) for a, b in enumerate(flat) if b == j]
    offsets = [0]
    for j in range(e):
        offsets.append(offsets[-1] + flat.count(j))
    slots = torch.full((t * k,), -1, dtype=torch.int32)
    for s, a in enumerate(order):
        slots[a] = s
    rows = [a // k for a in order] + [-1] * (t * k - len(order))
    return dict(weights=w, experts=ex, offsets=torch.tensor(offsets, dtype=torch.int32), rows=torch.tensor(rows, dtype=torch.int32), slots=slots.view(t, k))
