"""Linear and expert layers, CPU tier: what the entry points refuse (nothing is launched), and the plain forms that the GPU tests compare with."""
import ctypes as C

import pytest
import torch

import mx4ref
from smelter_amd import _native as N
from smelter_amd import ops

F16, BF16, F32, MX4 = 0, 1, 2, 3
P = C.c_void_p(4096)          # an aligned address that no refused call touches


def desc(**k):
    d = dict(M=4, T=4, N=8, K=64, E=1, x_type=F16, w_type=F16, y_type=F16, act=0, slope=0.0, gated=0, x_ld=0, y_ld=0)
    d.update(k)
    return N.LinearDesc(*[d[f[0]] for f in N.LinearDesc._fields_])


def linear(d, x=P, xs=P, w=P, ws=P, bias=None, offsets=None, rows=None, y=P):
    return N.lib().sm_linear_fwd(C.byref(d), x, xs, w, ws, bias, offsets, rows, y, None, 0, None)


def refused(rc, word):
    assert rc == -13 and word in N.lib().smelter_last_error_string().decode(), (rc, N.lib().smelter_last_error_string())


@pytest.mark.parametrize("change, word", [
    (dict(M=-1), "sizes"), (dict(K=-1), "sizes"), (dict(E=0), "sizes"), (dict(M=1 << 31), "beyond"), (dict(N=1 << 30), "beyond"),
    (dict(x_type=F32, w_type=F32), "type"), (dict(x_type=F32), "workspace"), (dict(w_type=BF16), "type"), (dict(x_type=MX4), "type"), (dict(x_type=7), "type"), (dict(y_type=BF16), "output type"), (dict(y_type=MX4), "output type"),
    (dict(act=13), "activation"), (dict(act=-1), "activation"), (dict(gated=1, act=1), "gated"), (dict(E=2), "offsets"), (dict(M=5), "row list"),
    (dict(x_ld=63), "stride"), (dict(y_ld=7), "stride"),
])
def test_linear_refuses(change, word):
    refused(linear(desc(**change)), word)


def test_linear_refuses_operands():
    refused(linear(desc(), x=None), "null")
    refused(linear(desc(), y=None), "null")
    refused(linear(desc(w_type=MX4), ws=None), "null")
    refused(linear(desc(x_type=MX4, w_type=MX4), xs=None), "null")
    refused(linear(desc(), x=C.c_void_p(4097)), "aligned")
    refused(linear(desc(w_type=MX4), w=C.c_void_p(4104)), "16-byte")
    refused(linear(desc(), bias=C.c_void_p(4098)), "aligned")
    refused(N.lib().sm_linear_fwd(None, P, P, P, P, None, None, None, P, None, 0, None), "null")


def test_linear_of_nothing_is_done_at_once():
    assert linear(desc(M=0)) == 0 and linear(desc(N=0)) == 0


def test_quantize_refuses():
    q, dq = N.lib().sm_mx4_quantize, N.lib().sm_mx4_dequantize
    refused(q(P, MX4, 2, 32, 32, P, P, None), "type")
    refused(q(P, F16, -1, 32, 32, P, P, None), "negative")
    refused(q(P, F16, 2, 32, 31, P, P, None), "stride")
    refused(q(None, F16, 2, 32, 32, P, P, None), "null")
    refused(q(P, F16, 2, 32, 32, C.c_void_p(4100), P, None), "alignment")
    refused(q(C.c_void_p(4097), F16, 2, 32, 32, P, P, None), "alignment")
    refused(dq(P, P, 2, 32, P, MX4, 32, None), "type")
    refused(dq(P, P, 2, 32, P, F16, 31, None), "stride")
    refused(dq(P, None, 2, 32, P, F16, 32, None), "null")
    assert q(None, F16, 0, 32, 32, None, None, None) == 0 and dq(None, None, 3, 0, None, F16, 0, None) == 0


def test_route_and_combine_refuse():
    r, c = N.lib().sm_moe_route, N.lib().sm_moe_combine
    ok = dict(type=F32, T=4, E=8, k=2, ld=8)

    def call(ws=0, wsp=None, z=P, off=P, **k):
        a = {**ok, **k}
        return r(z, a["type"], a["T"], a["E"], a["k"], a["ld"], 1, P, P, off, P, P, wsp, ws, None)
    refused(call(type=MX4), "type")
    refused(call(E=0), "experts")
    refused(call(E=1025, ld=1025), "experts")
    refused(call(k=9), "experts")
    refused(call(k=0), "experts")
    refused(call(E=64, ld=64, k=33), "experts")
    refused(call(T=-1), "tokens")
    refused(call(T=1 << 30, k=4), "tokens")
    refused(call(ld=7), "stride")
    refused(call(z=None), "null")
    refused(call(off=None), "null")
    refused(call(T=1000), "workspace")
    refused(c(P, MX4, 4, 8, 8, P, P, 2, 2, P, F16, 8, None), "type")
    refused(c(P, F16, 4, 8, 8, P, P, 2, 2, P, MX4, 8, None), "type")
    refused(c(P, F16, 4, 8, 7, P, P, 2, 2, P, F16, 8, None), "strides")
    refused(c(P, F16, 4, 8, 8, P, P, 2, 2, P, F16, 7, None), "strides")
    refused(c(None, F16, 4, 8, 8, P, P, 2, 2, P, F16, 8, None), "null")
    refused(c(P, F16, -1, 8, 8, P, P, 2, 2, P, F16, 8, None), "sizes")
    assert c(None, F16, 4, 8, 8, None, None, 0, 2, None, F16, 8, None) == 0


def test_python_entry_points_refuse_cpu_tensors():
    x = torch.zeros(2, 64, dtype=torch.float16)
    q = ops.Mx4(*mx4ref.pack(x), 64)
    assert q.shape == (2, 64)
    off = torch.zeros(3, dtype=torch.int32)
    for f in (lambda: ops.mx4_quantize(x), lambda: ops.mx4_dequantize(q), lambda: ops.mx4_linear(x, q), lambda: ops.mx4_linear(x, x), lambda: ops.expert_linear(x, x[None], off),
              lambda: ops.moe_route(x, 2), lambda: ops.moe_combine(x, off[None, :2], x[:1, :2].float())):
        with pytest.raises(N.SmelterError) as e:
            f()
        assert e.value.kind == "invalidArgument"


def test_row_strides():
    a = torch.zeros(4, 6, 8)
    assert ops._rows2d(a, "t") == (24, 8, 8)
    assert ops._rows2d(a[..., :5], "t") == (24, 5, 8)
    assert ops._rows2d(a[:, 0], "t") == (4, 8, 48)
    assert ops._rows2d(a[:1, :1, :3], "t") == (1, 3, 3)
    for bad in (a.transpose(1, 2), a[:, :4], a[..., ::2], a[:1, :1].expand(4, 6, 8)):
        with pytest.raises(N.SmelterError):
            ops._rows2d(bad, "t")


def test_plain_pack_by_hand():
    x = torch.tensor([[0.25, 0.75, -1.25, 1.75, 2.5, -3.5, 5.0, 7.9] + [0.0] * 24])            # ties, and a value above 6 scales
    c, s = mx4ref.pack(x)
    assert s.tolist() == [[127]]
    v = mx4ref.unpack(c, s, 8)
    assert v.tolist() == [[0.0, 1.0, -1.0, 2.0, 2.0, -4.0, 4.0, 6.0]]
    assert c[0, :4].tolist() == [0x20, 0x4a, 0xe4, 0x76]
    c, s = mx4ref.pack(torch.tensor([[1.0] * 32 + [float("nan")] + [2.0]]))
    assert s.tolist() == [[125, 255]] and c[0, 16:].eq(0).all() and mx4ref.unpack(c, s, 34)[0, 32:].isnan().all()
    assert mx4ref.pack(torch.zeros(1, 32))[1].item() == 0


def test_plain_route_by_hand():
    inf = float("inf")
    r = mx4ref.route(torch.tensor([[1.0, 3.0, 3.0, 0.0], [-inf] * 4, [-inf, float("nan"), 2.0, -inf]]), 2, True)
    assert r["experts"].tolist() == [[1, 2], [-1, -1], [2, -1]] and r["weights"].tolist() == [[0.5, 0.5], [0, 0], [1, 0]]
    assert r["offsets"].tolist() == [0, 0, 1, 3, 3] and r["rows"].tolist() == [0, 0, 2, -1, -1, -1] and r["slots"].tolist() == [[0, 1], [-1, -1], [2, -1]]


def test_sizes_that_would_overflow():
    """products of sizes that pass 64 bits are refused, not wrapped"""
    r = N.lib().sm_moe_route
    refused(r(P, F32, (1 << 63) - 1, 8, 2, 8, 1, P, P, P, P, P, P, 1 << 62, None), "tokens")
    refused(r(P, F32, 1 << 62, 8, 4, 8, 1, P, P, P, P, P, P, 1 << 62, None), "tokens")
    q, dq = N.lib().sm_mx4_quantize, N.lib().sm_mx4_dequantize
    refused(q(P, F16, 1 << 40, (1 << 31) - 1, (1 << 31) - 1, P, P, None), "elements")
    refused(dq(P, P, 1 << 40, (1 << 31) - 1, P, F16, (1 << 31) - 1, None), "elements")


def test_scratch_is_asked_for():
    """a product whose K is cut into runs, and fp32 rows, want scratch; a call without it is refused; few rows want none"""
    size = N.lib().sm_linear_workspace_bytes
    cut = desc(M=64, T=64, N=2048, K=8192)
    assert size(C.byref(cut), 0, 0) % (64 * 2048 * 4) == 0 and size(C.byref(cut), 0, 0) > 0
    refused(linear(cut), "workspace")
    assert size(C.byref(desc(M=16, T=16, N=2048, K=8192)), 0, 0) == 0
    wide = desc(M=4, T=4, N=8, K=64, x_type=F32)
    assert size(C.byref(wide), 1, 0) >= 2 * 4 * (64 * 2 + 8 * 4)
    refused(linear(wide), "workspace")
    refused(linear(desc(M=1 << 30, T=1 << 30, x_type=F32)), "fp32 rows")


def test_more_threads_than_one_launch_holds():
    """2^32 threads and more: refused by name before anything is launched"""
    refused(linear(desc(M=1 << 20, T=1 << 20, N=1 << 24, K=8)), "one launch")
    refused(linear(desc(M=1 << 20, T=1 << 20, N=1 << 16, K=8, E=1 << 17), offsets=P), "one launch")
    refused(linear(desc(M=1 << 20, T=1 << 20, N=1 << 24, K=7)), "one launch")
