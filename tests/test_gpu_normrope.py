"""dxh_normrope and dxh_normrope_backward against the formulas in 64 bits.

Bars, with u = 2^-24 and e_T half a step of the result's type (bf16 2^-8, f16 2^-11 with its smallest step 2^-25, f32 2^-24), V <= 8 values a lane:
  r = rsqrt(mean(x^2) + eps): the sum is V fused adds and at most 6 shuffle adds of positive terms, one product, one add: its relative
  error is at most (V + 8) u, half of that in r, plus 2 u of v_rsq_f32 (one step): under 10 u.
  forward: n = x (r w): 12 u.  y = n_a c + n_b s: |dy| <= (|n_a c| + |n_b s|) 15 u, and e_T |y| for the rounding.
  dx = r (g w) - r x k, k = mean(h x) r^2: g has (|a c| + |b s|) 3 u; the sum over D terms of either sign has an error of (V + 12) u times the sum
  of their magnitudes; r and k carry 10 u and 20 u: |d| <= 60 u (r sum-of-magnitudes form) below, and e_T |dx|.
  dw: f32 sums of N terms of either sign in a tree of depth at most (terms a lane) + 64 + 32: (depth + 30) u times the sum of magnitudes.
"""
import ctypes as C

import numpy as np
import pytest
import torch

from deepx_amd import lib as dx

pytestmark = pytest.mark.gpu
DT = {"f32": (dx.F32, torch.float32, 2.0 ** -24, 2.0 ** -149), "f16": (dx.F16, torch.float16, 2.0 ** -11, 2.0 ** -25), "bf16": (dx.BF16, torch.bfloat16, 2.0 ** -8, 2.0 ** -133)}
U = 2.0 ** -24


def heads(t):
    return dx.Heads(t.data_ptr(), t.stride(0), t.stride(1))


def tables(rows, rd, seed):
    g = torch.Generator().manual_seed(seed)
    a = torch.rand(max(rows, 1), max(rd // 2, 1), generator=g, dtype=torch.float64) * 6.3
    return a.cos().float().cuda(), a.sin().float().cuda()


def pairs(rd, inter, dim):
    """for every element its partner and the sign of the partner's product; itself past rd"""
    j = torch.arange(dim)
    if inter:
        partner, sign, idx = torch.where(j % 2 == 0, j + 1, j - 1), torch.where(j % 2 == 0, -1.0, 1.0), j // 2
    else:
        partner, sign, idx = torch.where(j < rd // 2, j + rd // 2, j - rd // 2), torch.where(j < rd // 2, -1.0, 1.0), torch.where(j < rd // 2, j, j - rd // 2)
    past = j >= rd
    return torch.where(past, j, partner), torch.where(past, 0.0, sign).double(), torch.where(past, 0, idx), past


def rotated(n, cos, sin, p, rd, inter, back=False):
    """(result, magnitude) of the rotation in 64 bits"""
    dim = n.shape[-1]
    if rd == 0:
        return n, n.abs()
    partner, sign, idx, past = pairs(rd, inter, dim)
    c = torch.where(past, 1.0, cos.cpu().double()[p][:, idx])[:, None]
    s = torch.where(past, 0.0, sin.cpu().double()[p][:, idx])[:, None] * sign * (-1 if back else 1)
    other = n[..., partner]
    other = torch.where(past, torch.zeros_like(other), other)
    return n * c + other * s, (n * c).abs() + (other * s).abs()


def ref_forward(x, w, cos, sin, p, rd, inter, eps, norm):
    x = x.cpu().double()
    if norm:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (1.0 if w is None else w.cpu().double())
    return rotated(x, cos, sin, p, rd, inter)


def ref_backward(x, dy, w, cos, sin, p, rd, inter, eps, norm):
    """(dx, bound on its fp32 error in units of u, dw, sum of magnitudes of dw)"""
    x, dy = x.cpu().double(), dy.cpu().double()
    g, mg = rotated(dy, cos, sin, p, rd, inter, back=True)
    if not norm:
        return g, mg, None, None
    r = 1 / (x.square().mean(-1, keepdim=True) + eps).sqrt()
    ww = torch.ones(x.shape[-1], dtype=torch.float64) if w is None else w.cpu().double()
    h, mh = g * ww, mg * ww.abs()
    dxv = r * h - x * r ** 3 * (h * x).mean(-1, keepdim=True)
    mag = r * mh + x.abs() * r ** 3 * (mh * x.abs()).mean(-1, keepdim=True)
    return dxv, mag, (g * x * r).sum((0, 1)), (mg * x.abs() * r).sum((0, 1))


def run_forward(L, dt, xs, outs, ws, wdt, norms, rows, dim, eps, rot):
    parts = (dx.NormropePart * len(xs))(*[dx.NormropePart(heads(x), heads(o), dx.Heads(), w.data_ptr() if w is not None else None, None, x.shape[1], n, wdt)
                                          for x, o, w, n in zip(xs, outs, ws, norms)])
    dx.check(L.dxh_normrope(dt, parts, len(xs), rows, dim, eps, rot, torch.cuda.current_stream().cuda_stream), "normrope")


SHAPES = [  # rows, q heads, k heads, dim, rotary, interleaved
    (1, 1, 1, 16, 16, False), (8, 14, 2, 64, 64, False), (8, 14, 2, 64, 64, True), (3, 5, 1, 80, 80, False), (7, 3, 3, 96, 48, False), (33, 7, 1, 112, 6, False),
    (5, 2, 1, 128, 34, True), (2, 9, 3, 256, 256, False), (300, 40, 8, 128, 128, False), (1031, 3, 1, 48, 44, False), (65, 4, 4, 32, 0, False), (4097, 14, 2, 64, 32, True),
    (1, 64, 64, 128, 128, False)]


@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward(dxh, name, shape):
    rows, hq, hk, dim, rd, inter = shape
    dt, tt, et, tiny = DT[name]
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + dim)
    qkv = (torch.randn(rows, (hq + 2 * hk) * dim, generator=g, device="cuda") * 3).to(tt)  # q and k are views of one product's rows
    q, k = qkv[:, :hq * dim].view(rows, hq, dim), qkv[:, hq * dim:(hq + hk) * dim].view(rows, hk, dim)
    wf32 = dim % 32 == 0  # weights of the tensors' type and in 32 bits
    wq = torch.randn(dim, generator=g, device="cuda").to(torch.float32 if wf32 else tt)
    cos, sin = tables(97, rd, dim)
    pdt = torch.int64 if rows % 2 else torch.int32
    pos = torch.randint(-3, 100, (rows,), generator=g, device="cuda", dtype=pdt)  # some outside the table
    p = pos.cpu().long().clamp(0, 96)
    rot = dx.Rotary(cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), 97, rd, int(inter), dx.I64 if rows % 2 else dx.I32)
    for norms in ((1, 1), (1, 0)):
        oq, ok = torch.full_like(q, 7.0).contiguous(), torch.full_like(k, 7.0).contiguous()
        run_forward(dxh, dt, [q, k], [oq, ok], [wq, None], dx.F32 if wf32 else dt, norms, rows, dim, 1e-6, rot)
        for x, o, w, n in ((q, oq, wq, norms[0]), (k, ok, None, norms[1])):
            want, mag = ref_forward(x, w, cos, sin, p, rd, inter, 1e-6, n)
            err = (o.cpu().double() - want).abs()
            assert (err <= mag * 15 * U + want.abs() * et * (1 + 2 ** -10) + tiny).all(), (err / (mag * 15 * U + want.abs() * et + tiny)).max()


@pytest.mark.parametrize("name", list(DT))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_backward(dxh, name, shape):
    rows, hq, hk, dim, rd, inter = shape
    dt, tt, et, tiny = DT[name]
    g = torch.Generator(device="cuda").manual_seed(rows * 7 + dim + 1)
    n = lambda h: torch.randn(rows, h, dim, generator=g, device="cuda").to(tt)  # noqa: E731
    q, k, dq, dk = n(hq), n(hk), n(hq), n(hk)
    wq = torch.randn(dim, generator=g, device="cuda").to(tt)
    cos, sin = tables(rows, rd, dim)
    rot = dx.Rotary(cos.data_ptr(), sin.data_ptr(), None, rows, rd, int(inter), dx.I32)  # no positions: the row's number
    p = torch.arange(rows)
    for norms in ((1, 1), (0, 1)):
        oq, ok = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
        dws = torch.full((2, dim), 7.0, device="cuda")
        parts = (dx.NormropePart * 2)(dx.NormropePart(heads(q), heads(dq), heads(oq), wq.data_ptr(), dws[0].data_ptr(), hq, norms[0], dt),
                                      dx.NormropePart(heads(k), heads(dk), heads(ok), None, dws[1].data_ptr(), hk, norms[1], dt))
        need = C.c_size_t(0)
        dx.check(dxh.dxh_normrope_backward_workspace_bytes(dt, parts, 2, rows, dim, C.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device="cuda")
        results = []
        for _ in range(2):  # the same bits twice
            dx.check(dxh.dxh_normrope_backward(dt, parts, 2, rows, dim, 1e-6, rot, ws.data_ptr(), need.value, torch.cuda.current_stream().cuda_stream), "backward")
            results.append([t.cpu().clone() for t in (oq, ok, dws)])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        for i, (x, dy, o, w, nn, h) in enumerate(((q, dq, oq, wq, norms[0], hq), (k, dk, ok, None, norms[1], hk))):
            want, mag, dw, mw = ref_backward(x, dy, w, cos, sin, p, rd, inter, 1e-6, nn)
            err = (o.cpu().double() - want).abs()
            assert (err <= mag * 60 * U + want.abs() * et * (1 + 2 ** -10) + tiny).all(), (err / (mag * 60 * U + want.abs() * et + tiny)).max()
            if nn:
                depth = rows * h / 256 + h + 4 + 64 + 32
                err = (dws[i].cpu().double() - dw).abs()
                assert (err <= mw * (depth + 30) * U).all(), (err / (mw * (depth + 30) * U)).max()
            else:
                assert (dws[i].cpu() == 7.0).all()  # without a norm there is no weight to have a gradient


def test_gradient_against_differences(dxh):
    """<dx, a> + <dw, b> of the kernel against the central difference of sum(y dy) of the 64-bit forward along (a, b).  The difference's own error is
    h^2 times a third derivative (h = 1e-4: under 1e-6 of the value's scale here), the kernel's under 1e-5 of the sum of magnitudes."""
    rows, h, dim, rd = 37, 5, 64, 48
    g = torch.Generator(device="cuda").manual_seed(11)
    n = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    x, dy, w = n(rows, h, dim), n(rows, h, dim), n(dim)
    cos, sin = tables(rows, rd, 1)
    out, dw, ws = torch.empty_like(x), torch.empty(dim, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    rot = dx.Rotary(cos.data_ptr(), sin.data_ptr(), None, rows, rd, 0, dx.I32)
    parts = (dx.NormropePart * 1)(dx.NormropePart(heads(x), heads(dy), heads(out), w.data_ptr(), dw.data_ptr(), h, 1, dx.F32))
    dx.check(dxh.dxh_normrope_backward(dx.F32, parts, 1, rows, dim, 1e-6, rot, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    for t in range(3):
        a, b = n(rows, h, dim).cpu().double(), n(dim).cpu().double()
        loss = lambda e: (ref_forward(x.cpu().double() + e * a, w.cpu().double() + e * b, cos, sin, torch.arange(rows), rd, False, 1e-6, 1)[0] * dy.cpu().double()).sum()  # noqa: E731, B023
        want = (loss(1e-4) - loss(-1e-4)) / 2e-4
        terms = torch.cat([(out.cpu().double() * a).flatten(), dw.cpu().double() * b])
        assert abs(terms.sum() - want) <= 1e-5 * terms.abs().sum()


def test_in_place_strides_streams_and_graphs(dxh):
    rows, h, dim = 129, 6, 96
    g = torch.Generator(device="cuda").manual_seed(5)
    cos, sin = tables(rows, dim, 2)
    rot = dx.Rotary(cos.data_ptr(), sin.data_ptr(), None, rows, dim, 0, dx.I32)
    x = torch.randn(rows, h, dim, generator=g, device="cuda").bfloat16()
    w = torch.randn(dim, generator=g, device="cuda").bfloat16()
    want = torch.empty_like(x)
    run_forward(dxh, dx.BF16, [x], [want], [w], dx.BF16, [1], rows, dim, 1e-5, rot)
    # [heads, rows, dim] views, in and out
    xt, ot = x.transpose(0, 1).contiguous().transpose(0, 1), torch.empty(h, rows, dim, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
    run_forward(dxh, dx.BF16, [xt], [ot], [w], dx.BF16, [1], rows, dim, 1e-5, rot)
    assert torch.equal(ot, want)
    # in place, on a stream of its own, recorded and replayed with other work between
    st = C.c_void_p()
    dx.check(dxh.dxh_stream_create(C.byref(st)))
    y, graph = x.clone(), C.c_void_p()
    torch.cuda.synchronize()
    part = (dx.NormropePart * 1)(dx.NormropePart(heads(y), heads(y), dx.Heads(), w.data_ptr(), None, h, 1, dx.BF16))
    dx.check(dxh.dxh_graph_begin_capture(st))
    dx.check(dxh.dxh_normrope(dx.BF16, part, 1, rows, dim, 1e-5, rot, st))
    dx.check(dxh.dxh_graph_end_capture(st, C.byref(graph)))
    for _ in range(3):
        y.copy_(x)
        run_forward(dxh, dx.BF16, [x], [ot], [w], dx.BF16, [1], rows, dim, 1e-5, rot)
        torch.cuda.synchronize()
        dx.check(dxh.dxh_graph_launch(graph, st))
        dx.check(dxh.dxh_stream_sync(st))
        assert torch.equal(y, want)
    dx.check(dxh.dxh_graph_destroy(graph))
    dx.check(dxh.dxh_stream_destroy(st))


@pytest.mark.parametrize("inter", [False, True])
def test_values_past_the_rotation_pass_unchanged(dxh, inter):
    """without a norm, what is not rotated is copied: infinities, NaN and the sign of zero among them"""
    rows, h, dim, rd = 5, 3, 64, 24
    x = torch.randn(rows, h, dim, device="cuda")
    x[..., rd:rd + 4] = torch.tensor([float("inf"), float("-inf"), -0.0, float("nan")], device="cuda")
    cos, sin = tables(rows, rd, 3)
    y = torch.empty_like(x)
    run_forward(dxh, dx.F32, [x], [y], [None], dx.F32, [0], rows, dim, 0.0, dx.Rotary(cos.data_ptr(), sin.data_ptr(), None, rows, rd, int(inter), dx.I32))
    assert np.array_equal(y[..., rd:].cpu().numpy().view(np.int32), x[..., rd:].cpu().numpy().view(np.int32))
    assert torch.isfinite(y[..., :rd]).all()


def test_zero_and_extreme_rows(dxh):
    """a head of zeros stays zero (eps > 0); heads of very large and very small values keep finite norms"""
    x = torch.zeros(4, 1, 64, device="cuda")
    x[1], x[2], x[3] = 1e18, 1e-18, torch.linspace(-1, 1, 64, device="cuda")
    y = torch.empty_like(x)
    run_forward(dxh, dx.F32, [x], [y], [None], dx.F32, [1], 4, 64, 1e-6, None)
    assert (y[0] == 0).all() and torch.allclose(y[1], torch.ones_like(y[1]), rtol=1e-6) and torch.allclose(y[2], x[2] * 1e3, rtol=1e-6)


def test_nothing_to_do(dxh):
    dw = torch.full((64,), 7.0, device="cuda")
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    part = (dx.NormropePart * 1)(dx.NormropePart(dx.Heads(), dx.Heads(), dx.Heads(), None, dw.data_ptr(), 3, 1, dx.F32))
    dx.check(dxh.dxh_normrope(dx.F32, part, 1, 0, 64, 1e-6, None, None))
    dx.check(dxh.dxh_normrope_backward(dx.F32, part, 1, 0, 64, 1e-6, None, ws.data_ptr(), ws.numel(), None))
    torch.cuda.synchronize()
    assert (dw == 0).all()  # the sum over no rows


@pytest.mark.parametrize("name", ["f32", "bf16"])
def test_squares_below_the_smallest_normal_float(dxh, name):
    """eps 0 and heads whose mean square is subnormal: x^2 is exact to half of 2^-149, the mean of x = 2^-63 ... 2^-70 is 2^-126 ... 2^-140, so the sum is off by
    at most a part in 2^9 there (2^-140 in steps of 2^-149) and the root by half of that; gradients: dx ~ 1 / |x| in fp32"""
    dt, tt, et, _ = DT[name]
    e = torch.arange(60, 71, dtype=torch.float32, device="cuda")
    sign = torch.where(torch.arange(64, device="cuda") % 3 == 0, -1.0, 1.0)
    x = (2.0 ** -e[:, None, None] * sign).to(tt)
    y, dxv = torch.empty_like(x), torch.empty_like(x)
    run_forward(dxh, dt, [x], [y], [None], dt, [1], 11, 64, 0.0, None)
    assert ((y.float() - sign).abs() <= 2.0 ** -9 + et).all()
    dy = torch.randn(11, 1, 64, generator=torch.Generator(device="cuda").manual_seed(2), device="cuda").to(tt)
    dw, ws = torch.empty(64, device="cuda"), torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    part = (dx.NormropePart * 1)(dx.NormropePart(heads(x), heads(dy), heads(dxv), None, dw.data_ptr(), 1, 1, dt))
    dx.check(dxh.dxh_normrope_backward(dt, part, 1, 11, 64, 0.0, None, ws.data_ptr(), ws.numel(), torch.cuda.current_stream().cuda_stream))
    want, mag, dwant, dmag = ref_backward(x, dy, None, None, None, None, 0, False, 0.0, 1)
    assert ((dxv.cpu().double() - want).abs() <= mag * 4 * 2.0 ** -9 + want.abs() * et).all()
    assert ((dw.cpu().double() - dwant).abs() <= dmag * 2.0 ** -9).all()
