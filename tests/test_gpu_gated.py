"""``ops.ternary_gated_linear``: ``silu(gate(x)) * up(x)`` on full-precision masters and its gradient, against 64 bits.

The 16-bit gradient has an operand of its own, ``G`` (the gradient of both projections times their scales, rounded to 16 bits): it is
checked element by element against the formula, and both products against 64-bit products of that very ``G``.
"""
import math

import pytest
import torch

from conftest import announce

U = 2.0 ** -24
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# rows, K, F: one of each; odd ones; halves that fill no tile, a last stage of the contraction, both sides of 64 and 128 rows, a contraction
# long enough for two groups of waves
# a feature too long for the registers of a wave
SHAPES = [(1, 8, 2), (3, 1, 1), (3, 7, 5), (2, 3, 9), (5, 1, 24), (1, 640, 48), (17, 100, 37), (64, 512, 256), (65, 1001, 33), (129, 520, 272), (300, 1100, 546),
          (40, 2560, 688), (1000, 264, 520), (35, 4096, 64), (33, 4093, 40), (9, 5003, 20),
          (20, 8192, 48), (17, 8200, 33)]


def _gated(*args, **kwargs):
    from bittorch_amd import ops
    return ops.ternary_gated_linear(*args, **kwargs)


def _inputs(rows, k, f, dt, wt=None, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed * 977 + rows * 31 + k * 7 + f)
    mk = lambda std, *shape: torch.randn(*shape, generator=g) * std
    wt = wt or dt
    x, wg, wu, dh = mk(1, rows, k).to(dt), mk(0.05, f, k).to(wt), mk(0.05, f, k).to(wt), mk(0.1, rows, f).to(dt)
    bg, bu = (mk(0.3, f).to(wt), mk(0.3, f).to(wt)) if bias else (None, None)
    return [None if t is None else t.cuda() for t in (x, wg, wu, bg, bu, dh)]


def _ternary(w, threshold_factor=0.05, per_channel=True):
    from bittorch_amd.quant import ternary_quantize
    q, s = ternary_quantize(w.detach().cpu(), threshold_factor, per_channel)
    return q.double().cuda(), s.double().reshape(-1).expand(w.shape[0]).cuda()


class _Reference:
    """The operator in 64 bits, with what fp32 evaluation may add to each value."""

    def __init__(self, x, wg, wu, bg, bu, dh, **quant):
        (self.tg, self.ag), (self.tu, self.au) = _ternary(wg, **quant), _ternary(wu, **quant)
        dt, x, dh, k = x.dtype, x.detach().double(), dh.double(), x.shape[1]
        self.x, self.dh = x, dh
        zero = torch.zeros(wg.shape[0], dtype=torch.float64, device=x.device)
        bg, bu = (zero if b is None else b.detach().double() for b in (bg, bu))
        g, u = x @ self.tg.t() * self.ag + bg, x @ self.tu.t() * self.au + bu
        # A product of K terms: in the matrix cores 32 of them at a time, K / 32 sums one after the other (twice that where K is split),
        # each rounded by at most one step; scale and bias once each.  fp32 rows: three 16-bit terms a value, so three times the sums, and
        # half a step of the value in the third.
        chain = U * 2 * (3 * k / 32 + 40)
        self.tol_g = chain * (x.abs() @ self.tg.abs().t()) * self.ag + 4 * U * (g.abs() + bg.abs())
        self.tol_u = chain * (x.abs() @ self.tu.abs().t()) * self.au + 4 * U * (u.abs() + bu.abs())
        sig = 1 / (1 + torch.exp(-g))
        self.g, self.u, silu = g, u, g * sig
        self.h, self.sig = silu * u, sig
        # silu' lies within -0.1 and 1.1; exp's argument is rounded (|g| U of the result), exp, the sum, the reciprocal, two products
        self.tol_h = 1.1 * u.abs() * self.tol_g + silu.abs() * self.tol_u + (g.abs() + 16) * U * self.h.abs()
        if dt != torch.float32:  # (the gradient reads g and u in 24 bits: half a step is 2^-16 of a value)
            self.tol_g, self.tol_u = self.tol_g + 2.0 ** -16 * g.abs(), self.tol_u + 2.0 ** -16 * u.abs()
        self.follow()

    def follow(self):
        dh, g, u, sig = self.dh, self.g, self.u, self.sig
        silu, slope = g * sig, sig * (1 + g * (1 - sig))
        self.dg, self.du = dh * u * slope, dh * silu
        # |silu''| is at most 1/2; 1 - sig is off by a step of 1, which g multiplies
        self.tol_dg = dh.abs() * (slope.abs() * self.tol_u + 0.5 * u.abs() * self.tol_g + u.abs() * sig * (3 * g.abs() + 16) * U)
        self.tol_du = dh.abs() * (1.1 * self.tol_g + silu.abs() * (g.abs() + 16) * U)


def _assert_within(got, want, tol, what):
    half, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps
    off = (got.double() - want).abs() - (tol + half * (want.abs() + tol) + tiny)
    assert bool((off <= 0).all()), f"{what}: {float(off.max())} over its bound"


def _norm_error(got, want):
    got = got.detach()
    return float((got.double() - want).norm() / want.norm().clamp(min=1e-300))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("rows,k,f", SHAPES)
def test_forward_and_gradient(rows, k, f, dt):
    announce("gated", rows, k, f, dt)
    x, wg, wu, bg, bu, dh = _inputs(rows, k, f, dt)
    ref = _Reference(x, wg, wu, bg, bu, dh)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = _gated(*leaves)
    assert h.shape == (rows, f) and h.dtype == dt
    _assert_within(h.detach(), ref.h, ref.tol_h, "h")
    with torch.no_grad():
        alone = _gated(*leaves)
        if rows > 1:
            assert torch.equal(alone, h)
        else:  # straight from the masters: other sums, the same bound
            _assert_within(alone, ref.h, ref.tol_h, "h without a gradient")
    dx, dwg, dwu, dbg, dbu = torch.autograd.grad(h, leaves, dh, retain_graph=True)
    again = torch.autograd.grad(h, leaves, dh)
    assert all(torch.equal(a, b) and a.is_contiguous() for a, b in zip(again, (dx, dwg, dwu, dbg, dbu)))
    assert dx.shape == x.shape and dwg.shape == wg.shape and dbu.shape == bu.shape and {t.dtype for t in again} == {dt}
    # the sums of the biases: `rows` additions at most, in fp32, before they are rounded
    for got, v, tol in ((dbg, ref.dg, ref.tol_dg), (dbu, ref.du, ref.tol_du)):
        _assert_within(got, v.sum(0), tol.sum(0) + U * (rows + 4) * v.abs().sum(0), "bias")
    # both products: each term's own error, and where rows are 16-bit half a step of G
    half = 0.0 if dt == torch.float32 else torch.finfo(dt).eps / 2
    chain = lambda n: U * 2 * (3 * n / 32 + 80)
    parts = [(ref.dg, ref.tol_dg, ref.ag, ref.tg), (ref.du, ref.tol_du, ref.au, ref.tu)]
    tiny = 0.0 if dt == torch.float32 else torch.finfo(dt).smallest_normal * half
    want = sum((v * a) @ t for v, _, a, t in parts)
    tol = sum(((tol * (1 + half) + (half + chain(2 * f)) * v.abs()) * a + tiny) @ t.abs() for v, tol, a, t in parts)
    _assert_within(dx, want, tol, "dx")
    for got, (v, tol, a, _) in zip((dwg, dwu), parts):
        want_w = ((v * a).t() @ ref.x)
        tol_w = ((tol * (1 + half) + (half + chain(rows)) * v.abs()) * a + tiny).t() @ ref.x.abs()
        _assert_within(got, want_w, tol_w, "dW")
        if dt != torch.float32 and rows * k >= 64:
            # two roundings of at most half a step, independent of each other and of their neighbours': their root of squares
            # (1.42 halves), the largest they could be in every single place
            assert _norm_error(got, want_w) <= 1.42 * half
    if dt != torch.float32 and rows * k >= 64:
        assert _norm_error(dx, want) <= 1.42 * half and _norm_error(h.detach(), ref.h) <= 1.01 * half


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wt", [(d, d) for d in DTYPES] + [(torch.bfloat16, torch.float32), (torch.float32, torch.float16)])
@pytest.mark.parametrize("rows,k,f", [(1, 8, 1), (1, 15, 3), (1, 1024, 9), (1, 1025, 40), (1, 2560, 16), (1, 2559, 70), (1, 2561, 33), (1, 4096, 33),
                                      (1, 4097, 16), (2, 64, 16), (1, 7, 16), (1, 1000, 20000)])
def test_one_row_without_a_gradient(rows, k, f, dt, wt):
    """The row that is multiplied as the masters are read, and the calls next to it that are not."""
    announce("gated masters", rows, k, f, dt, wt)
    from bittorch_amd import _C
    for bias in (True, False):
        x, wg, wu, bg, bu, dh = _inputs(rows, k, f, dt, wt, bias, seed=11)
        assert _C.gated_masters_serves(rows, wg) == (rows == 1 and k >= 8 and (k <= 2560 or (k <= 4096 and k % 8 == 0 and wt != torch.float32)))
        assert not _C.gated_masters_serves(rows, wg, False)
        wg[0] = 0
        ref = _Reference(x, wg, wu, bg, bu, dh)
        h = _gated(x, wg, wu, bg, bu)
        # (a lane adds up to 8 (K / 512 + 1) products one after the other here, then over the lanes: within the bound's 6 K / 32 + 80)
        _assert_within(h, ref.h, ref.tol_h, "h")
        assert torch.equal(h, _gated(x, wg, wu, bg, bu))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k,f", [(33, 264, 48), (300, 1100, 546), (257, 512, 1000)])
def test_stages_of_the_16_bit_gradient(rows, k, f, dt):
    announce("gated stages", rows, k, f, dt)
    from bittorch_amd import _C
    x, wg, wu, bg, bu, dh = _inputs(rows, k, f, dt, seed=1)
    ref = _Reference(x, wg, wu, bg, bu, dh)
    fp = (f + 15) // 16 * 16
    w, w_back, scale, bias = _C.gated_weights(wg, wu, bg, bu, back=True)
    h, pre, read = _C.ternary_gated_forward(x, w, scale, bias, f, True)
    assert torch.equal(h, _C.ternary_gated_forward(x, w, scale, bias, f)[0])
    assert torch.equal(read, torch.nn.functional.pad(x, (0, -k % 8)))
    # 24 bits a value: g, g, u, u of two columns in three dwords
    b = pre.view(torch.uint8).reshape(rows, fp // 2, 4, 3).to(torch.int32)
    pairs = (b[..., 0] << 8 | b[..., 1] << 16 | b[..., 2] << 24).view(torch.float32).reshape(rows, fp // 2, 2, 2)
    for n, (v, tol, what) in enumerate(((ref.g, ref.tol_g, "g"), (ref.u, ref.tol_u, "u"))):
        _assert_within(pairs[:, :, n].reshape(rows, fp)[:, :f], v, tol, what)
    g, db = _C.gated_grad(dh, pre, scale, torch.float32)
    assert g.shape == (rows, 2 * fp) and not g[:, f:fp].any() and not g[:, fp + f:].any()
    _assert_within(g[:, :f], ref.dg * ref.ag, ref.tol_dg * ref.ag, "G gate")
    _assert_within(g[:, fp:fp + f], ref.du * ref.au, ref.tol_du * ref.au, "G up")
    assert torch.equal(g, _C.gated_grad(dh, pre, scale)[0])
    # the copy for the input's gradient holds the codes' transpose: a product of a unit row reads one feature's weights
    eye = torch.zeros(2 * f, 2 * fp, dtype=dt, device="cuda")
    eye[torch.arange(f), torch.arange(f)] = 1
    eye[torch.arange(f) + f, torch.arange(f) + fp] = 1
    rows_of = _C.ternary_linear_tiled_forward(eye, w_back, scale[2 * fp:], None, 2 * fp, k)
    assert torch.equal(rows_of.double(), torch.cat((ref.tg, ref.tu)))
    dx = _C.ternary_linear_tiled_forward(g, w_back, scale[2 * fp:], None, 2 * fp, k)
    g64 = g.double()
    codes = torch.zeros(2 * fp, k, dtype=torch.float64, device="cuda")
    codes[:f], codes[fp:fp + f] = ref.tg, ref.tu
    _assert_within(dx, g64 @ codes, U * 2 * (2 * fp / 32 + 80) * (g64.abs() @ codes.abs()), "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wt", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.float32, torch.bfloat16),
                                   (torch.bfloat16, torch.float16)])
def test_masters_of_another_dtype(dt, wt):
    x, wg, wu, bg, bu, dh = _inputs(70, 264, 80, dt, wt, seed=2)
    ref = _Reference(x, wg, wu, bg, bu, dh)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = _gated(*leaves)
    _assert_within(h.detach(), ref.h, ref.tol_h, "h")
    grads = torch.autograd.grad(h, leaves, dh)
    assert [t.dtype for t in grads] == [dt, wt, wt, wt, wt]
    eps = max(torch.finfo(d).eps for d in (dt, wt))
    want = [(ref.dg * ref.ag) @ ref.tg + (ref.du * ref.au) @ ref.tu, (ref.dg * ref.ag).t() @ ref.x, (ref.du * ref.au).t() @ ref.x,
            ref.dg.sum(0), ref.du.sum(0)]
    for got, w in zip(grads, want):  # up to three roundings to 16 bits: G, the product, the masters' dtype
        assert _norm_error(got, w) <= 1.74 * eps / 2 + 1e-5


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_quantizer_settings_and_rows_without_weights(dt):
    x, wg, wu, _, _, dh = _inputs(20, 128, 40, dt, bias=False, seed=3)
    wg[3], wu[5] = 0, 0
    wg[4, 1:] = 0
    for quant in (dict(threshold_factor=0.7), dict(threshold_factor=0.0), dict(per_channel=False), dict(threshold_factor=0.5, per_channel=False)):
        ref = _Reference(x, wg, wu, None, None, dh, **quant)
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu)]
        h = _gated(*leaves, **quant)
        _assert_within(h.detach(), ref.h, ref.tol_h, quant)
        dx, dwg, dwu = torch.autograd.grad(h, leaves, dh)
        # (the third: a 16-bit master's scale of 1e-8 is 0 or a rounded 1e-8; those rows are too small to matter in a norm)
        half = torch.finfo(dt).eps / 2
        assert _norm_error(dx, (ref.dg * ref.ag) @ ref.tg + (ref.du * ref.au) @ ref.tu) <= 1.42 * half + 2e-6
        assert _norm_error(dwg, (ref.dg * ref.ag).t() @ ref.x) <= 1.42 * half + 2e-6


@pytest.mark.gpu
def test_projections_beyond_two_to_the_31_dwords():
    """70000 rows of 22000 features: the kept projections pass 2^31 dwords and 2^33 bytes, G 2^31 elements."""
    announce("gated", 70000, 64, 22000)
    from bittorch_amd import _C
    rows, k, f = 70000, 64, 22000
    g = torch.Generator().manual_seed(13)
    wg, wu = ((torch.randn(f, k, generator=g) * 0.05).bfloat16().cuda() for _ in range(2))
    pick = [0, 1, 34999, 65535, 65536, rows - 2, rows - 1]
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    x[pick] = torch.randn(7, k, generator=g).bfloat16().cuda()
    w, w_back, scale, _ = _C.gated_weights(wg, wu, back=True)
    h, pre, _ = _C.ternary_gated_forward(x, w, scale, None, f, True)
    few_h, few_pre, _ = _C.ternary_gated_forward(x[pick], w, scale, None, f, True)  # (one stage of k: the same sums in tiles of any size)
    assert torch.equal(h[pick], few_h) and torch.equal(pre[pick], few_pre) and not h[2:34999].any()
    dh = torch.zeros_like(h)
    dh[pick] = torch.randn(7, f, generator=g).bfloat16().cuda()
    grad, db = _C.gated_grad(dh, pre, scale, torch.float32)
    few, few_db = _C.gated_grad(dh[pick], few_pre, scale, torch.float32)
    assert torch.equal(grad[pick], few) and not grad[2:34999].any()
    # (seven terms other than zero, added in another order)
    assert bool(((db - few_db).abs() <= 8 * U * 7 * few_db.abs().clamp(min=dh.abs().max().float())).all())


@pytest.mark.gpu
def test_parts_of_the_call():
    """One bias, one leaf, one master twice, and inputs that lie in other ways."""
    x, wg, wu, bg, bu, dh = _inputs(48, 264, 72, torch.bfloat16, seed=4)
    full = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    want = torch.autograd.grad(_gated(*full), full, dh)
    for n in range(5):
        args = [t.detach() for t in full]
        args[n].requires_grad_()
        got, = torch.autograd.grad(_gated(*args), args[n], dh)
        assert torch.equal(got, want[n]), n
    for args in ((x, wg, wu, bg, None), (x, wg, wu, None, bu), (x, wg, wu, None, None)):
        ref = _Reference(*args, dh)
        _assert_within(_gated(*args), ref.h, ref.tol_h, "one bias")
    ref = _Reference(x, wg, wg, None, None, dh)
    w = wg.clone().requires_grad_()
    twice, = torch.autograd.grad(_gated(x, w, w), w, dh)
    assert _norm_error(twice, (ref.dg * ref.ag + ref.du * ref.au).t() @ ref.x) <= 2 * torch.finfo(torch.bfloat16).eps / 2
    # leading dimensions, columns before rows, rows inside a wider matrix, an odd start, strided and expanded gradients and masters
    h = _gated(*[t.detach() for t in full])
    wide = torch.randn(48, 264 * 2 + 1, device="cuda").bfloat16()
    wide[:, 1:265] = x
    flat = torch.zeros(48 * 264 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(48, 264).copy_(x)
    for other in (x.reshape(6, 8, 264), x.t().contiguous().t(), wide[:, 1:265], flat):
        o = other.detach().requires_grad_()
        out = _gated(o, wg.t().contiguous().t(), wu, bg, bu)
        assert out.shape == (*o.shape[:-1], 72) and torch.equal(out.reshape(48, 72), h)
        grad, = torch.autograd.grad(out, o, dh.reshape(out.shape))
        assert torch.equal(grad.reshape(48, 264), want[0])
    one = _gated(x[5], wg, wu, bg, bu)
    assert one.shape == (72,) and torch.equal(one, _gated(x[5:6], wg, wu, bg, bu)[0])
    odd = torch.zeros(2 * 72 * 264 + 1, dtype=torch.bfloat16, device="cuda")[1:].view(2, 72, 264).copy_(torch.stack((wg, wu)))
    assert torch.equal(_gated(x[5], odd[0], odd[1], bg, bu), one) and torch.equal(_gated(x, odd[0], odd[1], bg, bu), h)
    out = _gated(*full)
    a = torch.autograd.grad(out, full, dh.t().contiguous().t(), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(a, want))
    b = torch.autograd.grad(out.sum(), full, retain_graph=True)
    c = torch.autograd.grad(out, full, torch.ones_like(out), retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(b, c))
    dx, = torch.autograd.grad(out, full[0], dh.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_slopes(dt):
    """The gradient of the input and the biases against differences of the forward (the masters' is a straight-through one)."""
    x, wg, wu, bg, bu, dh = _inputs(9, 64, 24, torch.float32, seed=5)
    x, dh = x.to(dt).float(), dh.to(dt).float()
    args = [t.to(dt).requires_grad_() for t in (x, wg, wu, bg, bu)]
    grads = torch.autograd.grad(_gated(*args), args, dh.to(dt))
    args = [t.detach().float() for t in args]  # (differences in fp32, of the same values)
    for n in (0, 3, 4):
        step = torch.randn(args[n].shape, generator=torch.Generator().manual_seed(n)).cuda()
        ends = []
        for sign in (1, -1):
            moved = list(args)
            moved[n] = moved[n] + sign * 1e-2 * step
            ends.append(float((_gated(*moved).double() * dh).sum()))
        slope, want = (ends[0] - ends[1]) / 2e-2, float((grads[n].double() * step).sum())
        # the gradient's roundings (two halves of a step), and the differences': the third derivative in 1e-2, their own sum's steps
        size = float((grads[n].double().square() * step.double().square()).sum().sqrt())
        assert abs(slope - want) <= (1e-2 + 8 * torch.finfo(dt).eps) * size + 1e-3, (n, slope, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_saturated_and_unusual_rows_stay_by_themselves(dt):
    x, wg, wu, bg, bu, dh = _inputs(80, 256, 64, dt, seed=6)
    x[3], x[5] = 0, x[5] * 500  # (gates beyond +-88 where exp over- and underflows)
    ref = _Reference(x, wg, wu, bg, bu, dh)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    h = _gated(*leaves)
    dx, = torch.autograd.grad(h, leaves[0], dh)
    if dt != torch.float16:
        assert bool(h.isfinite().all()) and bool(dx.isfinite().all())
        assert float(ref.g[5].abs().max()) > 89
        _assert_within(h.detach(), ref.h, ref.tol_h, "saturated")
    y = x.detach().clone()
    y[7, 3], y[70, 9] = float("nan"), float("inf")
    y.requires_grad_()
    other = [i for i in range(80) if i not in (7, 70)]
    h2 = _gated(y, *leaves[1:])
    dx2, = torch.autograd.grad(h2, y, dh)
    assert torch.equal(h2[other], h[other]) and torch.equal(dx2[other], dx[other])
    assert bool(h2[7].isnan().all())


@pytest.mark.gpu
def test_autocast_is_the_half_precision_call():
    x, wg, wu, bg, bu, dh = _inputs(50, 136, 40, torch.float32, seed=7)
    full = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    with torch.autocast("cuda", dtype=torch.float16):
        h = _gated(*full)
    half = [t.detach().half().requires_grad_() for t in full]
    want = _gated(*half)
    assert h.dtype == torch.float16 and torch.equal(h, want)
    grads = torch.autograd.grad(h, full, dh.half())
    for got, w in zip(grads, torch.autograd.grad(want, half, dh.half())):
        # the same fp16 sums; biases and masters may keep more of them
        assert got.dtype == torch.float32 and _norm_error(got, w.double()) <= torch.finfo(torch.float16).eps / 2 + 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_streams_and_captured_graphs(dt):
    x, wg, wu, bg, bu, dh = _inputs(100, 264, 144, dt, seed=8)

    def step(*args):
        leaves = [t.detach().requires_grad_() for t in args[:5]]
        h = _gated(*leaves)
        return (h.detach(), *torch.autograd.grad(h, leaves, args[5]))

    want = step(x, wg, wu, bg, bu, dh)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, wg, wu, bg, bu, dh)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graphs = []
    for sign in (1, -1):
        static = [t.clone() for t in (x * sign, wg, wu, bg, bu, dh)]
        expect = [t.clone() for t in step(*static)]
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out, expect))
    for _ in range(3):
        for graph, static, out, expect in graphs:
            for t in out:
                t.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, expect))
            assert all(torch.equal(a, b) for a, b in zip(step(*static), expect))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wt", [(d, d) for d in DTYPES] + [(torch.bfloat16, torch.float32), (torch.float32, torch.float16), (torch.float16, torch.bfloat16)])
def test_native_and_python_calls_agree(dt, wt, monkeypatch):
    """csrc/calls.cpp and ops/gated.py, bit for bit, for every set of wanted gradients."""
    from bittorch_amd import _C, _lib
    x, wg, wu, bg, bu, dh = _inputs(36, 72, 44, dt, wt, seed=10)
    x, dh = x.reshape(4, 9, 72), dh.reshape(4, 9, 44)
    native, got = _C._N, []
    for calls in (native, _lib._PythonCalls()):
        monkeypatch.setattr(_C, "_N", calls)
        outs = []
        for biases in ((bg, bu), (bg, None), (None, bu), (None, None)):
            for quant in (dict(), dict(threshold_factor=0.4, per_channel=False)):
                args = [t if t is None else t.clone().requires_grad_() for t in (x, wg, wu, *biases)]
                leaves = [t for t in args if t is not None]
                h = _gated(*args, **quant)
                outs += [h.detach(), *torch.autograd.grad(h, leaves, dh, retain_graph=True)]
                outs += [torch.autograd.grad(h, leaf, dh, retain_graph=True)[0] for leaf in leaves]
                for n in range(len(leaves)):
                    one = [t if t is None else t.detach() for t in args]
                    at = [i for i, t in enumerate(args) if t is not None][n]
                    one[at].requires_grad_()
                    outs += torch.autograd.grad(_gated(*one, **quant), one[at], dh)
        got.append(outs)
        leaf = x.clone().requires_grad_()
        dx, = torch.autograd.grad(_gated(leaf, wg, wu), leaf, dh.clone().requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()
    assert len(got[0]) == len(got[1]) > 50
    for a, b in zip(*got):
        assert a.shape == b.shape and a.dtype == b.dtype and a.is_contiguous() and torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", DTYPES)
def test_generic_kernels_when_asked_for(dt, monkeypatch):
    """BITTORCH_KERNEL=generic: the shape-generic kernels of the layers, one by one, and the same values."""
    x, wg, wu, bg, bu, dh = _inputs(20, 72, 40, dt, seed=12)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    want = _gated(*leaves)
    grads = torch.autograd.grad(want, leaves, dh)
    monkeypatch.setenv("BITTORCH_KERNEL", "generic")
    got = _gated(*leaves)
    # the projections, silu and their product rounded one by one; the scales and the gradients of the projections too
    tol = 4 * torch.finfo(dt).eps / 2 + 1e-6
    assert _norm_error(got, want.double()) <= tol
    for a, b in zip(torch.autograd.grad(got, leaves, dh), grads):
        assert _norm_error(a, b.double()) <= tol


@pytest.mark.gpu
def test_agrees_with_two_layers_and_their_product():
    """The training form beside the layers that it stands for: the same codes and scales, so the same values up to their roundings."""
    import bittorch_amd as bt
    x, wg, wu, bg, bu, dh = _inputs(128, 256, 192, torch.float32, seed=9)
    layers = []
    for w, b in ((wg, bg), (wu, bu)):
        layer = bt.nn.TernaryLinear(256, 192).cuda()
        with torch.no_grad():
            layer.weight.copy_(w)
            layer.bias.copy_(b)
        layers.append(layer)
    y = x.clone().requires_grad_()
    h = torch.nn.functional.silu(layers[0](y)) * layers[1](y)
    h.backward(dh)
    leaves = [t.requires_grad_() for t in (x, wg, wu, bg, bu)]
    ours = _gated(*leaves)
    assert _norm_error(ours, h.double()) <= 1e-6
    for a, b in zip(torch.autograd.grad(ours, leaves, dh), (y.grad, layers[0].weight.grad, layers[1].weight.grad, layers[0].bias.grad, layers[1].bias.grad)):
        assert _norm_error(a, b.double()) <= 2e-6


@pytest.mark.parametrize("dt", [torch.float32, torch.float64])
def test_cpu_is_the_two_layers(dt):
    from bittorch_amd import nn
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 3, 20, generator=g, dtype=dt, requires_grad=True)
    layers = [nn.TernaryLinear(20, 12).to(dt) for _ in range(2)]
    args = [layers[0].weight, layers[1].weight, layers[0].bias, layers[1].bias]
    want = torch.nn.functional.silu(layers[0](x)) * layers[1](x)
    got = _gated(x, *args)
    assert torch.equal(got, want)
    dh = torch.randn(got.shape, generator=g, dtype=dt)
    for a, b in zip(torch.autograd.grad(got, [x, *args], dh), torch.autograd.grad(want, [x, *args], dh)):
        assert torch.equal(a, b)


def test_refusals():
    from bittorch_amd import _lib
    x, w = torch.randn(4, 16), torch.randn(8, 16)
    for args, text in [((x, w, w[:7]), "must match"), ((x, w, w.half()), "must match"), ((x, w[0], w[0]), "must match"),
                       ((x[:, :15], w, w), "input K"), ((x[:0], w, w), "x is empty"), ((x, w[:0], w[:0]), "weight is empty"),
                       ((x, w, w, torch.ones(7)), "bias shape"), ((x, w, w, None, torch.ones(8, 1)), "bias shape")]:
        with pytest.raises(RuntimeError, match=text):
            _gated(*args)
    lib, at = _lib.load(), 1 << 20  # (never read: every call ends before a launch)
    weights = lambda g=at, dt=2, pc=1, b=None, bdt=0, F=8, K=16, pairs=at, back=None, scale=at, bias=None, ws=None, n=0: lib.bt_gated_quantize(
        g, at, dt, F, K, 0.05, pc, b, b, bdt, pairs, back, scale, bias, ws, n, None)
    for kwargs, text in [(dict(g=None), "null"), (dict(scale=None), "null"), (dict(F=0), "empty"), (dict(pairs=None), "null"), (dict(dt=3), "dtype"), (dict(b=at), "bias"),
                         (dict(b=at, bias=at, bdt=3), "bias"), (dict(pairs=at + 16), "aligned"), (dict(back=at + 16), "aligned"),
                         (dict(F=1 << 23), "2^23"), (dict(K=1 << 23), "2^23"), (dict(F=1 << 20, K=1 << 20), "4 GiB")]:
        assert weights(**kwargs) == -1, kwargs
        assert text in _lib.last_error(), (kwargs, _lib.last_error())
    # a workspace where the rows are longer than a wave holds, or share one scale
    assert lib.bt_gated_quantize_workspace_bytes(8, 16, 1) == 0 and lib.bt_gated_quantize_workspace_bytes(0, 16, 0) == 0
    for kwargs in (dict(pc=0), dict(K=8200), dict(K=4)):
        need = lib.bt_gated_quantize_workspace_bytes(8, kwargs.get("K", 16), kwargs.get("pc", 1))
        assert need > 0 and weights(**kwargs) == -2 and weights(ws=at, n=need - 1, **kwargs) == -2 and weights(ws=at + 64, n=need, **kwargs) == -2
    forward = lambda X=at, dt=2, W=at, h=at, pre=None, B=4, F=8, K=16: lib.bt_ternary_gated_forward(X, dt, None, W, at, None, h, pre, B, F, K, None)
    for kwargs in (dict(X=None), dict(dt=0), dict(dt=5), dict(W=None), dict(h=None), dict(B=0), dict(K=12), dict(X=at + 8), dict(W=at + 128), dict(pre=at + 8),
                   dict(h=at + 4), dict(F=1 << 23), dict(B=1 << 31)):
        assert forward(**kwargs) == -1, kwargs
        assert "bt_ternary_gated_forward" in _lib.last_error()
    few = lambda X=at, xd=2, g=at, wd=2, b=None, bdt=0, h=at, F=8, K=16: lib.bt_gated_masters_forward(X, xd, g, at, wd, 0.05, b, b, bdt, h, F, K, None)
    for kwargs in (dict(X=None), dict(xd=3), dict(g=None), dict(wd=3), dict(b=at, bdt=3), dict(h=None), dict(K=4), dict(K=4097), dict(wd=0, K=2568), dict(K=2561), dict(F=0),
                   dict(F=1 << 23)):
        assert few(**kwargs) == -1, kwargs
        assert "bt_gated_masters_forward" in _lib.last_error()
    assert lib.bt_gated_masters_serves(1, 16, 2, 1) == 1 and lib.bt_gated_masters_serves(0, 16, 2, 1) == 0
    grad = lambda dh=at, dt=2, pre=at, scale=at, G=at, db=None, bdt=0, B=4, F=8, ws=None, n=0: lib.bt_gated_grad(
        dh, dt, pre, scale, G, db, bdt, B, F, ws, n, None)
    for kwargs in (dict(dh=None), dict(pre=None), dict(G=None), dict(scale=None), dict(dt=3), dict(F=0), dict(B=1 << 31), dict(pre=at + 4), dict(G=at + 4),
                   dict(db=at, bdt=3)):
        assert grad(**kwargs) == -1, kwargs
    need = lib.bt_gated_grad_workspace_bytes(4, 8)
    assert need > 0 and lib.bt_gated_grad_workspace_bytes(0, 8) == 0
    assert grad(db=at) == -2 and grad(db=at, ws=at, n=need - 1) == -2 and grad(db=at, ws=at + 8, n=need) == -2


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    x, w = torch.randn(4, 16, device="cuda"), torch.randn(8, 16, device="cuda")
    with pytest.raises(RuntimeError, match="one device"):
        _gated(x, w.cpu(), w.cpu())
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        _gated(x.double(), w, w)
    assert _gated(x, w[:1], w[:1]).shape == _gated(x.half(), w[:1], w[:1]).shape == (4, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("per_channel", [True, False])
@pytest.mark.parametrize("rows,k,f", [(3, 96, 5), (70, 512, 340), (65, 333, 200)])
def test_small_gradients_of_fp16_rows(rows, k, f, per_channel, autocast):
    """Incoming gradients near fp16's smallest numbers, scales of 1/100: G has to keep what fp16 keeps of them without the scale."""
    announce("gated small", rows, k, f, per_channel, autocast)
    g = torch.Generator().manual_seed(rows + f)
    x, dh = torch.randn(rows, k, generator=g).half().cuda(), (torch.randn(rows, f, generator=g) * 2.0 ** -12).half().cuda()
    wg, wu = ((torch.randn(f, k, generator=g) * 0.003).half().cuda() for _ in range(2))
    ref = _Reference(x, wg, wu, None, None, dh, per_channel=per_channel)
    leaves = [(t.float() if autocast else t).requires_grad_() for t in (x, wg, wu)]
    with torch.autocast("cuda", enabled=autocast):
        h = _gated(*leaves, per_channel=per_channel)
    assert h.dtype == torch.float16
    dx, dwg, dwu = torch.autograd.grad(h, leaves, dh)
    # half a step of G: 2^-11 of it, and 2^-25 among the subnormal numbers, in units of at most twice the largest scale
    half, chain = 2.0 ** -11, lambda n: U * 2 * (3 * n / 32 + 80)
    least = 2.0 ** -25 * 2 * float(max(ref.ag.max(), ref.au.max()))
    parts = [(ref.dg, ref.tol_dg, ref.ag, ref.tg), (ref.du, ref.tol_du, ref.au, ref.tu)]
    off = lambda n: [(tol * (1 + half) + (half + chain(n)) * v.abs()) * a + least for v, tol, a, _ in parts]
    want = sum((v * a) @ t for v, _, a, t in parts)
    tol = sum(o @ t.abs() for o, (_, _, _, t) in zip(off(2 * f), parts))
    # (under autocast dx is rounded to fp16 all the same, and widened)
    bound = tol + half * (want.abs() + tol) + 2.0 ** -25
    assert bool(((dx.double() - want).abs() <= bound).all())
    for got, o, (v, _, a, _) in zip((dwg, dwu), off(rows), parts):
        want_w, tol_w = (v * a).t() @ ref.x, o.t() @ ref.x.abs()
        bound = tol_w + half * (want_w.abs() + tol_w) + 2.0 ** -25
        assert bool(((got.double() - want_w).abs() <= bound).all())


@pytest.mark.gpu
@pytest.mark.parametrize("f,largest", [(1, 0.7), (16, 1.0), (5000, 0.011), (40, 3e-9), (40, 1e-30), (40, 3e38)])
def test_range_of_the_scales(f, largest):
    from bittorch_amd import _C
    fp = (f + 15) // 16 * 16
    scale = torch.rand(2 * fp + 1, generator=torch.Generator().manual_seed(f)).mul_(largest * 0.9).cuda()
    scale[fp // 2] = largest
    scale[2 * fp] = -1
    before = scale.clone()
    _C._status(_C._L.bt_gated_range(scale.data_ptr(), f, _C._stream(scale)))
    assert torch.equal(scale[:2 * fp], before[:2 * fp])
    top = float(scale[2 * fp])
    mantissa, exponent = math.frexp(top)
    assert mantissa == 0.5 and exponent - 1 == min(15, max(-24, math.frexp(float(before[fp // 2]))[1]))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k,f", [(1, 1, 1), (40, 13, 20), (300, 100, 33), (500, 1100, 2730), (5000, 1001, 2730), (2048, 2047, 1030), (2048, 2048, 1030),
                                      (4096, 1026, 4100)])
def test_weight_gradient_in_rows_of_its_own_length(rows, k, f, dt):
    """The masters' gradients without the padding of both dimensions: the bits of the padded product, in tiles of both sizes, whole and in parts."""
    announce("gated grad weight", rows, k, f, dt)
    from bittorch_amd import _C
    g = torch.Generator().manual_seed(rows + k)
    fp, kr = (f + 15) // 16 * 16, (k + 7) // 8 * 8
    G = torch.randn(rows, 2 * fp, generator=g).to(dt).cuda()
    x = torch.randn(rows, kr, generator=g).to(dt).cuda()  # (what lies behind k is not used)
    scale = torch.ones(2 * fp + 1, device="cuda")
    scale[2 * fp] = 0.25
    for out in (dt, torch.float32):
        full = _C.linear_grad_weight_16(G, x, scale[2 * fp:], out)
        got = _C.gated_grad_weight(G, x, scale, f, k, out)
        assert torch.equal(got[:f], full[:f, :k]) and torch.equal(got[f:], full[fp:fp + f, :k])
    guard = torch.full((2 * f * k + 64,), 7.0, dtype=dt, device="cuda")  # nothing in front of the first row or behind the last one
    ws = _C._workspace(_C._L.bt_linear_grad_weight_16_workspace_bytes(rows, 2 * fp, kr), guard.device)
    _C._status(_C._L.bt_gated_grad_weight(G.data_ptr(), x.data_ptr(), _C._DT[dt], scale[2 * fp:].data_ptr(), guard[32:].data_ptr(), _C._DT[dt], rows, f, k,
                                          _C._ptr(ws), 0 if ws is None else ws.numel(), _C._stream(G)))
    assert bool((guard[:32] == 7).all()) and bool((guard[32 + 2 * f * k:] == 7).all())
    assert torch.equal(guard[32:32 + 2 * f * k].view(2 * f, k), _C.gated_grad_weight(G, x, scale, f, k, dt))


def test_weight_gradient_and_range_refusals():
    from bittorch_amd import _C, _lib
    lib, at = _lib.load(), 4096
    grad = lambda G=at, X=at, dt=2, s=at, out=at, odt=2, B=4, F=8, K=16, ws=None, n=0: lib.bt_gated_grad_weight(G, X, dt, s, out, odt, B, F, K, ws, n, None)
    for bad in (dict(G=None), dict(X=None), dict(s=None), dict(out=None), dict(B=0), dict(F=0), dict(K=0), dict(F=1 << 23), dict(K=1 << 23), dict(dt=0),
                dict(odt=1), dict(G=4100), dict(X=4100), dict(out=4100, F=16), dict(out=4097, K=15)):
        assert grad(**bad) == -1, bad
    need = lib.bt_linear_grad_weight_16_workspace_bytes(4096, 32, 16)
    assert need > 0 and grad(B=4096, F=16) == grad(B=4096, F=16, ws=4096, n=need - 1) == grad(B=4096, F=16, ws=4100, n=need) == -2
    for args in ((None, 8), (at, 0), (at, 1 << 23)):
        assert lib.bt_gated_range(*args, None) == -1
    with pytest.raises(RuntimeError, match="16-bit"):
        _C.gated_grad_weight(torch.zeros(4, 32), torch.zeros(4, 16), torch.zeros(33), 16, 16, torch.float32)


def _assert_fp16_gradients(leaves, h, dh, ref, rows, f):
    """Every gradient within what fp16's G may add to it: half a step of each entry, 2^-11 of it and 2^-25 among the subnormal numbers, where
    G is the gradient times at least a half, so that a feature's own scale, not the largest one, says what that is."""
    dx, dwg, dwu, *_ = torch.autograd.grad(h, leaves, dh)
    half, chain = 2.0 ** -11, lambda n: U * 2 * (3 * n / 32 + 80)
    parts = [(ref.dg, ref.tol_dg, ref.ag, ref.tg), (ref.du, ref.tol_du, ref.au, ref.tu)]
    off = lambda n: [((tol * (1 + half) + (half + chain(n)) * v.abs()) + 2.0 ** -24) * a for v, tol, a, _ in parts]
    want = sum((v * a) @ t for v, _, a, t in parts)
    tol = sum(o @ t.abs() for o, (_, _, _, t) in zip(off(2 * f), parts))
    # (under autocast dx is rounded to fp16 all the same, and widened)
    over = (dx.double() - want).abs() / (tol + half * (want.abs() + tol) + 2.0 ** -25)
    assert bool((over <= 1).all()), f"dx: {float(over.max())} of its bound"
    for got, o, (v, _, a, _), what in zip((dwg, dwu), off(rows), parts, ("gate", "up")):
        want_w, tol_w = (v * a).t() @ ref.x, o.t() @ ref.x.abs()
        last = (half, 2.0 ** -25) if got.dtype == torch.float16 else (2.0 ** -8, 0.0) if got.dtype == torch.bfloat16 else (U, 0.0)
        over = (got.double() - want_w).abs() / (tol_w + last[0] * (want_w.abs() + tol_w) + last[1])
        assert bool((over <= 1).all()), f"{what}: {float(over.max())} of its bound"
    return dx, dwg, dwu


@pytest.mark.gpu
@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("rows,k,f", [(512, 264, 48), (600, 129, 40), (2048, 1024, 520)])
def test_large_gradients_of_small_masters(rows, k, f, autocast):
    """Sums over the rows beyond fp16 whose product with the masters' scales is far inside it."""
    announce("gated large", rows, k, f, autocast)
    g = torch.Generator().manual_seed(rows + f)
    x, dh = torch.randn(rows, k, generator=g).abs().half().cuda(), ((torch.rand(rows, f, generator=g) + 0.5) * 60 * 512 / rows).half().cuda()
    wg, wu = ((torch.randn(f, k, generator=g) * 0.003).half().cuda() for _ in range(2))
    bg, bu = (torch.full((f,), 4.0).half().cuda() for _ in range(2))
    ref = _Reference(x, wg, wu, bg, bu, dh)
    assert float((ref.dg.t() @ ref.x).max()) > 65504 and float(((ref.dg * ref.ag).t() @ ref.x).max()) < 4000
    leaves = [(t.float() if autocast else t).requires_grad_() for t in (x, wg, wu, bg, bu)]
    with torch.autocast("cuda", enabled=autocast):
        h = _gated(*leaves)
    _assert_fp16_gradients(leaves, h, dh, ref, rows, f)


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wt", [(torch.float16, torch.float32), (torch.bfloat16, torch.float32), (torch.float16, torch.bfloat16)])
@pytest.mark.parametrize("rows,k,f", [(40, 264, 48), (300, 1001, 37), (2048, 1024, 520)])
def test_masters_of_more_bits_get_gradients_rounded_once(rows, k, f, dt, wt):
    """The sums of 16-bit rows in fp32 for fp32 masters: of the product with G as it is, only fp32's own roundings remain."""
    announce("gated grad masters", rows, k, f, dt, wt)
    from bittorch_amd import _C
    g = torch.Generator().manual_seed(rows + k)
    fp, kr = (f + 15) // 16 * 16, (k + 7) // 8 * 8
    G = torch.randn(rows, 2 * fp, generator=g).to(dt).cuda()
    x = torch.randn(rows, kr, generator=g).to(dt).cuda()
    for scale in (torch.rand(2 * fp, generator=g).cuda() + 0.01, torch.full((1,), 2.0 ** -6).cuda()):
        got = _C.gated_grad_masters(G, x, scale, f, k, wt if wt == torch.float32 else dt)
        each = scale.double().expand(2 * fp)
        full, size = (G.double().t() @ x.double()) * each[:, None], (G.double().abs().t() @ x.double().abs()) * each[:, None]
        pick = torch.cat((torch.arange(f), torch.arange(f) + fp)).cuda()
        want, size = full[pick, :k], size[pick, :k]
        half = U if wt == torch.float32 else torch.finfo(dt).eps / 2
        assert bool(((got.double() - want).abs() <= U * 2 * (3 * rows / 32 + 80) * size + half * want.abs() + 2.0 ** -25 * (wt != torch.float32)).all())


def test_masters_gradient_refusals():
    from bittorch_amd import _C, _lib
    lib, at = _lib.load(), 4096
    grad = lambda G=at, X=at, dt=2, s=at, n_s=1, out=at, odt=2, B=4, F=8, K=16, ws=None, n=0: lib.bt_gated_grad_masters(
        G, X, dt, s, n_s, out, odt, B, F, K, ws, n, None)
    for bad in (dict(G=None), dict(X=None), dict(s=None), dict(out=None), dict(B=0), dict(F=0), dict(K=0), dict(F=1 << 23), dict(K=1 << 23), dict(dt=0),
                dict(odt=1), dict(G=4100), dict(X=4100), dict(out=4100, F=16), dict(out=4097, K=15), dict(n_s=0), dict(n_s=16), dict(n_s=33)):
        assert grad(**bad) == -1, bad
        assert "bt_gated_grad_masters" in _lib.last_error()
    need = lib.bt_linear_grad_weight_16_workspace_bytes(4096, 32, 16)
    assert need > 0 and grad(B=4096, F=16) == grad(B=4096, F=16, ws=4096, n=need - 1) == grad(B=4096, F=16, ws=4100, n=need) == -2
    with pytest.raises(RuntimeError, match="16-bit"):
        _C.gated_grad_masters(torch.zeros(4, 32), torch.zeros(4, 16), torch.zeros(32), 16, 16, torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("masters", ["fp16", "autocast", "fp32", "bf16"])
@pytest.mark.parametrize("kind", ["one entry", "rows", "halves"])
@pytest.mark.parametrize("rows,k,f", [(3, 96, 5), (70, 512, 340), (65, 333, 200), (300, 512, 256)])
def test_scales_far_apart_in_fp16(rows, k, f, kind, masters):
    """One large entry among masters of 0.003, features from 1e-4 to 1 (a spread of 1e4), one half 1000 times the other: every feature keeps
    what fp16 keeps of its gradient."""
    announce("gated scales apart", rows, k, f, kind, masters)
    g = torch.Generator().manual_seed(rows + f)
    x, dh = torch.randn(rows, k, generator=g).half().cuda(), (torch.randn(rows, f, generator=g) * 2.0 ** -12).half().cuda()
    wg, wu = (torch.randn(f, k, generator=g) * 0.003 for _ in range(2))
    if kind == "one entry":
        wu[f // 2, k // 3] = 4.0
    elif kind == "rows":
        wg, wu = (w / 0.003 * 0.25 * 10.0 ** -(4 * torch.rand(f, 1, generator=g)) for w in (wg, wu))
    else:
        wu = wu * 1000
    wt = {"fp16": torch.float16, "autocast": torch.float16, "fp32": torch.float32, "bf16": torch.bfloat16}[masters]
    wg, wu = wg.to(wt).cuda(), wu.to(wt).cuda()
    ref = _Reference(x, wg, wu, None, None, dh)
    leaves = [(t.float() if masters == "autocast" else t).requires_grad_() for t in (x, wg, wu)]
    with torch.autocast("cuda", enabled=masters == "autocast"):
        h = _gated(*leaves)
    assert h.dtype == torch.float16
    _assert_fp16_gradients(leaves, h, dh, ref, rows, f)


@pytest.mark.gpu
@pytest.mark.parametrize("f,largest,spread", [(1, 0.7, 0), (16, 1.0, 3), (5000, 0.011, 30), (40, 3e-9, 20), (40, 1e-30, 5), (40, 3e38, 90), (8, 2.0 ** 15, 40)])
def test_scales_taken_apart(f, largest, spread):
    from bittorch_amd import _C
    n = 2 * ((f + 15) // 16 * 16)
    g = torch.Generator().manual_seed(f)
    scale = torch.cat((largest * 2.0 ** -(spread * torch.rand(n, generator=g)), torch.tensor([1.0]))).cuda()
    scale[n // 4], scale[n - 1] = largest, 0
    before = scale.cpu()
    split = _C.gated_split(scale, f)
    scale, split = scale.cpu(), split.cpu()
    assert split.numel() * 4 == _C._L.bt_gated_split_bytes(f) and torch.equal(scale[:n], before[:n])
    top = min(15, max(-24, math.frexp(float(before[n // 4]))[1]))
    own = [max(top - 24, min(top + 15, math.frexp(v)[1])) if v else top - 24 for v in before[:n].tolist()]
    power = torch.tensor([2.0 ** e for e in own], dtype=torch.float64)
    assert float(scale[n]) == float(split[n + 1]) == 2.0 ** top and float(split[n]) == 1
    assert torch.equal(split[n + 16:2 * n + 16].double(), power)
    assert torch.equal(split[:n], (before[:n].double() / power).float())
    factors = split[2 * n + 16:].view(torch.float16)
    assert torch.equal(factors[:n].double(), power / 2.0 ** top) and not factors[n:].any() and factors.numel() == (n + 63) // 64 * 64


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,f", [(1, 1, 1), (1, 640, 48), (7, 8, 2), (33, 264, 48), (63, 129, 90), (70, 2560, 688), (300, 1100, 546), (500, 1100, 2730), (600, 2560, 1040),
                                      (1000, 2560, 2736), (129, 13824, 100), (2100, 4096, 520), (3000, 4098, 1030), (4096, 2560, 3456), (1300, 8192, 200)])
def test_input_gradient_with_a_power_of_two_for_each_feature(rows, k, f):
    """The product on its own, over factors from 2^-24 to 2^0 and a few above, in tiles of every height: against 64 bits, and the same bits again."""
    announce("gated grad input", rows, k, f)
    from bittorch_amd import _C
    g = torch.Generator().manual_seed(rows + k + f)
    fp = (f + 15) // 16 * 16
    wg, wu = ((torch.randn(f, k, generator=g) * 0.05).half().cuda() for _ in range(2))
    _, w_back, scale, _ = _C.gated_weights(wg, wu, back=True)
    scale[:2 * fp] = 0.4 * 2.0 ** -(torch.rand(2 * fp, generator=g) * 22).cuda()
    scale[f // 2] = 60000  # (a power of two of its own beyond the largest that the others are held against)
    split = _C.gated_split(scale, f)
    G = torch.randn(rows, 2 * fp, generator=g).half().cuda()
    by = split[2 * fp + 16:4 * fp + 16].double()
    codes = torch.zeros(2 * fp, k, dtype=torch.float64, device="cuda")
    codes[:f], codes[fp:fp + f] = _ternary(wg)[0], _ternary(wu)[0]
    got = _C.gated_grad_input(G, w_back, split, f, k)
    terms = G.double() * by
    want, size = terms @ codes, terms.abs() @ codes.abs()
    bound = U * 2 * (2 * fp / 32 + 80) * size
    bound = bound + 2.0 ** -11 * (want.abs() + bound) + 2.0 ** -25
    fits = want.abs() + bound < 65504
    assert bool((((got.double() - want).abs() <= bound) | ~fits).all()), float(((got.double() - want).abs() / bound)[fits].max())
    assert torch.equal(got, _C.gated_grad_input(G, w_back, split, f, k))
    guard = torch.full((rows * k + 64,), 7.0, dtype=torch.float16, device="cuda")
    ws = _C._workspace(_C._L.bt_gated_grad_input_workspace_bytes(rows, f, k), G.device)
    _C._status(_C._L.bt_gated_grad_input(G.data_ptr(), w_back.data_ptr(), split.data_ptr(), guard[32:].data_ptr(), rows, f, k,
                                          _C._ptr(ws), 0 if ws is None else ws.numel(), _C._stream(G)))
    assert bool((guard[:32] == 7).all()) and bool((guard[32 + rows * k:] == 7).all()) and torch.equal(guard[32:32 + rows * k].view(rows, k), got)


def test_split_and_input_gradient_refusals():
    from bittorch_amd import _C, _lib
    lib, at = _lib.load(), 4096
    assert lib.bt_gated_split_bytes(0) == lib.bt_gated_split_bytes(1 << 23) == 0 and lib.bt_gated_split_bytes(8) == 4 * (64 + 16) + 128
    for args in ((None, 8, at), (at, 8, None), (at, 0, at), (at, 1 << 23, at), (at, 8, at + 4)):
        assert lib.bt_gated_split(*args, None) == -1 and "bt_gated_split" in _lib.last_error()
    grad = lambda G=at, W=at, s=at, dx=at, B=4, F=8, K=16, ws=None, n=0: lib.bt_gated_grad_input(
        G, W, s, dx, B, F, K, ws, n, None)
    for bad in (dict(G=None), dict(W=None), dict(s=None), dict(dx=None), dict(B=0), dict(F=0), dict(K=0), dict(F=1 << 23), dict(K=1 << 23), dict(B=1 << 31),
                dict(F=(1 << 23) - 1), dict(F=1 << 20, K=1 << 20), dict(G=at + 8), dict(W=at + 128), dict(s=at + 4), dict(dx=at + 8)):
        assert grad(**bad) == -1, bad
        assert "bt_gated_grad_input" in _lib.last_error()
    need = lib.bt_gated_grad_input_workspace_bytes(4, 1024, 16)
    assert need > 0 and grad(F=1024) == grad(F=1024, ws=at, n=need - 1) == grad(F=1024, ws=at + 16, n=need) == -2
    assert lib.bt_gated_grad_input_workspace_bytes(0, 8, 16) == 0
    for call in (lambda: _C.gated_split(torch.ones(33), 16), lambda: _C.gated_grad_input(torch.zeros(4, 32), torch.zeros(1, dtype=torch.uint8), torch.zeros(8), 16, 16)):
        with pytest.raises(RuntimeError):
            call()
