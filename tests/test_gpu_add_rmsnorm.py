"""``ops.add_rmsnorm``: the residual connection, the norm behind it and the int8 form of that in one pass, and its gradient.

Forward: bit for bit the addition, ``ops.rmsnorm`` and ``ops.act_quant_int8``.  Gradient: the formula in 64 bits.
"""
import pytest
import torch

from conftest import announce

EPS = 1e-5
TYPES = [(torch.float32, torch.float32), (torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
         (torch.float16, torch.float32), (torch.bfloat16, torch.float32)]
# one piece of a lane, fewer values than one, a last piece that overlaps the one before, every number of waves to a row, longer rows
SHAPES = [(1, 8), (3, 7), (5, 1), (2, 9), (1, 2560), (17, 100), (9, 513), (4, 1001), (33, 1536), (7, 2560), (6, 4096), (5, 4100), (3, 8200),
          (2, 12296), (2, 16384), (3, 16391)]


def _ops():
    from bittorch_amd import ops
    return ops


def _inputs(rows, k, dt, rt, seed=0, w_dtype=None):
    g = torch.Generator().manual_seed(seed * 131 + rows * 7 + k)
    mk = lambda *shape: torch.randn(*shape, generator=g)
    x, res, w = mk(rows, k).to(dt), (3 * mk(rows, k)).to(rt), (1 + 0.2 * mk(k)).to(w_dtype or dt)
    ds, dy = (0.1 * mk(rows, k)).to(rt), (0.1 * mk(rows, k)).to(dt)
    return [t.cuda() for t in (x, res, w, ds, dy)]


def _reference_grads(s, w, ds, dy):
    """The gradient in 64 bits from the stored sum, with the magnitudes that its 32-bit evaluation rounds: (d, its bound), (dw, its bound)."""
    rows, k = s.shape
    u = 2.0 ** -24
    s, dy = s.double(), dy.double()
    w = torch.ones(k, dtype=torch.float64, device=s.device) if w is None else w.double()
    ds = torch.zeros_like(s) if ds is None else ds.double()
    r = 1 / (s.square().mean(-1, keepdim=True) + EPS).sqrt()
    xhat, dyw = s * r, dy * w
    c, c_abs = (dyw * xhat).mean(-1, keepdim=True), (dyw * xhat).abs().mean(-1, keepdim=True)
    d = ds + r * (dyw - xhat * c)
    # r: the sum of squares, the division by K, eps, the root and the reciprocal round once each, halved by the root: under 4 u.  c: two
    # products, a chain of 8 + 4 additions in a lane, 6 in the wave, 8 over waves, the division, r: under 40 u of the sum of magnitudes.
    # Then four operations on each term.  (Rows outside 8 .. 16384 add 64 values in a lane one after the other: 2 K / 256 more.)
    chain = 40 + (k / 128 if k < 8 or k > 16384 else 0)
    d_tol = u * (2 * ds.abs() + 10 * r * dyw.abs() + (12 + chain) * r * xhat.abs() * c_abs)
    dw, dw_abs = (dy * xhat).sum(0), (dy * xhat).abs().sum(0)
    # each term: three roundings and r's; the sum: at most `rows` additions one after the other
    return (d, d_tol), (dw, u * (8 + rows) * dw_abs)


def _assert_within(got, want, tol, what):
    half = torch.finfo(got.dtype).eps / 2
    bound = tol + half * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal * half
    off = (got.double() - want).abs() - bound
    assert not bool((off > 0).any()) and not bool(got.isnan().any()), f"{what}: {float(off.max())} over its bound"


@pytest.mark.gpu
@pytest.mark.parametrize("dt,rt", TYPES)
@pytest.mark.parametrize("rows,k", SHAPES)
def test_forward_is_the_three_operations_bit_for_bit(rows, k, dt, rt):
    announce("add_rmsnorm", rows, k, dt, rt)
    ops = _ops()
    x, res, w, *_ = _inputs(rows, k, dt, rt)
    s = (x.float() + res.float()).to(rt)
    got_s, got_y = ops.add_rmsnorm(x, res, w, EPS)
    assert torch.equal(got_s, s)
    if rt == dt:
        y = ops.rmsnorm(s, w, EPS)
    else:  # the norm of an fp32 row, rounded once to x's type
        y = ops.rmsnorm(s, w.float(), EPS).to(dt)
    assert torch.equal(got_y, y)
    q, s_x, sums = ops.act_quant_int8(y, return_rowsum=True)
    got = ops.add_rmsnorm(x, res, w, EPS, quantize=True, return_rowsum=True)
    for a, b in zip(got, (s, y, q, s_x, sums)):
        assert torch.equal(a, b)
    got_s, got_q, got_sx = ops.add_rmsnorm(x, res, w, EPS, store=False, quantize=True)
    assert torch.equal(got_s, s) and torch.equal(got_q, q) and torch.equal(got_sx, s_x)
    if k % 16 == 0:
        got = ops.add_rmsnorm(x, res, w, EPS, store=False, quantize=True, operand_order=True)
        assert torch.equal(got[1], ops.act_quant_int8(y, True)[0]) and torch.equal(got[2], s_x)
    alone = ops.add_rmsnorm(x, None, w, EPS)
    assert alone[0] is x and torch.equal(alone[1], ops.rmsnorm(x, w, EPS))
    assert torch.equal(ops.add_rmsnorm(x, res, None, EPS)[1], ops.rmsnorm(s, None, EPS).to(dt))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,rt", TYPES)
@pytest.mark.parametrize("rows,k", SHAPES + [(700, 257), (2100, 64)])
def test_gradient_is_the_formula(rows, k, dt, rt):
    announce("add_rmsnorm gradient", rows, k, dt, rt)
    ops = _ops()
    x, res, w, ds, dy = _inputs(rows, k, dt, rt, seed=1)
    leaves = [t.requires_grad_() for t in (x, res, w)]
    s, y = ops.add_rmsnorm(x, res, w, EPS)
    (d, d_tol), (dw, dw_tol) = _reference_grads(s.detach(), w.detach(), ds, dy)
    for _ in range(2):  # the same bits every time
        dx, dr, dwt = torch.autograd.grad((s, y), leaves, (ds, dy), retain_graph=True)
        assert (dx.dtype, dr.dtype, dwt.dtype) == (dt, rt, w.dtype)
        _assert_within(dx, d, d_tol, "dx")
        _assert_within(dr, d, d_tol, "dresidual")
        _assert_within(dwt, dw, dw_tol, "dweight")
    again = torch.autograd.grad((s, y), leaves, (ds, dy))
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dr, dwt)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,rt", TYPES)
def test_shape_generic_kernels(dt, rt):
    """Option ROWOP_GENERIC: the element-wise kernels at a size that the others serve; the same forward bits."""
    from _util import set_option
    ops = _ops()
    x, res, w, ds, dy = _inputs(70, 520, dt, rt, seed=4)
    want = ops.add_rmsnorm(x, res, w, EPS, quantize=True, return_rowsum=True)
    set_option("ROWOP_GENERIC", "1")
    for a, b in zip(ops.add_rmsnorm(x, res, w, EPS, quantize=True, return_rowsum=True), want):
        assert torch.equal(a, b)
    leaves = [t.requires_grad_() for t in (x, res, w)]
    s, y = ops.add_rmsnorm(*leaves, EPS)
    (d, d_tol), (dw, dw_tol) = _reference_grads(s.detach(), w.detach(), ds, dy)
    dx, dr, dwt = torch.autograd.grad((s, y), leaves, (ds, dy))
    _assert_within(dx, d, d_tol, "dx")
    _assert_within(dr, d, d_tol, "dresidual")
    _assert_within(dwt, dw, dw_tol, "dweight")


@pytest.mark.gpu
def test_gradient_of_parts_of_the_call():
    """One output used, one input wanted, no weight, an fp32 weight, no residual."""
    ops = _ops()
    x, res, w, ds, dy = _inputs(37, 520, torch.bfloat16, torch.bfloat16, seed=2)
    s0 = (x.float() + res.float()).bfloat16()
    x1 = x.clone().requires_grad_()
    s, y = ops.add_rmsnorm(x1, res, w, EPS)
    (d, tol), _ = _reference_grads(s0, w, None, dy)
    _assert_within(torch.autograd.grad(y, x1, dy)[0], d, tol, "norm alone")
    s, y = ops.add_rmsnorm(x1, res, w, EPS)
    assert torch.equal(torch.autograd.grad(s, x1, ds)[0], ds)
    wf = w.float().requires_grad_()
    s, y = ops.add_rmsnorm(x, res, wf, EPS)
    _, (dw, tol) = _reference_grads(s0, wf.detach(), None, dy)
    _assert_within(torch.autograd.grad(y, wf, dy)[0], dw, tol, "fp32 weight")
    r1 = res.clone().requires_grad_()
    s, y = ops.add_rmsnorm(x, r1, None, EPS)
    (d, tol), _ = _reference_grads(s0, None, ds, dy)
    _assert_within(torch.autograd.grad((s, y), r1, (ds, dy))[0], d, tol, "no weight")
    same, y = ops.add_rmsnorm(x1, None, w, EPS)
    assert same is x1
    (d, tol), _ = _reference_grads(x, w, None, dy)
    _assert_within(torch.autograd.grad(y, x1, dy)[0], d, tol, "no residual")
    # int8 rows beside the norm: they carry no gradient, the others do
    s, y, q, s_x = ops.add_rmsnorm(x1, res, w, EPS, quantize=True)
    assert not q.requires_grad and not s_x.requires_grad
    (d, tol), _ = _reference_grads(s0, w, ds, dy)
    _assert_within(torch.autograd.grad((s, y), x1, (ds, dy))[0], d, tol, "with int8 rows")
    s, q, s_x = ops.add_rmsnorm(x1, res, w, EPS, store=False, quantize=True)
    assert torch.equal(torch.autograd.grad(s, x1, ds)[0], ds)
    # one tensor as both: its gradient is the sum of the two, which are one tensor
    both = x.clone().requires_grad_()
    s, y = ops.add_rmsnorm(both, both, w, EPS)
    twice, = torch.autograd.grad((s, y), both, (ds, dy))
    x2, r2 = x.clone().requires_grad_(), x.clone().requires_grad_()
    once = torch.autograd.grad(ops.add_rmsnorm(x2, r2, w, EPS), (x2, r2), (ds, dy))
    assert torch.equal(once[0], once[1]) and torch.equal(twice, once[0] + once[1])
    row = res[:1].clone().requires_grad_()  # (a broadcast stream)
    s, y = ops.add_rmsnorm(x, row.expand_as(x), w, EPS)
    got, = torch.autograd.grad((s, y), row, (ds, dy))
    full = row.detach().expand_as(x).contiguous().requires_grad_()
    assert torch.equal(got, torch.autograd.grad(ops.add_rmsnorm(x, full, w, EPS), full, (ds, dy))[0].sum(0, keepdim=True))
    # a second derivative is refused
    s, y = ops.add_rmsnorm(x1, res, w, EPS)
    dx, = torch.autograd.grad(y, x1, dy, create_graph=True)
    with pytest.raises(RuntimeError, match="does not require grad|once_differentiable"):
        dx.sum().backward()
    dx, = torch.autograd.grad(ops.add_rmsnorm(x1, res, w, EPS)[1], x1, dy.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.sum().backward()


@pytest.mark.gpu
def test_gradient_is_the_slope():
    """Against differences of the forward itself: fp32, a step that moves the loss by far more than its rounding."""
    ops = _ops()
    x, res, w, ds, dy = _inputs(3, 40, torch.float32, torch.float32, seed=3)
    leaves = [t.requires_grad_() for t in (x, res, w)]

    def loss(a, b, c):
        s, y = ops.add_rmsnorm(a, b, c, EPS)
        return float((s.double() * ds).sum() + (y.double() * dy).sum())

    grads = torch.autograd.grad(ops.add_rmsnorm(*leaves, EPS), leaves, (ds, dy))
    h = 1e-2
    for n, (leaf, grad) in enumerate(zip(leaves, grads)):
        step = torch.randn(leaf.shape, generator=torch.Generator().manual_seed(n)).cuda()
        ends = []
        for sign in (1, -1):
            moved = [t.detach() for t in leaves]
            moved[n] = moved[n] + sign * h * step
            ends.append(loss(*moved))
        slope, want = (ends[0] - ends[1]) / (2 * h), float((grad.double() * step).sum())
        # central differences: the third derivative times h^2 / 6 (norm of the step times 1e-2 squared, order one values: under 1e-3 of
        # the terms' root sum), and the outputs' rounding, 2^-24 of some 240 terms of 0.3 over 2 h: 1e-5
        scale = float((grad.double().square().sum() * step.double().square().sum()).sqrt())
        assert abs(slope - want) <= 2e-3 * scale + 2e-5, (n, slope, want, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("k", [512, 509])
def test_strides_offsets_and_leading_dimensions(k):
    ops = _ops()
    g = torch.Generator().manual_seed(5)
    big = torch.randn(6, 5, 2 * k + 6, generator=g).bfloat16().cuda()
    x, res = big[..., 1:k + 1], big[..., k + 3:2 * k + 3]  # rows of a wider matrix, on odd elements
    w = torch.randn(k + 1, generator=g).bfloat16().cuda()[1:]
    want = ops.add_rmsnorm(x.contiguous(), res.contiguous(), w.clone(), EPS, quantize=True)
    for a, b in zip(ops.add_rmsnorm(x, res, w, EPS, quantize=True), want):
        assert a.shape == b.shape and torch.equal(a, b)
    xt, rt = x.transpose(0, 1), res.transpose(0, 1)  # another order of the rows, and below columns before rows
    for a, b in zip(ops.add_rmsnorm(xt, rt, w, EPS), want):
        assert torch.equal(a, b.transpose(0, 1))
    xc = torch.empty(k, 30, dtype=torch.bfloat16, device="cuda").t().copy_(x.reshape(30, k))
    assert torch.equal(ops.add_rmsnorm(xc, res.reshape(30, k), w, EPS)[1], want[1].reshape(30, k))
    one = ops.add_rmsnorm(x[2, 3], res[2, 3], w, EPS, quantize=True)  # a single row without leading dimensions
    assert one[3].shape == () and all(torch.equal(a, b[2, 3]) for a, b in zip(one, want))
    leaves = [t.clone().requires_grad_() for t in (x, res, w)]
    s, y = ops.add_rmsnorm(*leaves, EPS)
    ds, dy = big[..., 2:k + 2], torch.ones((), device="cuda", dtype=torch.bfloat16).expand(6, 5, k)  # strided, expanded
    got = torch.autograd.grad((s, y), leaves, (ds, dy), retain_graph=True)
    for a, b in zip(got, torch.autograd.grad((s, y), leaves, (ds.contiguous(), dy.contiguous()))):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_rows_of_zeros_infinities_and_nan_stay_by_themselves():
    ops = _ops()
    x, res, w, ds, dy = _inputs(12, 300, torch.bfloat16, torch.bfloat16, seed=6)
    clean = [t.clone() for t in (x, res)]
    x[2], res[2] = 0, 0
    x[4, 7], x[6, 7], res[8, 9] = float("nan"), float("inf"), float("-inf")
    others = [i for i in range(12) if i not in (2, 4, 6, 8)]
    want = ops.add_rmsnorm(*clean, w, EPS, quantize=True)
    got = ops.add_rmsnorm(x, res, w, EPS, quantize=True)
    for a, b in zip(got, want):
        assert torch.equal(a[others], b[others])
    s, y, q, s_x = got
    assert not s[2].any() and not y[2].any() and not q[2].any() and float(s_x[2]) == 1.0
    assert bool(y[4].isnan().all()) and bool(y[6, 7].isnan()) and bool(y[8, 9].isnan())
    assert torch.equal(s[4].isnan(), torch.arange(300, device="cuda") == 7)
    leaves = [t.requires_grad_() for t in (x, res)]
    out = ops.add_rmsnorm(*leaves, w, EPS)
    ref = ops.add_rmsnorm(*[t.requires_grad_() for t in clean], w, EPS)
    dx, = torch.autograd.grad(out, leaves[0], (ds, dy))
    rx, = torch.autograd.grad(ref, clean[0], (ds, dy))
    assert torch.equal(dx[others], rx[others]) and bool(dx[2].isfinite().all())


@pytest.mark.gpu
def test_rows_beyond_two_to_the_31_elements():
    """140000 rows of 16384: offsets pass 2^31 elements and 2^32 bytes."""
    announce("add_rmsnorm", 140000, 16384)
    ops = _ops()
    rows, k = 140000, 16384
    x, w = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda"), torch.ones(k, dtype=torch.bfloat16, device="cuda")
    last = [0, 65536, 131071, 131072, rows - 1]
    g = torch.Generator().manual_seed(7)
    x[last] = torch.randn(5, k, generator=g).bfloat16().cuda()
    s, y, q, s_x = ops.add_rmsnorm(x, x, w, EPS, quantize=True)
    want = ops.add_rmsnorm(x[last], x[last], w, EPS, quantize=True)
    for a, b in zip((s, y, q, s_x), want):
        assert torch.equal(a[last], b)
    from bittorch_amd import _C
    rstd = _C.add_rmsnorm(x, x, w, EPS, return_rstd=True)[-1]
    dx, _, dw = _C.add_rmsnorm_backward(s, rstd, w, x, y)
    wx, _, ww = _C.add_rmsnorm_backward(s[last], rstd[last], w, x[last], y[last])
    assert torch.equal(dx[last], wx)
    # (the other rows are zero: the same five terms in another order, each off by half a step of the result at most twice)
    assert bool(((dw.double() - ww.double()).abs() <= 2 * torch.finfo(torch.bfloat16).eps * ww.double().abs() + 1e-6).all())


@pytest.mark.gpu
def test_streams_and_captured_graphs():
    """Forward and gradient on another stream, and in two graphs captured one after the other and replayed in turn between eager calls."""
    ops = _ops()
    x, res, w, ds, dy = _inputs(65, 1000, torch.bfloat16, torch.float32, seed=8)

    def step(a, b, c, da, db):
        leaves = [t.detach().requires_grad_() for t in (a, b, c)]
        out = ops.add_rmsnorm(*leaves, EPS)
        return (*[t.detach() for t in out], *torch.autograd.grad(out, leaves, (da, db)))

    want = step(x, res, w, ds, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x, res, w, ds, dy)
        step(x, res, w, ds, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    del got
    graphs = []
    for scale in (1, 2):
        static = [t.clone() for t in (x * scale, res, w, ds, dy)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out, [t.clone() for t in step(*static)]))
    for _ in range(3):
        for graph, static, out, expect in graphs:
            for t in out:
                t.fill_(7)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, expect))
            assert all(torch.equal(a, b) for a, b in zip(step(*static), expect))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,rt", TYPES)
def test_native_and_python_calls_agree(dt, rt, monkeypatch):
    """csrc/calls.cpp and ops/fused.py, bit for bit, and each refuses a second derivative."""
    from bittorch_amd import _C, _lib
    ops = _ops()
    x, res, w, ds, dy = [t.reshape(t.shape[0] // 3, 3, -1) if t.dim() == 2 else t for t in _inputs(21, 264, dt, rt, seed=9)]
    native, got = _C._N, []
    for calls in (native, _lib._PythonCalls()):
        monkeypatch.setattr(_C, "_N", calls)
        outs = []
        for residual in (res, None):
            for weight in (w, w.float(), None):
                for flags in (dict(), dict(quantize=True, return_rowsum=True), dict(store=False, quantize=True)):
                    outs += ops.add_rmsnorm(x, residual, weight, EPS, **flags)
                    leaves = [t.clone().requires_grad_() for t in (x, residual, weight) if t is not None]
                    it = iter(leaves)
                    args = [None if t is None else next(it) for t in (x, residual, weight)]
                    out = ops.add_rmsnorm(*args, EPS, **flags)
                    outs += [t.detach() for t in out]
                    assert [t.requires_grad for t in out] == [True] * (1 + flags.get("store", True)) + [False] * (len(out) - 1 - flags.get("store", True))
                    for used, incoming in (((0, 1), (ds, dy)), ((0,), (ds,)), ((1,), (dy,))):
                        if max(used) == 1 and not flags.get("store", True):
                            continue
                        incoming = [g if i else g.to(out[0].dtype) for i, g in zip(used, incoming)]
                        grads = torch.autograd.grad([out[i] for i in used], leaves, incoming, retain_graph=True, allow_unused=True)
                        outs += [t for t in grads if t is not None]
        got.append(outs)
        leaf = x.clone().requires_grad_()
        dx, = torch.autograd.grad(ops.add_rmsnorm(leaf, res, w, EPS)[1], leaf, dy.clone().requires_grad_(), create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            dx.sum().backward()
    assert len(got[0]) == len(got[1]) > 50
    for a, b in zip(*got):
        assert a.shape == b.shape and a.dtype == b.dtype and torch.equal(a, b)


def test_refusals():
    from bittorch_amd import _C, _lib, ops
    x = torch.randn(4, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.add_rmsnorm(x, x, torch.ones(16))
    with pytest.raises(RuntimeError, match="residual shape"):
        ops.add_rmsnorm(x, x[:3])
    with pytest.raises(RuntimeError, match="residual must have x's dtype or be float32"):
        ops.add_rmsnorm(x, x.half())
    with pytest.raises(RuntimeError, match=r"weight must be 1D \[K\]"):
        ops.add_rmsnorm(x, x, torch.ones(15))
    with pytest.raises(RuntimeError, match="weight must have x's dtype or be float32"):
        ops.add_rmsnorm(x, x, torch.ones(16).bfloat16())
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        ops.add_rmsnorm(x.double(), x)
    with pytest.raises(RuntimeError, match="empty"):
        ops.add_rmsnorm(x[:0], x[:0])
    lib, addr = _lib.load(), 1 << 20  # (never read: every call ends before a launch)
    call = lambda ld=16, xd=2, res=addr, ldr=16, rd=2, wd=2, K=16, s=addr, y=addr, q=None, sx=None, rs=None, lay=0: lib.bt_add_rmsnorm(
        addr, ld, xd, res, ldr, rd, addr, wd, EPS, 4, K, s, y, None, q, sx, rs, lay, None)
    for kwargs, text in [(dict(s=None), "null"), (dict(xd=7), "dtype"), (dict(rd=1), "dtype"), (dict(wd=1), "dtype"), (dict(ld=15), "stride"),
                         (dict(ldr=8), "stride"), (dict(y=None), "no output"), (dict(q=addr), "s_x"), (dict(rs=addr), "q_rowsum"),
                         (dict(q=addr, sx=addr, lay=1, K=8), "operand order"), (dict(q=addr, sx=addr, lay=2), "operand order"),
                         (dict(K=0), "empty")]:
        assert call(**kwargs) == -1, kwargs
        assert text in _lib.last_error(), (kwargs, _lib.last_error())
    back = lambda s=addr, rd=2, w=addr, wd=2, xd=2, dx=addr, dw=None, ws=None, n=0: lib.bt_add_rmsnorm_backward(
        s, rd, addr, w, wd, addr, xd, None, 4, 16, dx, None, dw, ws, n, None)
    assert back(s=None) == -1 and back(rd=1) == -1 and back(dx=None) == -1 and back(wd=1) == -1
    assert back(dw=addr) == -2 and "workspace" in _lib.last_error()
    need = lib.bt_add_rmsnorm_backward_workspace_bytes(4, 16)
    assert need > 0 and back(dw=addr, ws=addr, n=need - 1) == -2 and back(dw=addr, ws=addr + 8, n=need) == -2
    assert lib.bt_add_rmsnorm_backward_workspace_bytes(0, 16) == 0



@pytest.mark.gpu
@pytest.mark.parametrize("rows,k", [((1 << 24) + 5, 4), ((1 << 26) + 3, 8)])
def test_more_rows_than_one_dimension_of_a_grid_has_threads(rows, k):
    """A workgroup, or a wave, of its own for each of that many rows passes 2^32 threads."""
    announce("add_rmsnorm", rows, k)
    ops = _ops()
    g = torch.Generator(device="cuda").manual_seed(1)
    mk = lambda: torch.randn(rows, k, generator=g, device="cuda").bfloat16()
    x, res, dy, w = mk(), mk(), mk(), (1 + 0.2 * torch.randn(k, generator=g, device="cuda")).bfloat16()
    ends = [0, 1, 2, (1 << 20) - 1, 1 << 20, (1 << 22) - 1, 1 << 22, rows // 2, rows - 3, rows - 2, rows - 1]
    got = ops.add_rmsnorm(x, res, w, EPS, quantize=True, return_rowsum=True)
    assert torch.equal(got[0], (x.float() + res.float()).bfloat16())
    for a, b in zip(got, ops.add_rmsnorm(x[ends], res[ends], w, EPS, quantize=True, return_rowsum=True)):
        assert torch.equal(a[ends], b)
    s, y = got[0], got[1]
    # (each row on its own, in 32 bits: a wrong row is off by more than two steps of bf16)
    want = s.float() * (s.float().square().mean(-1, keepdim=True) + EPS).rsqrt() * w.float()
    assert float(((y.float() - want).abs() - 2.0 ** -7 * want.abs()).max()) <= 1e-30
    del got, want, y
    leaves = [t.requires_grad_() for t in (x, w)]
    dx, dw = torch.autograd.grad(ops.add_rmsnorm(x, res, w, EPS)[1], leaves, dy)
    few = x.detach()[ends].requires_grad_()
    few_dx, = torch.autograd.grad(ops.add_rmsnorm(few, res[ends], w, EPS)[1], few, dy[ends])
    assert torch.equal(dx[ends], few_dx) and bool(dx.isfinite().all())
    terms, size = torch.zeros(k, dtype=torch.float64, device="cuda"), torch.zeros(k, dtype=torch.float64, device="cuda")
    for a, b in zip(s.split(1 << 22), dy.split(1 << 22)):
        t = a.double()
        t = b.double() * t * (t.square().mean(-1, keepdim=True) + EPS).rsqrt()
        terms += t.sum(0)
        size += t.abs().sum(0)
    # a chain of rows / 64 additions, each rounded by half a step of the sum so far, and bf16's own
    bound = 2.0 ** -24 * (rows / 64 + 80) * size
    assert bool(((dw.double() - terms).abs() <= bound + 2.0 ** -8 * terms.abs()).all())


@pytest.mark.gpu
def test_a_weight_of_more_columns_than_one_dimension_of_a_grid_has_threads():
    announce("column sum", (1 << 28) + 70)
    ops = _ops()
    k = (1 << 28) + 70
    x = torch.randn(1, k, device="cuda", generator=torch.Generator(device="cuda").manual_seed(2)).bfloat16()
    w = torch.ones(k, device="cuda", dtype=torch.bfloat16).requires_grad_()
    dy = torch.ones(1, k, device="cuda", dtype=torch.bfloat16)
    dw, = torch.autograd.grad(ops.add_rmsnorm(x, None, w, EPS)[1], w, dy)
    r = 1 / (x.double().square().mean() + EPS).sqrt()
    off = 0.0
    for a, b in zip(dw.split(1 << 26), x[0].split(1 << 26)):
        want = b.double() * r
        off = max(off, float(((a.double() - want).abs() - (2.0 ** -8 + 1e-6) * want.abs()).max()))
    assert off <= 1e-30
