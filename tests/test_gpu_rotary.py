"""``ops.rotary`` on the GPU against its definition in 64 bits, forward and backward, and what a caller may do with it."""
import pytest
import torch

from conftest import announce
from test_attention import complex_turn

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
# tokens, heads, kv_heads, dim, rotary_dim, interleaved: one token; heads that fill no 16 bytes; a part of the head; rotary_dim 2; many tokens
SHAPES = [(1, 20, 20, 128, 128, False), (1, 1, 1, 2, 2, True), (3, 5, 1, 71, 70, True), (7, 4, 2, 71, 70, False), (33, 12, 4, 80, 32, True),
          (65, 3, 3, 96, 48, False), (5, 2, 1, 250, 2, False), (1025, 6, 2, 64, 64, True), (2050, 3, 1, 40, 16, False), (4097, 2, 1, 128, 128, False),
          (9, 2, 2, 1000, 1000, False), (300, 1, 7, 12, 8, True)]


def _ops():
    from bittorch_amd import ops
    return ops


def _half(t):
    return torch.finfo(t).eps / 2


def assert_turned(got, x, positions, inv_freq, interleaved, amplitude=1.0):
    """The angle in turns is rounded to 32 bits once (half a turn at most: pi u), cosine and sine are within 4 u and one for the amplitude, the two
    products and their sum round: under 12 u of the pair's magnitudes; the angle itself in 64 bits.  Then the type's rounding."""
    x = x.detach()
    want = complex_turn(x, positions, inv_freq, interleaved, amplitude)
    n = 2 * inv_freq.shape[0]
    mag = x.double().abs()
    part = mag[..., :n]
    pair = (part[..., 0::2] + part[..., 1::2]).repeat_interleave(2, -1) if interleaved else (part[..., :n // 2] + part[..., n // 2:]).repeat(*(1,) * (x.dim() - 1), 2)
    tol = torch.zeros_like(mag)
    tol[..., :n] = abs(amplitude) * pair * (12 * U + float(positions.abs().max()) * 2.0 ** -49)
    bound = tol + _half(got.dtype) * (want.abs() + tol) + torch.finfo(got.dtype).smallest_normal * _half(got.dtype) * 2
    off = (got.detach().double() - want).abs() - bound
    assert got.shape == x.shape and got.dtype == x.dtype and not bool((off > 0).any()) and not bool(got.isnan().any()), float(off.max())
    assert torch.equal(got[..., n:], x[..., n:])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens,heads,kv,dim,rot,interleaved", SHAPES)
def test_forward_and_gradient(dt, tokens, heads, kv, dim, rot, interleaved):
    announce("rotary", tokens, heads, kv, dim, rot, interleaved, dt)
    ops, g = _ops(), torch.Generator().manual_seed(tokens + dim)
    q, k, dq, dk = (torch.randn(tokens, h, dim, generator=g).to(dt).cuda() for h in (heads, kv, heads, kv))
    pos = torch.randint(-5, 200000, (tokens,), generator=g).cuda()
    inv_freq = ops.rotary_frequencies(rot, device="cuda")[0]
    got = ops.rotary(q, k, pos, inv_freq, interleaved, 1.125)
    for a, x in zip(got, (q, k)):
        assert_turned(a, x, pos, inv_freq, interleaved, 1.125)
    assert torch.equal(ops.rotary(q, None, pos.int(), inv_freq, interleaved, 1.125), got[0])
    leaves = q.clone().requires_grad_(), k.clone().requires_grad_()
    out = ops.rotary(*leaves, pos, inv_freq, interleaved, 1.125)
    assert all(torch.equal(a, b) for a, b in zip(out, got))
    for a, x in zip(torch.autograd.grad(out, leaves, (dq, dk)), (dq, dk)):
        assert_turned(a, x, -pos, inv_freq, interleaved, 1.125)
    # linear in q: the difference of two calls along dq is the derivative along it (32 bits: 4 roundings of values up to 40 and the bound above)
    if dt == torch.float32:
        v = torch.randn(tokens, heads, dim, generator=g).cuda()
        turned = ops.rotary(q, None, pos, inv_freq, interleaved, 1.125)
        along = (ops.rotary(q + v, None, pos, inv_freq, interleaved, 1.125) - turned).double()
        grad, = torch.autograd.grad(ops.rotary(leaves[0], None, pos, inv_freq, interleaved, 1.125), leaves[0], dq)
        size = (q.abs() + v.abs()).double().norm() * dq.double().norm()
        assert abs(float((along * dq.double()).sum() - (v.double() * grad.double()).sum())) < 64 * U * float(size)


def test_far_positions_and_frequencies_in_32_bits():
    ops = _ops()
    q = torch.randn(6, 2, 64, device="cuda")
    pos = torch.tensor([0, 1, -1, 999983, 10 ** 7, 2 ** 31 - 1], device="cuda")
    f = ops.rotary_frequencies(64, scaling=dict(kind="ramp", factor=8, original=4096), device="cuda")
    assert_turned(ops.rotary(q, None, pos, *f[:1], False, f[1]), q, pos, f[0], False, f[1])
    f32 = f[0].float()
    assert_turned(ops.rotary(q, None, pos, f32), q, pos, f32, False)


def test_views_are_read_in_place_and_broadcast_positions():
    ops = _ops()
    b, t, heads, kv, dim = 3, 17, 4, 2, 64
    qkv = torch.randn(b, t, (heads + 2 * kv) * dim, device="cuda").bfloat16()
    q, k, _ = (x.unflatten(-1, (-1, dim)) for x in qkv.split([heads * dim, kv * dim, kv * dim], -1))
    f = ops.rotary_frequencies(dim, device="cuda")[0]
    pos = torch.arange(t, device="cuda")
    want = ops.rotary(q.contiguous(), k.contiguous(), pos.expand(b, t).contiguous(), f)
    assert all(torch.equal(x, y) for x, y in zip(ops.rotary(q, k, pos, f), want))
    assert all(torch.equal(x, y) for x, y in zip(ops.rotary(q, k, pos[None], f), want))
    # heads before tokens, reversed features, an odd start, one row for all
    swapped = q.transpose(1, 2).contiguous().transpose(1, 2)
    assert torch.equal(ops.rotary(swapped, None, pos, f), want[0])
    odd = torch.empty(b * t * heads * dim + 1, dtype=torch.bfloat16, device="cuda")[1:].view(b, t, heads, dim).copy_(q)
    assert torch.equal(ops.rotary(odd, None, pos, f), want[0])
    strided = torch.empty(b, t, heads, 2 * dim, dtype=torch.bfloat16, device="cuda")[..., ::2].copy_(q)
    assert torch.equal(ops.rotary(strided, None, pos, f), want[0])
    row = torch.randn(1, 1, heads, dim, device="cuda", requires_grad=True)
    out = ops.rotary(row.expand(b, t, heads, dim), None, pos, f)
    weight = torch.randn(b, t, heads, dim, device="cuda")
    grad, = torch.autograd.grad(out, row, weight)
    full = complex_turn(weight, -pos.expand(b, t), f, False)
    assert float((grad.double() - full.sum((0, 1), keepdim=True)).abs().max()) < 64 * 51 * U * float(weight.abs().max())
    # a gradient that is a view: expanded, transposed
    leaf = q.float().requires_grad_()
    grad, = torch.autograd.grad(ops.rotary(leaf, None, pos, f).sum(), leaf)
    assert_turned(grad, torch.ones_like(leaf), -pos.expand(b, t), f, False)
    grad, = torch.autograd.grad(ops.rotary(leaf, None, pos, f).transpose(1, 2), leaf, weight.transpose(1, 2))
    assert_turned(grad, weight, -pos.expand(b, t), f, False)


def test_partial_gradients_and_what_is_refused():
    ops = _ops()
    q, k = torch.randn(5, 2, 8, device="cuda", requires_grad=True), torch.randn(5, 1, 8, device="cuda")
    pos, f = torch.arange(5, device="cuda"), torch.ones(4, device="cuda")
    a, b = ops.rotary(q, k, pos, f)
    assert torch.autograd.grad(a, q, torch.ones_like(a), retain_graph=True)[0] is not None
    assert torch.autograd.grad((a, b), q, (torch.ones_like(a), torch.ones_like(b)), allow_unused=True)[0] is not None
    kk = k.clone().requires_grad_()
    a, b = ops.rotary(q.detach(), kk, pos, f)
    assert_turned(torch.autograd.grad(b, kk, torch.ones_like(b))[0], torch.ones_like(kk), -pos, f, False)
    a, b = ops.rotary(q, kk, pos, f)
    assert_turned(torch.autograd.grad(b, kk, torch.ones_like(b), retain_graph=True)[0], torch.ones_like(kk), -pos, f, False)
    assert torch.autograd.grad(b, q, torch.ones_like(b), allow_unused=True)[0] is None or not torch.autograd.grad(ops.rotary(q, kk, pos, f)[1].sum(), q, allow_unused=True)[0].any()
    # the positions were changed between the two passes
    a = ops.rotary(q, None, pos, f)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        a.sum().backward()
    pos.sub_(1)
    dq, = torch.autograd.grad(ops.rotary(q, None, pos, f), q, torch.ones(5, 2, 8, device="cuda", requires_grad=True), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiate twice"):
        dq.sum().backward()
    from torch.autograd import forward_ad
    with forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        ops.rotary(forward_ad.make_dual(q.detach(), torch.ones_like(q)), None, pos, f)
    for args in ((q.detach().double(), None, pos, f), (q, None, pos.cpu(), f), (q, None, pos, f.cpu()), (q, k.half(), pos, f), (q, None, pos[:3], f)):
        with pytest.raises(RuntimeError):
            ops.rotary(*args)
    assert ops.rotary(q.detach()[:0], k[:0], pos[:0], f)[1].shape == (0, 1, 8)


def test_another_stream_and_captured_graphs():
    """Forward and gradient on another stream, and in two graphs replayed in turn between eager calls; replays follow the positions."""
    ops = _ops()
    q, k = (torch.randn(40, h, 64, device="cuda").half() for h in (4, 2))
    pos, f = torch.arange(40, device="cuda"), ops.rotary_frequencies(64, device="cuda")[0]
    dq, dk = torch.randn_like(q), torch.randn_like(k)

    def step(a, b, at):
        leaves = [t.detach().requires_grad_() for t in (a, b)]
        out = ops.rotary(*leaves, at, f)
        return (*[t.detach() for t in out], *torch.autograd.grad(out, leaves, (dq, dk)))

    want = step(q, k, pos)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(q, k, pos)
        step(q, k, pos)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want))
    graphs = []
    for scale in (1, 2):
        static = (q * scale).clone(), k.clone(), pos.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(*static)
        graphs.append((graph, static, out))
    for i in range(3):
        for graph, static, out in graphs:
            static[2].add_(1000 * i)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(out, step(*static)))
