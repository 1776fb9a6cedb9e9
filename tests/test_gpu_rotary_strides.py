"""``ops.rotary`` on rows whose dimensions of one entry have strides of their own: what attention over one token a sequence hands back."""
import pytest
import torch

from conftest import announce
from test_gpu_rotary import TYPES, _ops, assert_turned

pytestmark = pytest.mark.gpu


def _grown(shape, strides, dt, seed):
    """A tensor of these strides inside a larger buffer of other values."""
    need = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    buffer = torch.randn(need, generator=torch.Generator().manual_seed(seed)).to(dt).cuda()
    return buffer.as_strided(shape, strides)


# leading dimensions, and the strides of the rows that come back as a gradient (heads 3, 16 features)
LEADS = [((4, 1), (48, 16, 16, 1)), ((4, 1), (48, 7, 16, 1)), ((4, 1), (96, 1, 16, 1)), ((1, 4), (5, 48, 16, 1)), ((1, 4), (5, 16, 64, 1)), ((1, 1), (3, 5, 16, 1)),
         ((2, 1, 3), (144, 16, 48, 16, 1)), ((2, 1, 3), (144, 3, 48, 16, 1)), ((1, 2, 3, 1), (1, 144, 48, 1, 16, 1)), ((2, 3), (48, 96, 16, 1)), ((1,), (2, 16, 1)), ((4, 1), (1, 16, 16, 4))]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("lead,strides", LEADS)
def test_gradients_and_rows_of_any_strides(dt, lead, strides):
    announce("rotary strides", lead, strides, dt)
    ops = _ops()
    shape = (*lead, 3, 16)
    pos = (torch.arange(torch.Size(lead).numel(), device="cuda") * 37 + 5).view(lead)
    f = ops.rotary_frequencies(16, device="cuda")[0]
    x, y = (_grown(shape, strides, dt, s) for s in (1, 2))
    for a in (ops.rotary(x, None, pos, f), *ops.rotary(x, x, pos, f)):
        assert_turned(a, x, pos, f, False)
    q, k = (torch.randn(shape, device="cuda").to(dt).requires_grad_() for _ in range(2))
    for a in (lambda: ops.rotary(q, None, pos, f), lambda: ops.rotary(q, k.detach(), pos, f)[0], lambda: ops.rotary(q, k, pos, f)[0]):
        grad, = torch.autograd.grad(a(), q, x)
        assert_turned(grad, x, -pos, f, False)
    grad, = torch.autograd.grad(ops.rotary(q.detach(), k, pos, f)[1], k, x)
    assert_turned(grad, x, -pos, f, False)
    for one, other in ((x, y), (x, y.contiguous()), (x.clone(memory_format=torch.contiguous_format), y)):
        dq, dk = torch.autograd.grad(ops.rotary(q, k, pos, f), (q, k), (one, other))
        assert_turned(dq, one, -pos, f, False)
        assert_turned(dk, other, -pos, f, False)


@pytest.mark.parametrize("dt", TYPES)
def test_one_token_of_each_sequence_through_attention(dt):
    """[sequences, 1, heads, D], as a step that is trained on calls it: the gradients through heads before tokens."""
    ops = _ops()
    b, heads, dim = 4, 8, 64
    f = ops.rotary_frequencies(dim, device="cuda")[0]
    pos = torch.tensor([[3], [700], [0], [41]], device="cuda")
    q, k = (torch.randn(b, 1, heads, dim, device="cuda").to(dt).requires_grad_() for _ in range(2))
    w, u = (torch.randn(b, heads, 1, dim, device="cuda").to(dt) for _ in range(2))
    out = ops.rotary(q, k, pos, f)
    for a, x, g in zip(torch.autograd.grad([t.transpose(1, 2) for t in out], (q, k), (w, u)), (q, k), (w, u)):
        assert_turned(a, g.transpose(1, 2), -pos, f, False)
    grad, = torch.autograd.grad(ops.rotary(q, None, pos, f).transpose(1, 2), q, w)
    assert_turned(grad, w.transpose(1, 2), -pos, f, False)
    grad, = torch.autograd.grad(ops.rotary(q.detach(), k, pos, f)[1].transpose(1, 2), k, u)
    assert_turned(grad, u.transpose(1, 2), -pos, f, False)
