"""``ops.cached_attention`` on the GPU where a rule of its kernels ends: pages outside the cache behind many others, weights far below a row's
largest, logits and scales at the ends of 32 bits."""
import math

import pytest
import torch

from conftest import announce
from test_attention_infinities import KINDS, check, filled
from test_gpu_attention import Batch, _ops
from test_gpu_rotary import U, _half

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _set_keys(b, keys, values=None):
    """The one sequence's keys [places, dim] of every key head (and values), in the caches' order."""
    from bittorch_amd.ops.attention import _natural, _tiled
    kn, vn = (t.clone() for t in _natural(b.k_cache, b.v_cache))
    places = torch.arange(keys.shape[0], device="cuda")
    number, at = b.table[0][places // b.page].long(), places % b.page
    kn[number, :, at, :b.dim] = keys.to(b.dt)[:, None]
    if values is not None:
        vn[number, :, at, :b.dim] = values.to(b.dt)[:, None]
    b.k_cache, b.v_cache = (t.contiguous() for t in _tiled(kn, vn))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("held", [2049, 2090, 2120, 2140])
def test_a_page_outside_the_cache_behind_64_others(dt, held):
    """The 65th page of a chunk and the 66th, with so few tiles behind the 64th that not every wave of a workgroup has one: all of the sequence's rows are not a
    number, the other sequences' as they were.  (101 sequences of 8 key heads: a chunk holds a whole sequence.)"""
    announce("bad page", held, dt)
    b = Batch([held] + [5, 40] * 50, [1] * 101, 32, 8, 128, 32, dt, width=72)
    want, want_lse = b.attend(starts=False, return_lse=True)
    b.check(want, want_lse)
    good = b.table
    for column in range(64, -(-held // 32)):
        for wrong in (-1, b.k_cache.shape[0]):
            b.table = good.clone()
            b.table[0, column] = wrong
            for starts in (False, True):
                out, lse = b.attend(starts=starts, return_lse=True)
                assert out[0].isnan().all() and lse[0].isnan().all(), (column, starts)
                assert torch.equal(out[1:], want[1:]) and torch.equal(lse[1:], want_lse[1:])


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("prefix", [2049, 2090])
def test_a_prefix_page_outside_the_cache_behind_64_others(dt, prefix):
    """200 tokens of 4 heads to each of 8 key heads: a workgroup sees the whole prefix."""
    announce("bad prefix page", prefix, dt)
    b = Batch([30] * 200, [1] * 200, 32, 8, 64, 32, dt, prefix)
    b.check(*b.attend(starts=False, return_lse=True))
    b.prefix_table = b.prefix_table.clone()
    b.prefix_table[64] = -1
    for starts in (False, True):
        out, lse = b.attend(starts=starts, return_lse=True)
        assert out.isnan().all() and lse.isnan().all()


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new,wide", [(1, False), (40, True)])
def test_the_smallest_scales(dt, new, wide):
    """All logits next to zero: means of the values, and the logarithm of the number of places."""
    announce("smallest scale", new, wide, dt)
    b = Batch([400], [new], 2, 1, 32, 32, dt).widened(wide)
    for scale in (1e-30, 1e-38):
        out, lse = b.attend(return_lse=True, scale=scale)
        b.check(out, lse, scale=scale)


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new,wide", [(1, False), (40, False), (40, True), (300, True)])
def test_logits_beyond_10_to_the_8(dt, new, wide):
    """Logits near 1.2e8, where 32 bits step by 8 and a weight's exponent by 16: what they make of it, results are means of the values."""
    announce("large logits", new, wide, dt)
    b = Batch([400], [new], 2, 1, 32, 32, dt).widened(wide)
    keys = torch.zeros(400, 32, device="cuda")
    keys[:, 0] = 58000.0 if dt != torch.bfloat16 else 57344.0
    keys[50:, 1] = 8.0
    values = torch.ones(400, 32, device="cuda")
    _set_keys(b, keys, values)
    b.q.zero_()
    b.q[..., 0], b.q[..., 1] = 2048.0, 1.0
    out = b.attend(scale=1.0)
    # (equal values: weights over their sum, whatever they are, rounded once each)
    assert bool(((out.double() - 1).abs() <= 3 * _half(dt) + 512 * U).all()), out.double().flatten()[:3]


@pytest.mark.parametrize("above", [15.0, 17.5])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new,wide", [(1, False), (40, False), (40, True), (300, True)])
def test_one_key_far_above_many(dt, new, wide, above):
    """One key 15 or 17.5 above 20000 others, whose weights of 2^-21.6 or 2^-25.2 have 6e-3 or 5e-4 of the sum together: a value that they alone hold comes out
    to the type's precision.  The logits are exact, so every weight is the exponential of one number: 4 u, its argument of up to 26 rounds twice (52 u), and the
    sums have as many additions as there are keys and a few dozen where parts are joined; weights and result are rounded to the type once each, fp16 weights by
    2^-32 of a row's largest at least where rows are taken as many, by 2^-40 where they are not."""
    announce("far above", new, wide, above, dt)
    held = 20000
    b = Batch([held], [new], 2, 1, 32, 64, dt).widened(wide)
    keys, values = torch.zeros(held, 32, device="cuda"), torch.zeros(held, 32, device="cuda")
    keys[0, 0] = above
    values[0, 1], values[1:, 0], values[1:, 2] = 1, 1, torch.arange(1, held, device="cuda") % 2
    _set_keys(b, keys, values)
    b.q.zero_()
    b.q[..., 0] = 1
    out, lse = b.attend(return_lse=True, scale=1.0)
    others = (held - new + torch.arange(new, device="cuda")).double()[:, None]     # seen besides the first
    total = math.exp(above) + others
    off = (held + 64 + 56) * U
    for f, want in ((0, others / total), (1, math.exp(above) / total), (2, (others / 2).ceil() / total)):
        floor = held * 2.0 ** (-32 if wide else -40) if dt == torch.float16 else 0.0
        bound = (want * (2 * off + _half(dt)) + floor) * (1 + _half(dt)) + want * _half(dt)
        assert bool(((out[..., f].double() - want).abs() <= bound).all()), (f, float(((out[..., f].double() - want).abs() / want).max()))
    assert not out[..., 3:].any()
    assert bool(((lse.double() - total.log()).abs() <= off + 4 * U * 18).all())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("kind", KINDS)
def test_infinite_keys_and_values(kind, dt):
    """As on the CPU, in both kernels: also with 23 tokens of the sequence in question, of which two that see the places are asked."""
    announce("infinite", kind, dt)
    q, kc, vc, table, lengths = filled(kind, dt, "cuda")
    check(kind, *_ops().cached_attention(q, kc, vc, table, lengths, return_lse=True))
    starts = torch.tensor([0, 1, 24, 25], dtype=torch.int32, device="cuda")
    rows = torch.cat((q[:1], q[1:2].expand(23, 2, 16), q[2:]))
    for width in (2, 1 << 21):  # (so many places that rows are taken as many)
        wide = torch.cat((table, torch.full((3, width - 2), -7, dtype=torch.int32, device="cuda")), 1)
        out, lse = _ops().cached_attention(rows, kc, vc, wide, lengths, starts, return_lse=True)
        for i in (10, 23):  # (their places are the 27th and the last: both see the 21st and 22nd)
            check(kind, *(torch.stack((t[0], t[i], t[24])) for t in (out, lse)))


def test_the_same_bits_on_every_call():
    """Both kernels and every join, called again between other work."""
    for held, new, prefix in (([2000] * 20, [1] * 20, 5000), ([1500, 900, 700, 1200], [256] * 4, 0), ([30000], [1], 0), ([700, 300, 5], [200, 9, 1], 2500)):
        b = Batch(held, new, 8, 2, 128, 64, torch.bfloat16, prefix)
        for wide in (False, True):
            first = b.widened(wide).attend(return_lse=True)
            for _ in range(8):
                torch.randn(1 << 22, device="cuda").sort()
                assert all(torch.equal(x, y) for x, y in zip(first, b.attend(return_lse=True)))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("tokens", [70, 4001, 70000])
def test_a_batch_that_is_mostly_padding(dt, tokens):
    """Rows behind the last sequence: up to many times the batch, all of them cleared, whatever they held."""
    announce("padding", tokens, dt)
    ops = _ops()
    b = Batch([40, 10, 33], [1, 9, 2], 3, 1, 33, 32, dt)
    want, want_lse = b.attend(return_lse=True)
    f = ops.rotary_frequencies(32, device="cuda")[0]
    q = torch.full((tokens, 3, 33), math.nan, dtype=dt, device="cuda")
    q[:12] = b.q
    k, v = (torch.randn(tokens, 1, 33, device="cuda").to(dt) for _ in range(2))
    for _ in range(2):
        held = [torch.full((tokens, 3, 33), math.nan, dtype=dt, device="cuda") for _ in range(3)]  # (what the results' memory holds)
        del held
        out, lse = b.attend(q, return_lse=True)
        assert not out[12:].any() and bool((lse[12:] == -math.inf).all())
        b.check(out, lse)
        assert torch.equal(out[:12], want) and torch.equal(lse[:12], want_lse)
        kc, vc = b.k_cache.clone(), b.v_cache.clone()
        turned = ops.cache_append(k, v, kc, vc, b.table, b.lengths, b.q_starts, q, f)
        assert not turned[12:].any() and bool(turned[:12].isfinite().all())
