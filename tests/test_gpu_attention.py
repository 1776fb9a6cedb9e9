"""``ops.cache_append`` and ``ops.cached_attention`` on the GPU against their definitions in 64 bits.

Everything in the caches that no sequence holds is not a number, so whatever a kernel reads too much shows.
"""
import math

import pytest
import torch

from conftest import announce
from test_gpu_rotary import U, _half, assert_turned

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _ops():
    from bittorch_amd import ops
    return ops


def natural(cache_k, cache_v):
    from bittorch_amd.ops.attention import _natural
    return _natural(cache_k, cache_v)


class Batch:
    """Sequences on scattered pages, each with `held` places of which the last `new` are new; a prefix."""

    def __init__(self, held, new, heads, kv, dim, page, dt, prefix=0, seed=0, spare=2, empty=False, width=None, std=1.0):
        from bittorch_amd import _C
        from bittorch_amd.ops.attention import _tiled
        g = torch.Generator().manual_seed(seed * 1009 + sum(held) + dim)
        self.held, self.new, self.heads, self.kv, self.dim, self.page, self.dt, self.prefix = held, new, heads, kv, dim, page, dt, prefix
        pages = lambda n: -(-n // page)  # noqa: E731
        total = sum(map(pages, held)) + pages(prefix) + spare
        order = torch.randperm(total, generator=g).int()
        padded = _C.cache_head_dim(dt, dim)
        k, v = (torch.full((total, kv, page, padded), math.nan) for _ in range(2))
        self.width = width or max(1, max(map(pages, held)))
        table, at = torch.full((len(held), self.width), -7, dtype=torch.int32), pages(prefix)
        self.keys, self.values = [], []  # of every sequence, prefix first, 64 bits
        pre = [(torch.randn(prefix, kv, dim, generator=g) * std).to(dt) for _ in range(2)]

        def put(rows, places, values, number):
            for i in range(0, values.shape[0], page):
                part = values[i:i + page].float().transpose(0, 1)
                rows[number[i // page], :, :part.shape[1]] = 0
                rows[number[i // page], :, :part.shape[1], :dim] = part

        for t, p in zip((k, v), pre):
            put(t, prefix, p, order[:pages(prefix)].long())
        for s, n in enumerate(held):
            mine = order[at:at + pages(n)]
            at += pages(n)
            table[s, :len(mine)] = mine
            rows = [(torch.randn(n, kv, dim, generator=g) * std).to(dt) for _ in range(2)]
            if not empty:
                for t, r in zip((k, v), rows):
                    put(t, n, r, mine.long())
            self.keys.append(torch.cat((pre[0], rows[0])).double().cuda())
            self.values.append(torch.cat((pre[1], rows[1])).double().cuda())
        kt, vt = _tiled(k.to(dt), v.to(dt))
        self.k_cache, self.v_cache, self.table = kt.contiguous().cuda(), vt.contiguous().cuda(), table.cuda()
        self.lengths = torch.tensor(held, dtype=torch.int32, device="cuda")
        self.starts = [0]
        for n in new:
            self.starts.append(self.starts[-1] + n)
        self.tokens = self.starts[-1]
        self.q_starts = torch.tensor(self.starts, dtype=torch.int32, device="cuda")
        self.prefix_table = order[:pages(prefix)].cuda() if prefix else None
        self.q = torch.randn(self.tokens, heads, dim, generator=g).to(dt).cuda()

    def widened(self, wide=True):
        """Tables that may hold so many places that sequences of many rows are taken as such."""
        if wide:
            width = max(self.width, -(-2 ** 31 // (self.tokens * self.heads * self.dim * self.page)))
            table = torch.full((len(self.held), width), -7, dtype=torch.int32, device="cuda")
            table[:, :self.width] = self.table
            self.table, self.width = table, width
        return self

    def attend(self, q=None, starts=True, **more):
        return _ops().cached_attention(self.q if q is None else q, self.k_cache, self.v_cache, self.table, self.lengths, self.q_starts if starts else None,
                                       prefix_table=self.prefix_table, prefix_length=self.prefix, **more)

    def check(self, out, lse, q=None, scale=None, weights_in_type=True):
        """Each row against the definition.  A logit is a sum of D products and a product with scale / ln 2: (D + 4) u of its magnitudes, and the
        exponential's argument and value round three times, its argument up to the largest logit; each weight is rounded to the type at most once; the
        sums have at most as many additions as there are keys, and a few dozen where parts are joined."""
        q = (self.q if q is None else q).double()
        scale = self.dim ** -0.5 if scale is None else scale
        group = self.heads // self.kv
        for s, (n, held) in enumerate(zip(self.new, self.held)):
            if n == 0:
                continue
            rows = q[self.starts[s]:self.starts[s] + n]
            k, v = (t[s].repeat_interleave(group, 1) for t in (self.keys, self.values))
            x = torch.matmul(rows.transpose(0, 1), k.permute(1, 2, 0)) * scale                      # [heads, new, keys]
            size = torch.matmul(rows.abs().transpose(0, 1), k.abs().permute(1, 2, 0)) * scale
            keys = k.shape[0]
            if keys == 0:
                assert not out[self.starts[s]:self.starts[s] + n].any() and (lse is None or bool((lse[self.starts[s]:self.starts[s] + n] == -math.inf).all()))
                continue
            seen = torch.arange(keys, device="cuda")[None] < self.prefix + held - n + 1 + torch.arange(n, device="cuda")[:, None]
            some = seen.any(-1)
            x = x.masked_fill(~seen, -math.inf)
            want_lse = x.logsumexp(-1)
            p = (x - want_lse[..., None]).exp().masked_fill(~seen, 0)
            p = torch.where(some[:, None], p, torch.zeros_like(p))
            want = torch.matmul(p, v.transpose(0, 1)).transpose(0, 1)
            spread = torch.matmul(p, v.abs().transpose(0, 1)).transpose(0, 1)
            top = x.masked_fill(~seen, 0).abs().amax(-1)
            delta = ((self.dim + 4) * U * size.masked_fill(~seen, 0).amax(-1) + 6 * U * (top + 1)) + (keys + 64) * U   # [heads, new]
            off = delta.transpose(0, 1)[..., None]
            tol = spread * (2 * off + (_half(self.dt) if weights_in_type and self.dt != torch.float32 else 0.0))
            got = out[self.starts[s]:self.starts[s] + n].double()
            bound = tol + _half(self.dt) * (want.abs() + tol) + torch.finfo(self.dt).smallest_normal * _half(self.dt)
            over = (got - want).abs() - bound
            assert not bool(got.isnan().any()) and not bool((over > 0).any()), (s, n, held, float(over.max()))
            if lse is not None:
                got = lse[self.starts[s]:self.starts[s] + n].double().transpose(0, 1)
                assert torch.equal(got.isinf(), (~some).expand_as(got)) and not bool(got.isnan().any())
                over = ((got - want_lse).abs() - delta - 4 * U * (want_lse.abs() + top))[:, some]
                assert not bool((over > 0).any()), (s, float(over.max()))


# held, new, heads, kv, dim, page, prefix
DECODE = [([1], [1], 1, 1, 128, 64, 0), ([500], [1], 20, 20, 128, 64, 0), ([31, 32, 33, 1, 64, 65], [1] * 6, 8, 2, 64, 32, 0), ([700, 3, 129, 128], [1] * 4, 32, 2, 128, 64, 0),
          ([5, 600], [1, 1], 34, 1, 80, 32, 77), ([260, 1000], [1, 1], 6, 3, 33, 256, 0), ([200], [1], 4, 1, 256, 64, 300), ([90, 2], [1, 1], 5, 5, 1, 32, 64), ([300, 0, 20], [1, 1, 1], 4, 4, 96, 64, 0),
          ([300, 0, 20], [1, 1, 1], 4, 2, 192, 64, 33), ([5000], [1], 8, 1, 160, 64, 0), ([2100, 9], [1, 1], 16, 8, 128, 32, 129)]
RAGGED = [([7], [7], 4, 2, 64, 32, 0), ([50, 0, 33, 200], [3, 0, 33, 1], 6, 2, 80, 32, 0), ([400, 129, 64], [100, 129, 2], 8, 8, 128, 64, 0), ([17, 300, 5], [17, 9, 5], 10, 2, 72, 32, 1000),
          ([90, 600], [70, 200], 4, 1, 256, 64, 40), ([1, 2, 3, 0, 4, 5] * 15, [1, 1, 2, 0, 4, 2] * 15, 3, 1, 20, 32, 50), ([700], [513], 12, 3, 128, 128, 0), ([12, 6], [10, 6], 16, 1, 64, 32, 5),
          ([2, 40], [6, 40], 4, 2, 64, 32, 0), ([1300, 1111], [1300, 260], 8, 2, 128, 64, 200), ([640], [640], 2, 2, 40, 64, 0)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("held,new,heads,kv,dim,page,prefix", DECODE)
def test_one_token_each(dt, held, new, heads, kv, dim, page, prefix):
    announce("attend one", held, heads, kv, dim, page, prefix, dt)
    b = Batch(held, new, heads, kv, dim, page, dt, prefix)
    out, lse = b.attend(starts=False, return_lse=True)
    b.check(out, lse)
    same = b.attend(return_lse=True)
    b.check(*same)
    assert torch.equal(b.attend(starts=False), out)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("held,new,heads,kv,dim,page,prefix", RAGGED)
def test_several_tokens_each(dt, held, new, heads, kv, dim, page, prefix, wide):
    announce("attend several", held[:9], new[:9], heads, kv, dim, page, prefix, dt, wide)
    b = Batch(held, new, heads, kv, dim, page, dt, prefix).widened(wide)
    b.check(*b.attend(return_lse=True))
    b.check(*b.attend(return_lse=True, scale=0.3), scale=0.3)


# every number of 32-feature blocks with many rows, odd heads; more than 64 sequences, some of them of many rows; many heads to a key head
WIDE = [([90, 70], [80, 64], 4, 2, d, 64, 33) for d in (1, 8, 31, 33, 64, 65, 96, 100, 129, 160, 161, 192, 200, 224, 225, 256)] + [
    ([50, 3, 200, 9] * 20, [50, 1, 90, 9] * 20, 4, 2, 64, 32, 0), ([50, 3, 200, 9] * 17, [50, 1, 90, 0] * 17, 6, 2, 40, 32, 21), ([6000, 300], [300, 40], 2, 1, 64, 64, 0),
    ([3000], [40], 2, 2, 128, 64, 0), ([700, 2500, 40, 5], [129, 65, 33, 1], 3, 3, 128, 32, 0), ([50, 3, 200, 9] * 80, [50, 1, 90, 9] * 80, 4, 2, 64, 32, 0),
    ([700, 350] * 10, [300, 350] * 10, 8, 8, 64, 64, 0)]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("held,new,heads,kv,dim,page,prefix", WIDE)
def test_many_rows(dt, held, new, heads, kv, dim, page, prefix, wide):
    announce("attend many", held[:5], new[:5], heads, kv, dim, page, prefix, dt, wide)
    b = Batch(held, new, heads, kv, dim, page, dt, prefix).widened(wide)
    b.check(*b.attend(return_lse=True))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("held,new,heads,kv,dim,page,prefix", [([600, 300], [500, 260], 8, 2, 64, 64, 4200), ([300], [290], 8, 2, 128, 64, 5633), ([200, 90], [190, 60], 8, 2, 256, 32, 3300),
                                                              ([400, 500], [390, 500], 10, 5, 40, 128, 4700), ([20, 0, 90] * 35, [1] * 105, 32, 4, 64, 64, 8000)])
def test_long_prefixes_of_many_rows(dt, held, new, heads, kv, dim, page, prefix):
    announce("attend prefix", held[:5], new[:5], heads, kv, dim, page, prefix, dt)
    b = Batch(held, new, heads, kv, dim, page, dt, prefix)
    b.check(*b.attend(return_lse=True))
    if max(new) == 1:
        b.check(*b.attend(starts=False, return_lse=True))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("held,heads,kv,dim,page,prefix", [([300, 90], 80, 2, 64, 32, 0), ([70], 200, 1, 128, 64, 40), ([5, 0, 600], 33, 1, 256, 64, 0), ([4200] * 97, 8, 8, 16, 32, 0),
                                                          ([9000, 8000], 2, 2, 24, 32, 0)])
def test_many_heads_and_many_pages(dt, held, heads, kv, dim, page, prefix):
    """More heads to a key head than a tile of rows, one token each; more pages in a chunk than a wave has lanes."""
    announce("attend heads", held[:5], heads, kv, dim, page, prefix, dt)
    b = Batch(held, [1] * len(held), heads, kv, dim, page, dt, prefix)
    b.check(*b.attend(starts=False, return_lse=True))
    b.check(*b.attend(return_lse=True))


@pytest.mark.parametrize("quiet", [0, 100])
@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", TYPES)
def test_logits_of_any_size(dt, wide, quiet):
    """Rows of many tokens whose logits are in the thousands and in the hundred thousands, behind `quiet` places whose are zero: the weights are those of
    their differences.  Keys and queries are whole numbers, so that products are exact; a key's weight is one or none."""
    ops = _ops()
    for size in (16, 256):
        b = Batch([300], [120], 2, 1, 32, 32, dt).widened(wide)
        kn = torch.zeros(b.k_cache.shape)
        ids = torch.randperm(300, generator=torch.Generator().manual_seed(size))
        number = b.table[0].cpu().long()
        for place in range(300):
            kn[number[place // 32], 0, place % 32, 0] = float(ids[place] % 61) * size / 8 if place >= quiet else 0.0
        from bittorch_amd.ops.attention import _tiled
        kc = _tiled(kn.to(dt), kn.to(dt))[0].contiguous().cuda()
        q = torch.zeros_like(b.q)
        q[..., 0] = 8 * size
        out = ops.cached_attention(q, kc, b.v_cache, b.table, b.lengths, b.q_starts, scale=1.0)
        assert kn.to(dt).float().equal(kn)
        for i in (0, 50, 119):
            seen = torch.stack([kn[number[p // 32], 0, p % 32, 0] for p in range(181 + i)])
            best = (seen == seen.max()).nonzero()[:, 0]
            want = b.values[0][best.cuda()].mean(0)  # equal logits share
            off = (out[i].double() - want).abs()
            # (equal weights of exact logits; rounded once, their sum and their values as always)
            assert bool((off <= (_half(dt) * 2 + 64 * U) * b.values[0][best.cuda()].abs().mean(0) + 1e-30).all()), (size, i)


@pytest.mark.parametrize("dt", TYPES)
def test_long_contexts_and_large_logits(dt):
    announce("attend long", dt)
    b = Batch([20011, 70000], [1, 1], 8, 2, 128, 64, dt, std=2.0)
    b.check(*b.attend(starts=False, return_lse=True))
    b = Batch([9000], [40], 8, 2, 64, 64, dt, 5000, std=3.0)
    for wide in (False, True):
        b.check(*b.widened(wide).attend(return_lse=True))


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new,wide", [(1, False), (9, False), (200, False), (40, True), (200, True)])
def test_what_a_row_does_not_see_does_not_matter(dt, new, wide):
    """Later tokens of the same chunk whose keys and values are infinite or not a number, in the tile where the mask runs."""
    ops = _ops()
    b = Batch([new + 45], [new], 4, 2, 64, 32, dt).widened(wide)
    clean = b.attend(return_lse=True)
    place = new + 44  # the last token's own
    number, at = int(b.table[0, place // 32]), place % 32
    kn, vn = (t.clone() for t in natural(b.k_cache, b.v_cache))
    for bad in (math.nan, math.inf, -math.inf):
        kn[number, :, at, :64], vn[number, :, at, :64] = bad, bad
        from bittorch_amd.ops.attention import _tiled
        kc, vc = (t.contiguous() for t in _tiled(kn, vn))
        out, lse = ops.cached_attention(b.q, kc, vc, b.table, b.lengths, b.q_starts, return_lse=True)
        assert torch.equal(out[:-1], clean[0][:-1]) and torch.equal(lse[:-1], clean[1][:-1]), bad
        assert not bool(out[-1].isfinite().any())
    # a key of the type's lowest value that is seen: its weight is zero or one, never not a number, as long as its product with q (its one
    # feature that is not zero) is below 2^128, what 32 bits hold
    low = torch.finfo(dt).min
    kn, vn = (t.clone() for t in natural(b.k_cache, b.v_cache))
    kn[int(b.table[0, 0]), :, 0, :64] = 0
    kn[int(b.table[0, 0]), :, 0, 0] = low if dt != torch.float32 else low / 2 ** 40
    kc, vc = (t.contiguous() for t in _tiled(kn, vn))
    out = ops.cached_attention(b.q, kc, vc, b.table, b.lengths, b.q_starts)
    fits = b.q[..., 0].double() * kc.nan_to_num(0).double().min() < 2.0 ** 128 * (1 - 2 * U)
    assert bool(out[fits].isfinite().all()) and bool(fits.any())


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new,wide", [(1, False), (200, False), (200, True)])
def test_places_whose_logits_are_minus_infinity(dt, new, wide):
    """Whole tiles of keys of -inf at the start, seen by all rows: their weights are zero."""
    from bittorch_amd.ops.attention import _tiled
    b = Batch([400], [new], 4, 2, 64, 32, dt).widened(wide)
    kn, vn = (t.clone() for t in natural(b.k_cache, b.v_cache))
    for place in range(130):
        kn[int(b.table[0, place // 32]), :, place % 32, 0] = -math.inf
    kc, vc = (t.contiguous() for t in _tiled(kn, vn))
    q = b.q.clone()
    q[..., 0] = q[..., 0].abs() + 0.5
    out, lse = _ops().cached_attention(q, kc, vc, b.table, b.lengths, b.q_starts, return_lse=True)
    k, v = (t[0][130:].repeat_interleave(2, 1) for t in (b.keys, b.values))
    x = torch.matmul(q.double().transpose(0, 1), k.permute(1, 2, 0)) / 8
    x = x.masked_fill(torch.arange(130, 400, device="cuda")[None] > torch.arange(400 - new, 400, device="cuda")[:, None], -math.inf)
    p = x.softmax(-1)
    want, spread = (torch.matmul(p, t.transpose(0, 1)).transpose(0, 1) for t in (v, v.abs()))
    # (as Batch.check: weights and results rounded to the type once each, 256 u for the 32-bit sums and exponentials of logits below 16)
    assert bool(((out.double() - want).abs() <= (_half(dt) * 2 + 256 * 16 * U) * spread + _half(dt) * want.abs()).all())
    assert bool(((lse.double() - x.logsumexp(-1).T).abs() <= 256 * 16 * U).all())


def test_lengths_pages_and_rows_that_are_not_there():
    ops = _ops()
    b = Batch([70, 10, 33], [1, 1, 1], 4, 2, 64, 32, torch.bfloat16, width=4)
    want, want_lse = b.attend(starts=False, return_lse=True)
    # a page outside the cache: that sequence alone
    for wrong in (-1, b.k_cache.shape[0], 2 ** 31 - 1, -2 ** 31):
        table = b.table.clone()
        table[0, 1] = wrong
        out, lse = ops.cached_attention(b.q, b.k_cache, b.v_cache, table, b.lengths, return_lse=True)
        assert out[0].isnan().all() and lse[0].isnan().all() and torch.equal(out[1:], want[1:]) and torch.equal(lse[1:], want_lse[1:])
    # a length beyond the table, or beyond max_length; below zero
    lengths = b.lengths.clone()
    lengths[1] = 4 * 32 + 1
    out = ops.cached_attention(b.q, b.k_cache, b.v_cache, b.table, lengths)
    assert out[1].isnan().all() and torch.equal(out[0], want[0]) and torch.equal(out[2], want[2])
    out = b.attend(starts=False, max_length=33)
    assert out[0].isnan().all()
    b.check(*b.attend(starts=False, return_lse=True, max_length=70))
    lengths[1] = -5
    out, lse = ops.cached_attention(b.q, b.k_cache, b.v_cache, b.table, lengths, return_lse=True)
    assert not out[1].any() and bool((lse[1] == -math.inf).all()) and torch.equal(out[0], want[0])
    # a prefix page outside the cache: every row
    out = ops.cached_attention(b.q, b.k_cache, b.v_cache, b.table, b.lengths, prefix_table=torch.tensor([99], dtype=torch.int32, device="cuda"), prefix_length=5)
    assert out.isnan().all()
    # rows behind the last sequence, with parts to join and without
    for width in (1, 4):
        more = torch.cat((b.q, torch.full_like(b.q, math.nan)))
        lengths = b.lengths.clamp(max=32 * width)
        out, lse = ops.cached_attention(more, b.k_cache, b.v_cache, b.table[:, :width], lengths, b.q_starts, return_lse=True)
        assert not out[3:].any() and bool((lse[3:] == -math.inf).all())
        ref = ops.cached_attention(b.q, b.k_cache, b.v_cache, b.table[:, :width], lengths)
        assert bool(((out[:3] - ref).abs() <= 4 * _half(torch.bfloat16) * 4).all())
    # pages outside the cache and lengths beyond the table among many rows: that sequence alone
    for wide in (False, True):
        many = Batch([200, 90, 70], [100, 70, 3], 4, 2, 64, 32, torch.bfloat16).widened(wide)
        want, want_lse = many.attend(return_lse=True)
        good, good_lengths = many.table, many.lengths
        for wrong in (-1, many.k_cache.shape[0], 2 ** 31 - 1, -2 ** 31):
            many.table = good.clone()
            many.table[0, 1] = wrong
            out, lse = many.attend(return_lse=True)
            assert out[:100].isnan().all() and lse[:100].isnan().all() and torch.equal(out[100:], want[100:]) and torch.equal(lse[100:], want_lse[100:])
        many.table, many.lengths = good, torch.tensor([200, many.width * 32 + 1, 70], dtype=torch.int32, device="cuda")
        out = many.attend()
        assert out[100:170].isnan().all() and torch.equal(out[:100], want[:100]) and torch.equal(out[170:], want[170:])
        many.lengths = good_lengths
        many.q_starts = torch.tensor([0, 100, 100, 173], dtype=torch.int32, device="cuda")
        out, lse = many.attend(return_lse=True)  # the third's 73 tokens on 70 places: three that see nothing
        assert torch.equal(out[:100], want[:100]) and not out[100:103].any() and bool((lse[100:103] == -math.inf).all()) and bool(out[103:].isfinite().all())
        for starts in ([0, 900, 100, 173], [-4, 100, 50, 173], [173, 90, 1, 0], [0, 2 ** 31 - 1, -2 ** 31, 173], [0, 0, 0, 0]):
            many.q_starts = torch.tensor(starts, dtype=torch.int32, device="cuda")
            many.attend()
    # starts that make no sense stay inside the tensors
    for starts in ([0, 900, 2, 3], [-4, 1, 2, 3], [3, 2, 1, 0], [0, 2 ** 31 - 1, -2 ** 31, 3]):
        ops.cached_attention(b.q, b.k_cache, b.v_cache, b.table, b.lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"))
        kc, vc = b.k_cache.clone(), b.v_cache.clone()
        ops.cache_append(b.q[:, :2].contiguous(), b.q[:, :2].contiguous(), kc, vc, b.table, b.lengths, torch.tensor(starts, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("prefix", [0, 70])
def test_rows_behind_the_last_sequence_among_many(prefix, wide):
    """With rows of both kernels, finished and joined from parts."""
    for held, new in (([700, 2500, 40, 5], [129, 65, 33, 1]), ([300, 200], [130, 3]), ([90], [90])):
        b = Batch(held, new, 4, 2, 64, 32, torch.float16, prefix).widened(wide)
        more = torch.cat((b.q, torch.full((77, 4, 64), math.nan, device="cuda").half()))
        out, lse = b.attend(more, return_lse=True)
        assert not out[b.tokens:].any() and bool((lse[b.tokens:] == -math.inf).all())
        b.check(out, lse)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_caches_of_more_than_2_to_the_31_elements(dt):
    """Pages at both ends of the cache, written and read by both kernels."""
    ops, page, dim = _ops(), 64, 128
    pages = 2 ** 31 // (page * dim) + 9
    announce("large cache", pages, dt)
    kc, vc = (torch.empty(pages, 1, page, dim, dtype=dt, device="cuda") for _ in range(2))
    order = torch.tensor([pages - 1, 0, pages - 5, 3, pages - 2, pages - 7], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(5)
    q, k, v = (torch.randn(300, h, dim, generator=g).to(dt).cuda() for h in (2, 1, 1))
    starts = torch.tensor([0, 300], dtype=torch.int32, device="cuda")
    lengths = starts[1:]
    ops.cache_append(k, v, kc, vc, order[None], lengths, starts)
    small = [torch.zeros(6, 1, page, dim, dtype=dt, device="cuda") for _ in range(2)]
    ops.cache_append(k, v, *small, torch.arange(6, dtype=torch.int32, device="cuda")[None], lengths, starts)
    for big, own in zip((kc, vc), small):
        got = big[order.long()]
        assert torch.equal(got[:4], own[:4])  # (the fifth page is whole up to place 300)
    own = torch.arange(6, dtype=torch.int32, device="cuda")[None]
    wide = torch.cat((own, torch.full((1, 500), -7, dtype=torch.int32, device="cuda")), 1)  # (so many places that 300 rows are taken as many)
    for args, tables in (((q, starts), own), ((q, starts), wide), ((q[-1:], None), own)):
        want = ops.cached_attention(args[0], *small, tables, lengths, args[1])
        there = torch.cat((order[None], tables[:, 6:]), 1)
        assert torch.equal(ops.cached_attention(args[0], kc, vc, there, lengths, args[1]), want)


def test_views_streams_and_order():
    """q as a part of one projection's output, at an odd start and with features behind heads; another stream; the same bits on every call."""
    ops = _ops()
    b = Batch([300, 41], [5, 2], 4, 2, 64, 32, torch.float16, 90)
    want = b.attend()
    qkv = torch.randn(7, 8 * 64, device="cuda").half()
    qkv[:, :256] = b.q.flatten(1)
    assert torch.equal(b.attend(qkv[:, :256].unflatten(-1, (4, 64))), want)
    odd = torch.empty(7 * 256 + 1, dtype=torch.float16, device="cuda")[1:].view(7, 4, 64).copy_(b.q)
    assert torch.equal(b.attend(odd), want)
    assert torch.equal(b.attend(b.q.transpose(0, 1).contiguous().transpose(0, 1)), want)
    assert torch.equal(b.attend(torch.empty(7, 4, 128, dtype=torch.float16, device="cuda")[..., ::2].copy_(b.q)), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [b.attend() for _ in range(3)]
    both = b.attend()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(g, want) for g in (*got, both))


# tokens of each sequence, lengths with them, heads, kv, dim, rot, interleaved, page, first position
APPENDS = [([1], [1], 4, 4, 128, 128, False, 64, 0), ([1, 1, 1], [33, 64, 1], 8, 2, 128, 128, False, 32, 5), ([7, 0, 40], [7, 0, 45], 6, 3, 80, 32, True, 32, 1000),
           ([130], [130], 2, 2, 64, 64, False, 64, 0), ([3, 9, 1, 66], [100, 30, 1, 70], 5, 1, 71, 70, True, 32, 0), ([16, 8], [16, 24], 2, 1, 20, 8, False, 32, 3),
           ([200], [333], 3, 3, 256, 256, True, 128, 0), ([5, 2], [5, 2], 1, 1, 1, 0, False, 32, 0), ([600, 300], [700, 300], 4, 2, 96, 48, False, 64, 12)]


@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("new,held,heads,kv,dim,rot,interleaved,page,first", APPENDS)
def test_append(dt, new, held, heads, kv, dim, rot, interleaved, page, first):
    announce("append", new, held, heads, kv, dim, rot, interleaved, page, dt)
    ops = _ops()
    b = Batch(held, new, heads, kv, dim, page, dt, empty=True)
    g = torch.Generator().manual_seed(7)
    k, v = (torch.randn(b.tokens, kv, dim, generator=g).to(dt).cuda() for _ in range(2))
    f = ops.rotary_frequencies(rot, device="cuda")[0] if rot else None
    q = ops.cache_append(k, v, b.k_cache, b.v_cache, b.table, b.lengths, b.q_starts, b.q if rot else None, f, interleaved, 1.0, first)
    kn, vn = natural(b.k_cache, b.v_cache)
    written = torch.zeros(kn.shape[0], page, dtype=torch.bool)
    for s, (n, h) in enumerate(zip(new, held)):
        rows = slice(b.starts[s], b.starts[s] + n)
        places = torch.arange(h - n, h)
        if n == 0:
            continue
        at = b.table[s].cpu()[places // page].long(), places % page
        written[at] = True
        got_k, got_v = kn[at[0].cuda(), :, at[1].cuda()], vn[at[0].cuda(), :, at[1].cuda()]
        assert torch.equal(got_v[..., :dim], v[rows])
        if rot:
            assert_turned(got_k[..., :dim].contiguous(), k[rows], places.cuda() + first, f, interleaved)
            assert_turned(q[rows], b.q[rows], places.cuda() + first, f, interleaved)
        else:
            assert torch.equal(got_k[..., :dim], k[rows]) and q is None
        assert not got_k[..., dim:].any()
    # nothing else was written
    rest = ~written.cuda()
    assert bool(kn.transpose(1, 2)[rest].isnan().all()) and bool(vn.transpose(1, 2)[rest].isnan().all())
    # one token each without starts: the same bits
    if all(n == 1 for n in new):
        kc, vc = torch.full_like(b.k_cache, math.nan), torch.full_like(b.v_cache, math.nan)
        again = ops.cache_append(k, v, kc, vc, b.table, b.lengths, None, b.q if rot else None, f, interleaved, 1.0, first)
        assert torch.equal(kc.nan_to_num(7), b.k_cache.nan_to_num(7)) and torch.equal(vc.nan_to_num(7), b.v_cache.nan_to_num(7)) and torch.equal(again, q)


def test_append_views_bad_pages_and_rows_behind():
    ops = _ops()
    b = Batch([40, 10], [12, 3], 4, 2, 64, 32, torch.bfloat16, empty=True)
    f = ops.rotary_frequencies(64, device="cuda")[0]
    qkv = torch.randn(17, 8 * 64, device="cuda").bfloat16()
    q, k, v = (t.unflatten(-1, (-1, 64)) for t in qkv.split([256, 128, 128], -1))
    args = b.table, b.lengths, b.q_starts
    kc, vc = b.k_cache.clone(), b.v_cache.clone()
    turned = ops.cache_append(k, v, kc, vc, *args, q, f)
    assert not turned[15:].any()  # rows behind the last sequence
    version = b.k_cache._version
    same = ops.cache_append(k.contiguous(), v.contiguous(), b.k_cache, b.v_cache, *args, q.contiguous(), f)
    assert b.k_cache._version > version and torch.equal(same, turned)
    assert torch.equal(kc.nan_to_num(7), b.k_cache.nan_to_num(7)) and torch.equal(vc.nan_to_num(7), b.v_cache.nan_to_num(7))
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t) for t in (k, v, q)]
    kc, vc = torch.full_like(kc, math.nan), torch.full_like(vc, math.nan)
    assert torch.equal(ops.cache_append(odd[0], odd[1], kc, vc, *args, odd[2], f), turned)
    assert torch.equal(kc.nan_to_num(7), b.k_cache.nan_to_num(7)) and torch.equal(vc.nan_to_num(7), b.v_cache.nan_to_num(7))
    # pages outside the cache, places behind the table: left out, the rest as before
    table = b.table.clone()
    table[0, 1] = b.k_cache.shape[0]
    kc, vc = torch.full_like(kc, math.nan), torch.full_like(vc, math.nan)
    ops.cache_append(k, v, kc, vc, table, b.lengths, b.q_starts, q, f)
    page = int(b.table[0, 1])
    assert kc[page].isnan().all() and vc[page].isnan().all() and not kc[int(b.table[1, 0])].isnan().all()
    lengths = b.lengths + 100
    kc, vc = torch.full_like(kc, math.nan), torch.full_like(vc, math.nan)
    ops.cache_append(k, v, kc, vc, b.table, lengths, b.q_starts, q, f)
    assert kc.isnan().all() and vc.isnan().all()
    for bad in (dict(k=k.requires_grad_()), dict(v=v.half())):
        with pytest.raises(RuntimeError):
            ops.cache_append(bad.get("k", k), bad.get("v", v), kc, vc, *args)


@pytest.mark.parametrize("dt", TYPES)
def test_a_conversation(dt):
    """As they are used: a shared prefix, prompts, then a token at a time, against rotary and causal attention over the whole of it."""
    ops = _ops()
    heads, kv, dim, page, prefix = 8, 2, 64, 32, 50
    g = torch.Generator().manual_seed(1)
    prompts, steps = [37, 5, 64], 4
    f = ops.rotary_frequencies(dim, device="cuda")[0]
    kc, vc = ops.paged_cache(32, kv, dim, page, dt)
    order = torch.randperm(32, generator=g).int().cuda()
    prefix_table, table = order[:2], order[2:2 + 9].view(3, 3)
    mk = lambda n, h: torch.randn(n, h, dim, generator=g).to(dt).cuda()  # noqa: E731
    pk, pv = mk(prefix, kv), mk(prefix, kv)
    whole = torch.tensor([prefix], dtype=torch.int32, device="cuda")
    assert ops.cache_append(pk, pv, kc, vc, prefix_table[None], whole, torch.tensor([0, prefix], dtype=torch.int32, device="cuda"), inv_freq=f) is None
    rows = [[mk(n + steps, h) for h in (heads, kv, kv)] for n in prompts]
    got = [[] for _ in prompts]
    lengths = torch.tensor(prompts, dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 37, 42, 106], dtype=torch.int32, device="cuda")
    q, k, v = (torch.cat([r[i][:n] for r, n in zip(rows, prompts)]) for i in range(3))
    for step in range(steps + 1):
        turned = ops.cache_append(k, v, kc, vc, table, lengths, starts if step == 0 else None, q, f, first_position=prefix)
        out = ops.cached_attention(turned, kc, vc, table, lengths, starts if step == 0 else None, prefix_table=prefix_table, prefix_length=prefix)
        for s, n in enumerate(prompts):
            got[s].append(out[int(starts[s]):int(starts[s + 1])] if step == 0 else out[s:s + 1])
        if step < steps:
            q, k, v = (torch.stack([r[i][n + step] for r, n in zip(rows, prompts)]) for i in range(3))
            lengths += 1
    for s, n in enumerate(prompts):
        m = n + steps
        turn = lambda x, at: ops.rotary(x, None, torch.arange(at, at + x.shape[0], device="cuda"), f).double()  # noqa: E731
        qs, ks = turn(rows[s][0], prefix), torch.cat((turn(pk, 0), turn(rows[s][1], prefix))).repeat_interleave(4, 1)
        vs = torch.cat((pv, rows[s][2])).double().repeat_interleave(4, 1)
        x = torch.matmul(qs.transpose(0, 1), ks.permute(1, 2, 0)) / 8
        x = x.masked_fill(torch.ones(m, prefix + m, dtype=torch.bool, device="cuda").triu(prefix + 1), -math.inf)
        p = x.softmax(-1)
        want, spread = (torch.matmul(p, t.transpose(0, 1)).transpose(0, 1) for t in (vs, vs.abs()))
        off = (torch.cat(got[s]).double() - want).abs()
        # (as Batch.check: weights and results rounded to the type once each, 256 u for the 32-bit sums and exponentials of logits below 16)
        assert bool((off <= (_half(dt) * 2 + 256 * 16 * U) * spread + _half(dt) * want.abs()).all())


def test_captured_calls_follow_lengths_and_tables():
    """A step of append and attention in a graph, replayed as lengths grow and pages are handed out, two graphs at once, eager calls between."""
    ops = _ops()
    dt, heads, kv, dim, page, n = torch.bfloat16, 4, 2, 64, 32, 3
    f = ops.rotary_frequencies(dim, device="cuda")[0]
    kc, vc = ops.paged_cache(40, kv, dim, page, dt)
    q, k, v = (torch.randn(n, h, dim, device="cuda").to(dt) for h in (heads, kv, kv))
    table = torch.full((n, 9), -1, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.tensor([5, 9, 1])
    lengths = torch.tensor([1, 20, 31], dtype=torch.int32, device="cuda")

    def step():
        return ops.cached_attention(ops.cache_append(k, v, kc, vc, table, lengths, None, q, f), kc, vc, table, lengths)

    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        step()
    torch.cuda.current_stream().wait_stream(warm)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(step())
    for i in range(6):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, device="cuda"))
        if i == 2:
            table[:, 1] = torch.tensor([30, 31, 32])
        if i == 4:
            table[:, 1:8] = torch.arange(10, 31, device="cuda").view(3, 7)
            lengths.copy_(torch.tensor([40, 200, 64]))
        kc2, vc2 = kc.clone(), vc.clone()
        want = ops.cached_attention(ops.cache_append(k, v, kc2, vc2, table, lengths, None, q, f), kc2, vc2, table, lengths)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[i % 2].nan_to_num(9), want.nan_to_num(9)), i
        assert torch.equal(kc, kc2) and torch.equal(vc, vc2)
        if i != 1:
            lengths += 1


@pytest.mark.parametrize("wide", [False, True])
def test_captured_prompts_follow_tokens_and_lengths(wide):
    """Rows of both kernels, a prefix and its parts in two graphs, replayed in turn and on two streams at once, eager calls between."""
    b = Batch([300, 90, 200, 33], [150, 70, 3, 1], 4, 2, 64, 32, torch.bfloat16, 70).widened(wide)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        b.attend(return_lse=True)
    torch.cuda.current_stream().wait_stream(warm)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(b.attend(return_lse=True))
    for i in range(5):
        b.q.copy_(torch.randn(b.q.shape, device="cuda"))
        if i == 2:
            b.lengths -= 30  # (the third sequence's tokens move up, the last has fewer places than a tile)
        want = b.attend(return_lse=True)
        if i < 4:
            graphs[i % 2].replay()
            got = [outs[i % 2]]
        else:
            warm.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(warm):
                graphs[0].replay()
            graphs[1].replay()
            torch.cuda.current_stream().wait_stream(warm)
            got = outs
        torch.cuda.synchronize()
        for g in got:
            assert torch.equal(g[0], want[0]) and torch.equal(g[1], want[1]), i


def test_many_sequences_on_a_wide_table():
    """So many that their parts would take more than a GiB in chunks of the usual length."""
    held = [20, 1, 32, 7] * 600
    held[5], held[2399] = 20000, 9000
    b = Batch(held, [1] * 2400, 2, 2, 128, 32, torch.bfloat16, width=4096)
    b.check(*b.attend(return_lse=True))


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("page", [4096, 65536])
def test_pages_longer_than_chunks(dt, page, wide):
    announce("attend long pages", dt, page, wide)
    b = Batch([5000, 300], [150, 40], 4, 2, 64, page, dt, 4500).widened(wide)
    b.check(*b.attend(return_lse=True))
    one = Batch([70000, 300], [1, 1], 8, 2, 64, page, dt, 100)
    one.check(*one.attend(starts=False, return_lse=True))


def test_calls_made_in_python_give_the_same(monkeypatch):
    """The native host side and the Python functions it stands in for."""
    from bittorch_amd import _C, _lib
    ops = _ops()
    f = ops.rotary_frequencies(64, device="cuda")[0]

    def everything():
        b = Batch([300, 41, 7], [5, 2, 0], 4, 2, 64, 32, torch.bfloat16, 90)
        one = Batch([300, 41], [1, 1], 4, 2, 64, 32, torch.float32)
        qkv = torch.arange(7 * 8 * 64, device="cuda").view(7, 512).sin().bfloat16()
        q, k, v = (t.unflatten(-1, (-1, 64)) for t in qkv.split([256, 128, 128], -1))
        leaf = qkv.clone().requires_grad_()
        lq, lk = leaf[:, :256].unflatten(-1, (-1, 64)), leaf[:, 256:384].unflatten(-1, (-1, 64))
        turned = ops.rotary(lq, lk, torch.arange(7, device="cuda"), f, True, 1.5)
        grads = torch.autograd.grad(turned, leaf, [t.detach().cos() for t in turned])
        alone = ops.rotary(lq.detach()[None], None, torch.arange(7, device="cuda")[None].int(), f.float())
        attended = [*b.attend(return_lse=True), b.attend(scale=0.5, max_length=300), *one.attend(starts=False, return_lse=True)]
        out = ops.cache_append(k, v, b.k_cache, b.v_cache, b.table, b.lengths, b.q_starts, q, f, False, 1.0, 90)
        return [*turned, *grads, alone, *attended, out, b.k_cache, b.v_cache]

    native = everything()
    monkeypatch.setattr(_C, "_N", _lib._PythonCalls())
    for i, (x, y) in enumerate(zip(native, everything())):
        assert torch.equal(x.nan_to_num(9), y.nan_to_num(9)), i
