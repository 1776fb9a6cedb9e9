"""``ops.rotary``, ``ops.cache_append`` and ``ops.cached_attention`` on the CPU: their definitions, the order of the cache, and their refusals."""
import ctypes
import math

import pytest
import torch

from bittorch_amd import _C, _lib, ops
from bittorch_amd.ops.attention import _natural, _tiled


def complex_turn(x, positions, inv_freq, interleaved, amplitude=1.0):
    """The definition by complex numbers, in 64 bits."""
    n, x = 2 * inv_freq.shape[0], x.double()
    angle = positions.double()[..., None, None] * inv_freq.double()
    unit = torch.polar(torch.full_like(angle, amplitude), angle)
    part = x[..., :n]
    z = torch.complex(part[..., 0::2], part[..., 1::2]) if interleaved else torch.complex(part[..., :n // 2], part[..., n // 2:])
    z = z * unit
    part = torch.stack((z.real, z.imag), -1).flatten(-2) if interleaved else torch.cat((z.real, z.imag), -1)
    return torch.cat((part, x[..., n:]), -1)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,rot", [(8, 8), (20, 10), (7, 6), (16, 2)])
def test_rotary_is_a_turn_of_pairs(interleaved, dim, rot):
    g = torch.Generator().manual_seed(dim)
    q, k = torch.randn(3, 5, 4, dim, generator=g, dtype=torch.float64), torch.randn(3, 5, 2, dim, generator=g, dtype=torch.float64)
    inv_freq, one = ops.rotary_frequencies(rot)
    assert one == 1.0
    pos = torch.randint(0, 100000, (5,), generator=g)
    got_q, got_k = ops.rotary(q, k, pos, inv_freq, interleaved, 1.25)
    # (64 bits: 100000 radians are off by 2^-36)
    assert torch.allclose(got_q, complex_turn(q, pos.expand(3, 5), inv_freq, interleaved, 1.25), rtol=0, atol=1e-9)
    assert torch.allclose(got_k, complex_turn(k, pos.expand(3, 5), inv_freq, interleaved, 1.25), rtol=0, atol=1e-9)
    assert torch.equal(ops.rotary(q, None, pos, inv_freq, interleaved, 1.25), got_q)
    assert torch.equal(got_q[..., rot:], q[..., rot:])
    assert torch.autograd.gradcheck(lambda a, b: ops.rotary(a, b, pos % 50, inv_freq, interleaved, 0.5), (q.requires_grad_(), k.requires_grad_()))


def test_frequencies():
    f, a = ops.rotary_frequencies(8)
    assert f.dtype == torch.float64 and a == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-12)
    assert torch.allclose(ops.rotary_frequencies(8, scaling=dict(kind="linear", factor=4))[0], f / 4, rtol=1e-12)
    base = ops.rotary_frequencies(8, scaling=dict(kind="base", factor=4))[0]
    assert base[0] == 1 and math.isclose(base[-1], f[-1] / 4, rel_tol=1e-12) and bool((base <= f).all())
    ramp, a = ops.rotary_frequencies(64, scaling=dict(kind="ramp", factor=4, original=8192))
    plain = ops.rotary_frequencies(64)[0]
    turns = 8192 * plain / (2 * math.pi)
    assert torch.equal(ramp[turns > 32], plain[turns > 32]) and torch.allclose(ramp[turns < 1], plain[turns < 1] / 4, rtol=1e-12)
    between = (turns > 1) & (turns < 32)
    assert bool(((ramp <= plain) & (ramp >= plain / 4))[between].all()) and bool(between.any()) and math.isclose(a, 0.1 * math.log(4) + 1)
    for bad in (dict(kind="linear"), dict(kind="linear", factor=0.5), dict(kind="other", factor=2), dict(kind="ramp", factor=2),
                dict(kind="ramp", factor=2, original=10, slow=3, fast=3), dict(kind="linear", factor=2, original=1)):
        with pytest.raises(RuntimeError):
            ops.rotary_frequencies(8, scaling=bad)
    for args in ((7,), (0,), (8, -1.0), (2, 10000.0, dict(kind="base", factor=2))):
        with pytest.raises(RuntimeError):
            ops.rotary_frequencies(*args)


@pytest.mark.parametrize("dtype,dim,page", [(torch.bfloat16, 80, 32), (torch.float16, 33, 64), (torch.float32, 20, 32), (torch.float32, 16, 128)])
def test_order_of_the_cache(dtype, dim, page):
    """The order is that of the header, whatever the type; pages are independent of each other."""
    kc, vc = ops.paged_cache(3, 2, dim, page, dtype, "cpu")
    e, padded = 16 // kc.element_size(), kc.shape[3]
    assert kc.shape == vc.shape == (3, 2, page, padded) and padded * kc.element_size() % 64 == 0 and dim <= padded < dim + 64 // kc.element_size()
    for place in (0, 1, 5, 8, 17, page - 1):
        for f in (0, 3, 9, dim - 1):
            t, r = place // (4 * e), place % (4 * e)
            tile = t * 4 * e * padded
            key = ((((f // (4 * e)) * (e // 4) + r % e // 4) * 4 + f % (4 * e) // e) * 16 + r // e * 4 + r % 4) * e + f % e
            value = ((f // 16 * 4 + r // e) * 16 + f % 16) * e + r % e
            k, v = torch.zeros_like(kc), torch.zeros_like(vc)
            k.view(-1)[(2 * 2 + 1) * page * padded + tile + key] = 1
            v.view(-1)[(2 * 2 + 1) * page * padded + tile + value] = 1
            kn, vn = _natural(k, v)
            assert kn[2, 1, place, f] == 1 and kn.sum() == 1 and vn[2, 1, place, f] == 1 and vn.sum() == 1
    rows = torch.randn(3, 2, page, padded).to(dtype), torch.randn(3, 2, page, padded).to(dtype)
    assert all(torch.equal(a, b) for a, b in zip(_natural(*_tiled(*rows)), rows))


def test_append_read_and_attend():
    """Prompt, then a token at a time: the pages hold the turned keys, and the results are those of the whole sequence's causal attention."""
    g = torch.Generator().manual_seed(3)
    heads, kv, dim, n = 6, 2, 12, 41
    inv_freq, _ = ops.rotary_frequencies(8)
    q, k, v = (torch.randn(n, h, dim, generator=g) for h in (heads, kv, kv))
    kc, vc = ops.paged_cache(4, kv, dim, 32, torch.float32, "cpu")
    table = torch.tensor([[3, 1]], dtype=torch.int32)
    out = []
    for a, b in [(0, 37)] + [(i, i + 1) for i in range(37, n)]:
        lengths = torch.tensor([b], dtype=torch.int32)
        starts = torch.tensor([0, b - a], dtype=torch.int32)
        turned = ops.cache_append(k[a:b], v[a:b], kc, vc, table, lengths, starts, q[a:b], inv_freq)
        out.append(ops.cached_attention(turned, kc, vc, table, lengths, starts))
    kt, vt = ops.cache_read(kc, vc, table[0], n, dim)
    assert torch.allclose(kt, ops.rotary(k, None, torch.arange(n), inv_freq), atol=1e-6) and torch.equal(vt, v)
    qt = ops.rotary(q, None, torch.arange(n), inv_freq)
    want = torch.nn.functional.scaled_dot_product_attention(*(t.transpose(0, 1).double() for t in (qt, kt.repeat_interleave(3, 1), vt.repeat_interleave(3, 1))),
                                                            is_causal=True).transpose(0, 1)
    assert torch.allclose(torch.cat(out).double(), want, atol=1e-5)
    assert not kc[0].any() and not kc[2].any()


def test_what_is_not_written_and_what_is_not_a_number():
    """No place, no page, a page outside the cache, a length beyond the table, rows behind the last sequence."""
    dim, kc, vc = 16, *ops.paged_cache(2, 1, 16, 32, torch.float32, "cpu")
    before = kc.clone()
    k = torch.ones(4, 1, dim)
    table = torch.tensor([[7], [-1], [0], [1]], dtype=torch.int32)
    lengths = torch.tensor([1, 1, 0, 40], dtype=torch.int32)
    ops.cache_append(k, k, kc, vc, table, lengths)
    assert torch.equal(kc, before) and torch.equal(vc, before)
    out, lse = ops.cached_attention(k, kc, vc, table, lengths, return_lse=True)
    assert out[0].isnan().all() and out[1].isnan().all() and out[3].isnan().all()
    assert not out[2].any() and lse[2] == -math.inf
    starts = torch.tensor([0, 0, 2, 2, 2], dtype=torch.int32)
    inv_freq, _ = ops.rotary_frequencies(4)
    turned = ops.cache_append(k, k, kc, vc, table, torch.tensor([0, 2, 0, 0], dtype=torch.int32), starts, q=k, inv_freq=inv_freq)
    assert not turned[2:].any() and turned[:2].all()
    out, lse = ops.cached_attention(k, kc, vc, table, torch.tensor([0, 0, 0, 0], dtype=torch.int32), starts, return_lse=True)
    assert not out.any() and bool((lse == -math.inf).all())


def _call(**change):
    args = dict(k=torch.zeros(2, 2, 16), v=torch.zeros(2, 2, 16), q=torch.zeros(2, 4, 16), table=torch.zeros(2, 3, dtype=torch.int32),
                lengths=torch.zeros(2, dtype=torch.int32), starts=None, inv_freq=torch.ones(8), cache=ops.paged_cache(5, 2, 16, 32, torch.float32, "cpu"),
                prefix_table=None, prefix_length=0, scale=None, max_length=None)
    args.update(change)
    return args


BAD = [
    dict(k=torch.zeros(2, 16), v=torch.zeros(2, 16)), dict(v=torch.zeros(2, 1, 16)), dict(k=torch.zeros(2, 1, 16), v=torch.zeros(2, 1, 16)),
    dict(k=torch.zeros(2, 2, 17), v=torch.zeros(2, 2, 17)), dict(q=torch.zeros(3, 4, 16)), dict(q=torch.zeros(2, 4, 16).half()), dict(inv_freq=torch.ones(9)),
    dict(inv_freq=torch.ones(8).half()), dict(inv_freq=torch.ones(2, 4)), dict(inv_freq=None), dict(table=torch.zeros(2, 3)), dict(table=torch.zeros(3, 3, dtype=torch.int32)),
    dict(table=torch.zeros(2, 0, dtype=torch.int32)), dict(lengths=torch.zeros(2, dtype=torch.int64)), dict(lengths=torch.zeros(2, 1, dtype=torch.int32)),
    dict(starts=torch.zeros(2, dtype=torch.int32)), dict(starts=torch.zeros(3, dtype=torch.int64)), dict(table=torch.zeros(3, 3, dtype=torch.int32), lengths=torch.zeros(3, dtype=torch.int32)),
    dict(cache=(torch.zeros(5, 2, 32, 16), torch.zeros(5, 2, 32, 32))), dict(cache=(torch.zeros(5, 2, 16, 16),) * 2), dict(cache=(torch.zeros(5, 2, 48, 16),) * 2),
    dict(cache=(torch.zeros(5, 2, 32, 16),) * 2), dict(cache=(torch.zeros(5, 2, 32, 32)[..., ::2], torch.zeros(5, 2, 32, 16))),
    dict(cache=(torch.zeros(5, 2, 32, 16).double(), torch.zeros(5, 2, 32, 16).double())), dict(k=torch.zeros(2, 2, 16, requires_grad=True)),
]


@pytest.mark.parametrize("change", BAD, ids=lambda c: "-".join(c))
def test_append_refuses(change):
    a = _call(**change)
    before = [t.clone() for t in a["cache"]]
    with pytest.raises(RuntimeError):
        ops.cache_append(a["k"], a["v"], *a["cache"], a["table"], a["lengths"], a["starts"], a["q"], a["inv_freq"])
    assert all(torch.equal(x, y) for x, y in zip(before, a["cache"]))


@pytest.mark.parametrize("change", [dict(q=torch.zeros(2, 3, 16)), dict(q=torch.zeros(2, 16)), dict(q=torch.zeros(2, 4, 300)), dict(scale=0.0), dict(scale=-1.0),
                                    dict(scale=math.nan), dict(scale=math.inf), dict(max_length=-1), dict(max_length=97), dict(prefix_length=-1),
                                    dict(prefix_length=1), dict(prefix_length=33, prefix_table=torch.zeros(1, dtype=torch.int32)),
                                    dict(prefix_length=1, prefix_table=torch.zeros(1)), dict(prefix_length=1, prefix_table=torch.zeros(1, 1, dtype=torch.int32)),
                                    dict(q=torch.zeros(2, 4, 16, requires_grad=True)), *[c for c in BAD if {"table", "lengths", "starts"} & set(c)]],
                         ids=lambda c: "-".join(c))
def test_attention_refuses(change):
    a = _call(**change)
    with pytest.raises(RuntimeError):
        ops.cached_attention(a["q"], *a["cache"], a["table"], a["lengths"], a["starts"], a["scale"], a["prefix_table"], a["prefix_length"], max_length=a["max_length"])


def test_rotary_refuses():
    q, pos, f = torch.zeros(4, 2, 8), torch.arange(4), torch.ones(4)
    for args in ((q, torch.zeros(4, 2, 9), pos, f), (q, torch.zeros(3, 2, 8), pos, f), (q, q.half(), pos, f), (q, None, pos.float(), f), (q, None, pos, torch.ones(5)),
                 (q, None, pos, f.half()), (q, None, torch.arange(3), f), (torch.zeros(8), None, pos, f), (q.long(), None, pos, f),
                 (q, None, pos, torch.ones(4, requires_grad=True))):
        with pytest.raises(RuntimeError):
            ops.rotary(*args)


def test_no_tokens():
    kc, vc = ops.paged_cache(1, 1, 16, 32, torch.float32, "cpu")
    none, table, lengths = torch.zeros(0, 1, 16), torch.zeros(0, 1, dtype=torch.int32), torch.zeros(0, dtype=torch.int32)
    assert ops.cache_append(none, none, kc, vc, table, lengths, q=none, inv_freq=torch.ones(1)).shape == (0, 1, 16)
    assert ops.cached_attention(none, kc, vc, table, lengths).shape == (0, 1, 16)
    with pytest.raises(RuntimeError):
        ops.cached_attention(torch.zeros(1, 1, 16), kc, vc, table, lengths, torch.zeros(1, dtype=torch.int32))


def test_library_refuses_without_a_gpu():
    lib, buf = _lib.load(), ctypes.create_string_buffer(64)
    at = (ctypes.addressof(buf) + 15) // 16 * 16
    rotary = lambda dt=0, tokens=1, heads=1, dim=8, rot=8, q=at, freq=at: lib.bt_rotary(  # noqa: E731
        q, 8, 8, None, 0, 0, dt, at, 0, freq, 0, 0, 1.0, 0, tokens, heads, 0, dim, rot, at, None, None)
    for bad in (dict(dt=3), dict(tokens=0), dict(heads=0), dict(dim=0), dict(rot=7), dict(rot=10), dict(q=None), dict(freq=None), dict(dim=2048), dict(heads=20000)):
        assert rotary(**bad) == -1 and "bt_rotary" in _lib.last_error(), bad
    append = lambda page=32, pages=1, width=1, n_seq=1, dim=8, k=at, cache=at, tokens=1: lib.bt_cache_append(  # noqa: E731
        k, 8, 8, at, 8, 8, None, 0, 0, 0, None, 0, 0, 1.0, 0, tokens, 0, 1, dim, 0, cache, at, pages, page, at, width, at, None, n_seq, None, None)
    for bad in (dict(page=16), dict(page=48), dict(pages=0), dict(width=0), dict(n_seq=2), dict(dim=257), dict(k=None), dict(cache=at + 4), dict(tokens=0),
                dict(width=1 << 27)):
        assert append(**bad) == -1 and "bt_cache_append" in _lib.last_error(), bad
    attend = lambda page=32, width=1, longest=32, n_seq=1, dim=8, heads=2, kv=1, scale=1.0, cache=at, prefix=0, ws=None, size=0: lib.bt_cached_attention(  # noqa: E731
        at, 8, 8, 0, cache, at, 1, page, at, width, longest, at, None, n_seq, None, prefix, scale, 1, heads, kv, dim, at, None, ws, size, None)
    for bad in (dict(page=33), dict(width=0), dict(longest=33), dict(n_seq=2), dict(dim=300), dict(heads=3, kv=2), dict(scale=0.0), dict(scale=math.nan), dict(cache=at + 8),
                dict(prefix=4)):
        assert attend(**bad) == -1 and "bt_cached_attention" in _lib.last_error(), bad
    need = lib.bt_cached_attention_workspace_bytes(0, 1, 1, 2, 1, 8, 32, 1024, 32768, 0, 1, 0)
    assert need > 0 and attend(width=1024, longest=32768) == -2 and attend(width=1024, longest=32768, ws=256, size=need - 1) == -2
    assert lib.bt_cached_attention_workspace_bytes(0, 1, 0, 2, 1, 8, 32, 1024, 32768, 0, 1, 0) == 0
    assert [lib.bt_cache_head_dim(d, n) for d, n in ((0, 1), (0, 80), (1, 80), (2, 128), (2, 257), (3, 8), (0, 0))] == [16, 80, 96, 128, 0, 0, 0]


def test_native_calls_leave_cpu_tensors_to_python():
    a = _call()
    n = _C._N
    assert n.rotary(a["q"], a["k"], torch.arange(2), a["inv_freq"], False, 1.0) is None
    assert n.cache_append(a["k"], a["v"], *a["cache"], a["table"], a["lengths"], None, a["q"], a["inv_freq"], False, 1.0, 0) is None
    assert n.cached_attention(a["q"], *a["cache"], a["table"], a["lengths"], None, None, None, 0, False, None) is None
    for f in (n.rotary, n.cache_append, n.cached_attention):
        assert f() is None and f(*(None,) * 6) is None


def test_workspaces_of_many_sequences_on_wide_tables():
    """Parts that few rows leave take a GiB at most, however many places the table may hold."""
    lib = _lib.load()
    for sequences in (1, 100, 3000, 50000):
        for starts, tokens in ((0, sequences), (1, 2 * sequences)):
            need = lib.bt_cached_attention_workspace_bytes(_C._DT[torch.bfloat16], 1, tokens, 32, 8, 128, 64, 4096, 4096 * 64, starts, sequences, 0)
            many = tokens * 32 * (128 * 4 + 8) * 2  # (those of rows by token and head: two chunks of the least workgroups)
            assert need <= 2 ** 30 * 1.02 + max(many, 2 ** 27), (sequences, starts, need)
