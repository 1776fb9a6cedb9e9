"""``ops.cached_attention`` on the CPU where keys and values are infinite: the rules that the GPU's kernels keep too."""
import math

import pytest
import torch

from bittorch_amd import ops


def filled(kind, dt=torch.float32, device="cpu"):
    """Three sequences of 3, 40 and 33 places, one token each; the second's keys, or one of its values, are what ``kind`` says.  q of one feature that is
    one: a key's first feature is its logit (times the scale)."""
    g = torch.Generator().manual_seed(2)
    kc, vc = ops.paged_cache(6, 1, 16, 32, dt, "cpu")
    table = torch.tensor([[4, -1], [0, 2], [5, 1]], dtype=torch.int32)
    lengths, starts = torch.tensor([3, 40, 33], dtype=torch.int32), torch.tensor([0, 3, 43, 76], dtype=torch.int32)
    k, v = (torch.randn(76, 1, 16, generator=g).to(dt) for _ in range(2))
    if kind == "all":
        k[3:43, 0, 0] = -math.inf
    elif kind == "plus":
        k[20, 0, 0] = math.inf
    elif kind == "nan":
        k[20, 0, 0] = math.nan
    elif kind == "value":
        v[20, 0, 5] = math.inf
    elif kind == "values":
        v[20, 0, 5], v[21, 0, 5] = math.inf, -math.inf
    ops.cache_append(k, v, kc, vc, table, lengths, starts)
    q = torch.zeros(3, 2, 16, dtype=dt)
    q[:, :, 0] = 1
    return [t.to(device) for t in (q, kc, vc, table, lengths)]


def check(kind, out, lse):
    assert bool(out[0].isfinite().all()) and bool(out[2].isfinite().all()) and bool(lse[0].isfinite().all()) and bool(lse[2].isfinite().all())
    out, lse = out[1], lse[1]
    if kind == "all":
        assert not out.any() and bool((lse == -math.inf).all())
    elif kind in ("plus", "nan"):
        assert bool(out.isnan().all()) and bool(lse.isnan().all())
    else:
        there = torch.arange(16, device=out.device) == 5
        assert not bool(out[:, there].isfinite().any()) and bool(out[:, ~there].isfinite().all()) and bool(lse.isfinite().all())


KINDS = ["all", "plus", "nan", "value", "values"]


@pytest.mark.parametrize("kind", KINDS)
def test_infinite_keys_and_values(kind):
    q, kc, vc, table, lengths = filled(kind)
    check(kind, *ops.cached_attention(q, kc, vc, table, lengths, return_lse=True))
    # behind a prefix of finite places a sequence of keys of minus infinity has the prefix alone
    if kind == "all":
        prefix = torch.tensor([4], dtype=torch.int32)
        out, lse = ops.cached_attention(q, kc, vc, table, lengths, prefix_table=prefix, prefix_length=3, return_lse=True)
        alone, alone_lse = ops.cached_attention(q[:1], kc, vc, table[:1], lengths[:1], return_lse=True)
        assert torch.allclose(out[1:2], alone) and torch.allclose(lse[1:2], alone_lse)
