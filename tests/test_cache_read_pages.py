"""``ops.cache_read`` on pages that the cache does not have."""
import pytest
import torch

from bittorch_amd import ops


def check(device, dt):
    kc, vc = ops.paged_cache(3, 2, 20, 32, dt, device)
    k, v = (torch.randn(80, 2, 20, generator=torch.Generator().manual_seed(i)).to(dt).to(device) for i in range(2))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=device)
    ops.cache_append(k, v, kc, vc, table, torch.tensor([80], dtype=torch.int32, device=device), torch.tensor([0, 80], dtype=torch.int32, device=device))
    for wrong in (-1, -3, 3, 2 ** 31 - 1, -2 ** 31):
        row = table[0].clone()
        row[1] = wrong
        for got, want in zip(ops.cache_read(kc, vc, row, 80, 20), (k, v)):
            assert torch.equal(got[:32], want[:32]) and torch.equal(got[64:], want[64:]) and bool(got[32:64].isnan().all())
        assert all(torch.equal(got, want[:32]) for got, want in zip(ops.cache_read(kc, vc, row, 32, 20), (k, v)))


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_pages_outside_the_cache_are_not_a_number(dt):
    """Neither another sequence's page nor an index error: as the attention takes them."""
    check("cpu", dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16, torch.float16])
def test_pages_outside_the_cache_are_not_a_number_on_the_gpu(dt):
    check("cuda", dt)
