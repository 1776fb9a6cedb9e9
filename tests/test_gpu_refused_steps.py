"""A step of the block stack that the operators refuse can be made again, put right."""
import pytest
import torch

from test_gpu_cached_stack import _rel, _stack

pytestmark = pytest.mark.gpu


def test_a_refused_step_can_be_made_again():
    c5 = _stack(32)
    prefix = c5.tokens[0, :25]
    c5.tokens[1:, :25] = prefix
    c5.convert()
    c5.fuse()
    want = c5.forward_fused(False)
    c5.start_cache(3, 15, prefix=25, page_size=32)
    with pytest.raises(RuntimeError):
        c5.forward_prefix(prefix.double())
    assert _rel(c5.forward_prefix(prefix), want[0, :25]) < 2e-4
    starts = torch.tensor([0, 4, 4, 5], dtype=torch.int32, device="cuda")
    tokens = torch.cat((c5.tokens[0, 25:29], c5.tokens[2, 25:26]))
    for bad in ((tokens, starts.long()), (tokens, starts.cpu()), (tokens.double(), starts), (tokens[:, None], starts)):
        with pytest.raises(RuntimeError):
            c5.forward_cached(*bad)
        assert c5.cache["lengths"].tolist() == [0, 0, 0]
    got = c5.forward_cached(tokens, starts)
    assert c5.cache["lengths"].tolist() == [4, 0, 1]
    assert _rel(got, torch.cat((want[0, 25:29], want[2, 25:26]))) < 2e-4
    got = c5.forward_cached(torch.stack((c5.tokens[0, 29], c5.tokens[1, 25], c5.tokens[2, 26])))
    assert _rel(got, torch.stack((want[0, 29], want[1, 25], want[2, 26]))) < 2e-4
