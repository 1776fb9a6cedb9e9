"""The block stack with rotary positions, and decoding with caches: the same hidden states as the whole sequences at once."""
import pytest
import torch

from conftest import announce

pytestmark = pytest.mark.gpu


def _stack(rotary_dim, dt=torch.float32, **more):
    from bittorch_amd.utils.block_stack import BlockStack
    torch.manual_seed(0)
    std = dict(q=0.02, k=0.02, v=0.02, o=0.02, gate=0.02, up=0.02, down=0.02)
    return BlockStack("cuda", layers=2, d_model=128, heads=4, ffn=208, batch=3, seq=40, vocab=64, act_dtype=dt, master_std=std, rotary_dim=rotary_dim, **more)


def _rel(a, b):
    return float((a.detach().double() - b.detach().double()).norm() / b.detach().double().norm())


@pytest.mark.parametrize("rotary_dim", [0, 32, 16])
@pytest.mark.parametrize("int8", [False, True])
def test_cached_steps_give_the_whole_sequences_states(rotary_dim, int8):
    """Prompts of unlike lengths, then a token at a time, then two for one sequence and none for another.  fp32: the projections' kernels for few and many
    rows and the two attentions round differently, by under 1e-5 each; an int8 code next to a border may fall to its other side (1/127 of a
    row's largest value, in few places)."""
    announce("cached stack", rotary_dim, int8)
    c5 = _stack(rotary_dim)
    tokens = c5.tokens
    want = None
    c5.convert()
    c5.fuse()
    want = c5.forward_fused(int8)
    c5.start_cache(3, 40, page_size=32)
    prompt = [30, 1, 17]
    at = list(prompt)
    int32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = [[] for _ in prompt]

    def run(new):
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        picked = torch.cat([tokens[s, a - n:a] for s, (a, n) in enumerate(zip(at, new))])
        out = c5.forward_cached(picked, None if new == [1, 1, 1] else int32(starts), int8)
        for s, n in enumerate(new):
            got[s].append(out[starts[s]:starts[s] + n])

    run(prompt)
    for new in ([1, 1, 1], [1, 1, 1], [2, 0, 1], [1, 1, 1], [0, 20, 2]):
        at = [a + n for a, n in zip(at, new)]
        run(new)
    for s, a in enumerate(at):
        have = torch.cat(got[s])
        assert have.shape == (a, 128) and _rel(have, want[s, :a]) < (2e-2 if int8 else 2e-4)


def test_shared_prefix():
    c5 = _stack(32)
    prefix = c5.tokens[0, :25]
    c5.tokens[1:, :25] = prefix
    c5.convert()
    c5.fuse()
    want = c5.forward_fused(False)
    c5.start_cache(3, 15, prefix=25, page_size=32)
    first = c5.forward_prefix(prefix)
    assert _rel(first, want[0, :25]) < 2e-4
    with pytest.raises(RuntimeError, match="prefix"):
        c5.forward_prefix(prefix)
    for i in range(25, 40):
        assert _rel(c5.forward_cached(c5.tokens[:, i].contiguous()), want[:, i]) < 2e-4


def test_a_captured_step_follows_the_caches():
    """One step in a graph, replayed for token after token."""
    c5 = _stack(32, torch.bfloat16)
    c5.convert()
    c5.fuse()
    c5.start_cache(3, 64)
    static = c5.tokens[:, 0].contiguous()
    eager = []
    for i in range(12):
        eager.append(c5.forward_cached(c5.tokens[:, i].contiguous()))
    c5.start_cache(3, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c5.forward_cached(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = c5.forward_cached(static)
    c5.cache["lengths"].zero_()
    for i in range(12):
        static.copy_(c5.tokens[:, i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i]), i


@pytest.mark.parametrize("rotary_dim", [0, 32])
def test_training_variants_agree(rotary_dim):
    """The modules, the fused training form and the converted ones; gradients of the first two."""
    c5 = _stack(rotary_dim)
    plain = c5.forward()
    x = c5.emb(c5.tokens)
    for blk in c5.blocks:
        x = blk(x)
    reference = c5.final(x)
    loss = torch.randn_like(reference)
    params = [p for p in c5.blocks.parameters()]
    want = torch.autograd.grad(reference, params, loss)
    fused = c5.forward_train()
    assert _rel(fused, plain) < 1e-4
    for a, b in zip(torch.autograd.grad(fused, params, loss), want):
        assert _rel(a, b) < 1e-3
    c5.convert(inplace=False)
    c5.fuse()
    assert _rel(c5.forward_fused(False), plain) < 1e-4


def test_refused_steps_leave_the_caches_as_they_are():
    c5 = _stack(32)
    c5.convert()
    c5.fuse()
    for call in (c5.forward_prefix, c5.forward_cached):
        with pytest.raises(RuntimeError, match="start_cache"):
            call(c5.tokens[:, 0].contiguous())
    c5.start_cache(3, 15, prefix=25, page_size=32)
    starts = torch.tensor([0, 1, 2], dtype=torch.int32, device="cuda")
    for args in ((c5.tokens[:2, 0].contiguous(),), (c5.tokens[0, :2].contiguous(), starts)):
        with pytest.raises(RuntimeError, match="3 sequences"):
            c5.forward_cached(*args)
    assert not c5.cache["lengths"].any()
    c5.forward_cached(c5.tokens[:, 0].contiguous())
    with pytest.raises(RuntimeError, match="prefix"):  # (the tokens behind it would move)
        c5.forward_prefix(c5.tokens[0, :9])
    assert c5.cache["lengths"].tolist() == [1, 1, 1]
