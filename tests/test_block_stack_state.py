"""``BlockStack``: what it holds goes when it goes, and a step that is refused leaves its caches as they were."""
import gc
import weakref

import pytest
import torch

from bittorch_amd.utils.block_stack import BlockStack


def _stack(**more):
    return BlockStack("cpu", layers=1, d_model=32, heads=2, ffn=32, batch=2, seq=8, vocab=8, act_dtype=torch.float32, **more)


@pytest.mark.parametrize("rotary_dim", [0, 8])
@pytest.mark.parametrize("converted", [False, True])
def test_a_stack_is_freed_without_the_collector(rotary_dim, converted):
    """Its weights are gigabytes at full size: no reference cycle may hold them until the next collection."""
    gc.collect()
    gc.disable()
    try:
        stack = _stack(rotary_dim=rotary_dim)
        stack.forward()
        if converted:
            stack.convert()
            stack.fuse()
            stack.start_cache(2, 8)
        held = [stack, stack.emb.weight, *((stack.infer or stack.blocks).buffers() if converted else stack.blocks.parameters())]
        alive = [weakref.ref(t) for t in held]
        del held, stack
        assert not any(r() is not None for r in alive)
    finally:
        gc.enable()


def test_a_step_that_fails_leaves_the_caches_as_they_are(monkeypatch):
    """Whatever it fails of, behind the checks of its arguments."""
    stack = _stack(rotary_dim=8)
    stack.convert()
    stack.fuse()
    stack.start_cache(2, 8, prefix=4)
    seen = []

    def fails(tokens, table, lengths, *more, **prefix):
        seen.append(lengths.tolist())
        raise RuntimeError("refused")

    def passes(tokens, table, lengths, *more, **prefix):
        seen.append(lengths.tolist())
        return torch.zeros(tokens.numel(), 32)

    state = lambda: (stack.cache["lengths"].tolist(), stack.cache["prefix_length"], stack.cache["begun"])  # noqa: E731
    counts = stack.cache["lengths"]
    starts = torch.tensor([0, 2, 3], dtype=torch.int32)
    for _ in range(2):
        monkeypatch.setattr(stack, "_cached", fails)
        with pytest.raises(RuntimeError, match="refused"):
            stack.forward_prefix(torch.zeros(3, dtype=torch.int64))
        assert state() == ([0, 0], 0, False)
        with pytest.raises(RuntimeError, match="refused"):
            stack.forward_cached(torch.zeros(2, dtype=torch.int64))
        assert state() == ([0, 0], 0, False)
    monkeypatch.setattr(stack, "_cached", passes)
    stack.forward_prefix(torch.zeros(3, dtype=torch.int64))
    assert state() == ([0, 0], 3, False)
    stack.forward_cached(torch.zeros(3, dtype=torch.int64), starts)
    assert state() == ([2, 1], 3, True) and stack.cache["lengths"] is counts
    monkeypatch.setattr(stack, "_cached", fails)
    with pytest.raises(RuntimeError, match="refused"):
        stack.forward_cached(torch.zeros(3, dtype=torch.int64), starts)
    assert state() == ([2, 1], 3, True)
    assert seen == [[3], [1, 1]] * 2 + [[3], [2, 1], [4, 2]]


def test_a_prefix_has_tokens():
    stack = _stack()
    stack.convert()
    stack.fuse()
    stack.start_cache(2, 8, prefix=4)
    with pytest.raises(RuntimeError, match="prefix"):
        stack.forward_prefix(torch.zeros(0, dtype=torch.int64))
    assert stack.cache["prefix_length"] == 0
