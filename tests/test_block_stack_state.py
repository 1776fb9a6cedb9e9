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
