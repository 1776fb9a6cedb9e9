"""Per-module cache of the packed ternary weights.

The reference re-runs ``ternary_quantize`` on the master weights in every forward
(``bittorch/nn/ternary_linear.py:196-200``, ``bittorch/nn/ternary_linear_cuda.py:52-54``).
The result depends on the weights only, so a forward that cannot be a training step (gradient
mode off, or frozen weights) keeps it until the weights change: the key is the parameter's
version counter (every tracked in-place update, ``load_state_dict`` or optimizer step bumps it),
its storage address, dtype and device, and the quantizer's two settings, and the tensor has to be the
one that was packed (another may lie at its address; a parametrized weight is another at every reading).  Such a forward then
reads K*N/4 bytes of packed weights instead of 4*K*N bytes of masters -- and reads them from a decode-tiled copy
built next to the packed bytes (``_C.retile_weights``; whole-cache-line loads: what ``TernaryLinearInference`` runs
on), which such a module then holds as well, another K*N/4 bytes.  Up to 32 rows the output is the training forward's
bit for bit; a larger batch on the streaming kernel may split K differently on the tiled copy and on the row-major bytes,
and then sums in fp32 in another order (a difference in the last bits of the sums).

A training forward (gradient mode on and ``weight.requires_grad``) never uses the cache and
quantizes every time, exactly as the reference does: training code is where weights get written
through ``.data`` (``w.data.clamp_()``, ``p.data.add_(...)``, EMA copies), and writes through
``.data`` do not bump the version counter.  The one case that remains the caller's is an
evaluation-time write through ``.data``; ``module.invalidate_packed_cache()`` (or any tracked
write, e.g. ``with torch.no_grad(): w.copy_(...)``) makes the next forward re-quantize.
"""

from __future__ import annotations

import weakref
from typing import Optional, Sequence, Tuple

import torch
from torch import Tensor


def _capturing(device: torch.device, stream: int) -> bool:
    """Whether `stream`, that device's current one, is being captured into a graph (the default stream cannot be)."""
    if stream == 0:
        return False
    with torch.cuda.device(device):
        return torch.cuda.is_current_stream_capturing()


def _state(weight: Tensor) -> tuple:
    return weight._version, weight.data_ptr(), weight.dtype, weight.device


class _KeptWeights:
    """Packed weights and what they were packed of.  Another stream than the one that packed them waits for it.  A graph being captured
    packs for itself, whether anything is kept or not, and nothing of that is kept: its replays follow the masters, and read no memory that a
    later evaluation gives back."""

    __slots__ = ("held",)  # (one tuple, so that a call of another thread finds weights and what they are of together)

    def __init__(self) -> None:
        self.clear()

    def __reduce__(self):  # (a copy packs for itself)
        return type(self), ()

    def clear(self) -> None:
        self.held = None, (), None, None, None  # key, of, value, stream, packed

    @property
    def key(self):
        return self.held[0]

    @property
    def value(self):
        return self.held[2]

    def _kept(self, stream: int, of: Sequence[Tensor], key: tuple, pack):
        held, refs, value, of_stream, packed = self.held
        if key != held or any([r() is not t for r, t in zip(refs, of)]):
            value = pack()
            with torch.cuda.device(of[0].device):
                packed = torch.cuda.Event()
                packed.record()
            self.held = key, tuple(weakref.ref(t) for t in of), value, stream, packed
        elif stream != of_stream:
            here = torch.cuda.current_stream(of[0].device)
            here.wait_event(packed)
            for t in value:
                if t is not None:
                    t.record_stream(here)
        return value


class PackedWeightCache(_KeptWeights):
    __slots__ = ()

    @staticmethod
    def _pack(weight: Tensor, threshold_factor: float, per_channel: bool) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
        from .. import _C

        with torch.no_grad():
            packed, scale, _ = _C.ternary_quantize_pack(weight.detach(), threshold_factor, per_channel)
            n, k = weight.shape
            tiled_bytes = ((n + 15) // 16) * ((((k + 3) // 4) + 15) // 16) * 256
            return packed, scale, _C.retile_weights(packed, k) if tiled_bytes < 2 ** 32 else None

    def get(self, weight: Tensor, threshold_factor: float, per_channel: bool) -> Tuple[Tensor, Tensor, Optional[Tensor]]:
        """``(packed_T uint8 [ceil(K/4), N], scale fp32 [N] or 0-dim, tiled)`` of the current weights; ``tiled`` is
        the decode-tiled copy of ``packed_T`` (``_C.retile_weights``), or None where the tiled kernels' 32-bit
        offsets do not reach."""
        from .. import _C

        stream = _C._stream(weight)
        if _capturing(weight.device, stream):
            return self._pack(weight, threshold_factor, per_channel)
        key = *_state(weight), float(threshold_factor), bool(per_channel)
        return self._kept(stream, (weight,), key, lambda: self._pack(weight, threshold_factor, per_channel))


class GatedWeightCache(_KeptWeights):
    """The packed weights of a gated pair (``_C.gated_weights``: both layers in one tiled copy, tiles of gate and up in turn), kept by the
    same rules."""

    __slots__ = ()

    @staticmethod
    def _pack(gate, up):
        from .. import _C

        with torch.no_grad():
            w, _, scale, bias = _C.gated_weights(gate.weight, up.weight, gate.bias, up.bias, gate.threshold_factor, gate.per_channel)
        return w, scale[:-1], bias

    def get(self, gate, up):
        from .. import _C

        stream = _C._stream(gate.weight)
        if _capturing(gate.weight.device, stream):
            return self._pack(gate, up)
        of = [t for t in (gate.weight, up.weight, gate.bias, up.bias) if t is not None]
        key = *map(_state, of), gate.bias is None, up.bias is None, float(gate.threshold_factor), bool(gate.per_channel)
        return self._kept(stream, of, key, lambda: self._pack(gate, up))

    def forward(self, x: Tensor, gate, up) -> Tensor:
        """``silu(gate(x)) * up(x)`` as ``TernarySwiGLU`` computes it."""
        from .. import _C

        w, scale, bias = self.get(gate, up)
        f = gate.out_features
        h = _C.ternary_linear_tiled_forward(x.contiguous(), w, scale, bias, gate.in_features, scale.numel(), swiglu_pairs=True)
        return h if h.shape[-1] == f else h[..., :f].contiguous()


def cache_usable(x: Tensor, *of: Tensor) -> bool:
    """The cache holds the quantization of the stored weights (``of``, with the biases where those are kept too) in their own dtype.  A
    training forward re-quantizes (see above).  Under autocast the autograd function quantizes an fp16 copy instead
    (reference semantics), and float64 runs on the dense entry point, so neither uses it.  A tensor made in inference
    mode has no version counter."""
    learning = torch.is_grad_enabled()
    if any((learning and t.requires_grad) or t.is_inference() or t.dtype == torch.float64 for t in of):
        return False
    return not torch.is_autocast_enabled() and x.dtype != torch.float64
