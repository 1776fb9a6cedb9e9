"""The attention half of a block around its projections (HIP, no counterpart in ``bittorch.ops``): rotary positions, a paged cache of keys
and values, and the attention of new tokens over it.

* :func:`rotary` -- queries and keys turned by their positions, differentiable; :func:`rotary_frequencies` makes its table;
* :func:`paged_cache` -- the cache of one layer; :func:`cache_append` writes new tokens to it, their keys turned on the way, and turns their
  queries in the same launch; :func:`cache_read` gives back what a sequence holds;
* :func:`cached_attention` -- the new tokens over a prefix that all sequences share and over their own sequence's pages: one token a
  sequence or any number each.

The cache is two tensors ``[pages, kv_heads, page_size, features]`` in an order of its own (the one in which the matrix cores take its values,
``include/bittorch_hip.h``); a page can be copied, shared and handed on as a whole.  ``features`` is the head dimension rounded up to 64 bytes.
Sequence ``s`` owns the pages ``block_table[s]`` and ``lengths[s]`` places in them, its new tokens included: those are the last, and the rows
``q_starts[s] .. q_starts[s + 1] - 1`` of the call's tokens (ascending from 0; without ``q_starts``: one token a sequence).  All three are int32 on the GPU and are read
there, so that a captured call follows them.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Tuple, Union

import torch
from torch import Tensor

from ._autograd import differentiated


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[Dict] = None, device=None) -> Tuple[Tensor, float]:
    """``(inv_freq, amplitude)`` of :func:`rotary`: ``base ** (-2 i / rotary_dim)`` radians a position, float64 ``(rotary_dim / 2,)``, and 1.

    ``scaling`` fits them to contexts ``factor`` times as long as the model was trained on:

    * ``{"kind": "linear", "factor": f}``: every frequency divided by ``f``;
    * ``{"kind": "base", "factor": f}``: the base raised so that the lowest frequency is divided by ``f`` and the highest stays;
    * ``{"kind": "ramp", "factor": f, "original": n, "slow": 1, "fast": 32}``: waves that turn less than ``slow`` times in ``n`` positions are
      divided by ``f``, those that turn more than ``fast`` times stay, between them a linear ramp; the amplitude is ``0.1 ln f + 1``."""
    if rotary_dim < 2 or rotary_dim % 2:
        raise RuntimeError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not base > 0:
        raise RuntimeError("base must be positive")
    exponent = torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim
    amplitude = 1.0
    if scaling is None:
        return (base ** -exponent).to(device), amplitude
    given = dict(scaling)
    kind, factor = given.pop("kind", None), given.pop("factor", None)
    if factor is None or not factor >= 1:
        raise RuntimeError("scaling needs a factor of at least 1")
    if kind == "linear":
        inv_freq = base ** -exponent / factor
    elif kind == "base":
        if rotary_dim < 4:
            raise RuntimeError("scaling by the base needs two frequencies")
        inv_freq = (base * factor ** (rotary_dim / (rotary_dim - 2))) ** -exponent
    elif kind == "ramp":
        original, slow, fast = given.pop("original", None), given.pop("slow", 1.0), given.pop("fast", 32.0)
        if original is None or not original > 0 or not fast > slow:
            raise RuntimeError("a ramp needs original > 0 and fast > slow")
        inv_freq = base ** -exponent
        stays = ((original * inv_freq / (2 * math.pi) - slow) / (fast - slow)).clamp(0, 1)
        inv_freq = inv_freq * stays + inv_freq / factor * (1 - stays)
        amplitude = 0.1 * math.log(factor) + 1.0
    else:
        raise RuntimeError(f"scaling kind must be 'linear', 'base' or 'ramp', got {kind!r}")
    if given:
        raise RuntimeError(f"unknown entries of scaling: {', '.join(sorted(given))}")
    return inv_freq.to(device), amplitude


def _turned(x: Tensor, positions: Tensor, inv_freq: Tensor, interleaved: bool, amplitude: float) -> Tensor:
    """The definition in torch operations, in 32 bits (64 of 64-bit values); angles in 64."""
    n, dtype = 2 * inv_freq.shape[0], x.dtype
    wide = torch.float64 if dtype == torch.float64 else torch.float32
    angle = positions.double()[..., None, None] * inv_freq.double()
    cos, sin = (amplitude * angle.cos()).to(wide), (amplitude * angle.sin()).to(wide)
    part = x[..., :n].to(wide)
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :n // 2], part[..., n // 2:])
    a, b = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((part.to(dtype), x[..., n:]), -1)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q: Tensor, k: Optional[Tensor], positions: Tensor, inv_freq: Tensor, interleaved: bool, amplitude: float):
        from .. import _C

        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, inv_freq)
        ctx.how = interleaved, amplitude
        out = _C.rotary(q, k, positions, inv_freq, interleaved, amplitude)
        return out[0] if k is None else out

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads: Optional[Tensor]):
        from .. import _C

        positions, inv_freq = ctx.saved_tensors
        dq, dk = (*grads, None)[:2]
        dq, dk = dq if ctx.needs_input_grad[0] else None, dk if ctx.needs_input_grad[1] else None
        first, second = (dq, dk) if dq is not None else (dk, None)
        if first is not None:
            first, second = _C.rotary(first, second, positions, inv_freq, *ctx.how, backward=True)
        return (first, second, None, None, None, None) if dq is not None else (None, first, None, None, None, None)


def rotary(q: Tensor, k: Optional[Tensor], positions: Tensor, inv_freq: Tensor, interleaved: bool = False,
           amplitude: float = 1.0) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """Rotary positions: ``q`` ``(*, heads, D)`` and ``k`` ``(*, kv_heads, D)`` (or None) turned by ``positions`` (int32 or int64, any shape that broadcasts to
    ``*``).  The first ``2 len(inv_freq)`` features of a head are pairs ``(a, b)``, neighbours with ``interleaved`` and a half of them apart without, each turned
    by ``position * inv_freq`` radians (:func:`rotary_frequencies`; float32 or float64) and multiplied by ``amplitude``; the others stay.

    On the GPU fp32, fp16 or bf16, views with a stride for their tokens and heads read in place; rounded once, angles in 64 bits.  Differentiable (once)
    in ``q`` and ``k``; forward-mode derivatives are refused.  On the CPU: the same in plain torch operations."""
    from .. import _C

    out = _C._N.rotary(q, k, positions, inv_freq, interleaved, amplitude)
    if out is not None:
        return out
    if inv_freq.requires_grad:
        raise RuntimeError("inv_freq carries no gradient")
    if not q.is_cuda:
        _C.rotary_args(q, k, positions, inv_freq)
        pos = positions.expand(q.shape[:-2])
        out = _turned(q, pos, inv_freq, interleaved, amplitude)
        return out if k is None else (out, _turned(k, pos, inv_freq, interleaved, amplitude))
    if differentiated(q, k):
        return _Rotary.apply(q, k, positions, inv_freq, bool(interleaved), float(amplitude))
    out = _C.rotary(q, k, positions, inv_freq, interleaved, amplitude)
    return out[0] if k is None else out


def paged_cache(pages: int, kv_heads: int, head_dim: int, page_size: int = 64, dtype: torch.dtype = torch.bfloat16,
                device="cuda") -> Tuple[Tensor, Tensor]:
    """An empty cache of one layer, ``(k_cache, v_cache)``: ``pages`` pages of ``page_size`` places (a power of two from 32 on)."""
    from .. import _C

    if pages <= 0 or kv_heads <= 0 or page_size < 32 or page_size & (page_size - 1):
        raise RuntimeError("a cache needs pages, kv_heads and a page_size that is a power of two from 32 on")
    shape = (pages, kv_heads, page_size, _C.cache_head_dim(dtype, head_dim))
    return torch.zeros(shape, dtype=dtype, device=device), torch.zeros(shape, dtype=dtype, device=device)


def _natural(k: Tensor, v: Tensor) -> Tuple[Tensor, Tensor]:
    """Whole pages of a cache in the order ``[pages, kv_heads, places, features]``."""
    (n, h, p, d), e = k.shape, 16 // k.element_size()
    k = k.reshape(n, h, p // (4 * e), d // (4 * e), e // 4, 4, 4, 4, e).permute(0, 1, 2, 6, 4, 7, 3, 5, 8).reshape(n, h, p, d)
    return k, v.reshape(n, h, p // (4 * e), d // 16, 4, 16, e).permute(0, 1, 2, 4, 6, 3, 5).reshape(n, h, p, d)


def _tiled(k: Tensor, v: Tensor) -> Tuple[Tensor, Tensor]:
    """The reverse of :func:`_natural`."""
    (n, h, p, d), e = k.shape, 16 // k.element_size()
    k = k.reshape(n, h, p // (4 * e), 4, e // 4, 4, d // (4 * e), 4, e).permute(0, 1, 2, 6, 4, 7, 3, 5, 8).reshape(n, h, p, d)
    return k, v.reshape(n, h, p // (4 * e), 4, e, d // 16, 16).permute(0, 1, 2, 5, 3, 6, 4).reshape(n, h, p, d)


def cache_read(k_cache: Tensor, v_cache: Tensor, pages: Tensor, length: int, head_dim: int) -> Tuple[Tensor, Tensor]:
    """What the first ``length`` places of ``pages`` (a row of a block table) hold: keys and values ``[length, kv_heads, head_dim]``.  Places on pages outside
    the cache are not a number."""
    page = k_cache.shape[2]
    if not 0 <= length <= pages.numel() * page or not 0 < head_dim <= k_cache.shape[3]:
        raise RuntimeError("length or head_dim is beyond the pages")
    index, last = pages[:(length + page - 1) // page].long(), k_cache.shape[0] - 1
    wrong, index = ((index < 0) | (index > last))[:, None, None, None], index.clamp(0, last)
    k, v = _natural(*(t[index].masked_fill(wrong, math.nan) for t in (k_cache, v_cache)))
    return tuple(t.transpose(1, 2).flatten(0, 1)[:length, :, :head_dim] for t in (k, v))


def _refuse_gradients(*tensors: Optional[Tensor]) -> None:
    if differentiated(*tensors):
        raise RuntimeError("the cache and the attention over it carry no gradient: call under torch.no_grad()")


def _tokens_of(lengths: Tensor, q_starts: Optional[Tensor], tokens: int):
    """Of every sequence: its first token, number of tokens and length (CPU forms)."""
    starts = list(range(len(lengths) + 1)) if q_starts is None else q_starts.tolist()
    for s, length in enumerate(lengths.tolist()):
        begin = max(starts[s], 0)
        yield s, begin, max(min(starts[s + 1], tokens) - begin, 0), length


def cache_append(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor, q_starts: Optional[Tensor] = None,
                 q: Optional[Tensor] = None, inv_freq: Optional[Tensor] = None, interleaved: bool = False, amplitude: float = 1.0,
                 first_position: int = 0) -> Optional[Tensor]:
    """Writes the new tokens' keys and values ``[tokens, kv_heads, D]`` to the last places of their sequences (``lengths`` counts them already).  With
    ``inv_freq`` the keys are turned as in :func:`rotary`, at position ``first_position`` (a shared prefix's length) plus their place, and so is ``q``
    ``[tokens, heads, D]``, which is returned (None without).  ``k``, ``v`` and ``q`` may be views of one projection's output.

    Places below 0, behind ``block_table`` and on pages outside the cache are not written; of two tokens that the tables send to one place
    either stays; rows of the result behind the last sequence are zero.  No gradient.
    On the CPU: the same in plain torch operations."""
    from .. import _C

    out = _C._N.cache_append(k, v, k_cache, v_cache, block_table, lengths, q_starts, q, inv_freq, interleaved, amplitude, first_position)
    if out is not None:
        return out
    _refuse_gradients(k, v, q, inv_freq, k_cache, v_cache)
    if k.is_cuda:
        return _C.cache_append(k, v, k_cache, v_cache, block_table, lengths, q_starts, q, inv_freq, interleaved, amplitude, first_position)
    _C.append_args(k, v, k_cache, v_cache, block_table, lengths, q_starts, q, inv_freq)
    page, dim, out = k_cache.shape[2], k.shape[2], None if q is None else torch.zeros_like(q, memory_format=torch.contiguous_format)
    kn, vn = (t.clone() for t in _natural(k_cache, v_cache))
    for s, begin, n, length in _tokens_of(lengths, q_starts, k.shape[0]):
        place = torch.arange(length - n, length)
        rows = slice(begin, begin + n)
        keys = k[rows] if inv_freq is None else _turned(k[rows], place + first_position, inv_freq, interleaved, amplitude)
        if out is not None:
            out[rows] = _turned(q[rows], place + first_position, inv_freq, interleaved, amplitude)
        for i, at in enumerate(place.tolist()):
            number = int(block_table[s, at // page]) if 0 <= at < block_table.shape[1] * page else -1
            if 0 <= number < k_cache.shape[0]:
                kn[number, :, at % page, :dim], vn[number, :, at % page, :dim] = keys[i], v[begin + i]
    for cache, t in zip((k_cache, v_cache), _tiled(kn, vn)):
        cache.copy_(t)
    return out


def cached_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor, q_starts: Optional[Tensor] = None,
                     scale: Optional[float] = None, prefix_table: Optional[Tensor] = None, prefix_length: int = 0, return_lse: bool = False,
                     max_length: Optional[int] = None) -> Union[Tensor, Tuple[Tensor, Tensor]]:
    """``softmax(scale q K^T) V`` of the new tokens ``q`` ``[tokens, heads, D]`` over ``prefix_length`` places of the pages ``prefix_table`` ``[width]`` (int32), which
    all sequences share, and over the places of their own sequence up to their own; head ``h`` reads key head ``h // (heads / kv_heads)``.  ``scale``:
    ``D ** -0.5``.  The result is ``[tokens, heads, D]``; with ``return_lse`` the logarithms of the sums of exponentials follow, fp32 ``[tokens, heads]``.

    Tokens without a place to see, and rows behind the last sequence, are zero (``-inf``), and so are heads whose logits are all minus infinity; a logit of plus
    infinity, or one that is no number, makes the head not a number, an infinite value that it sees that feature infinite or not a number.  Places that a token does
    not see do not change its result, whatever they hold.  ``max_length``, if given, bounds the sequences' lengths on the host, where ``block_table`` is much wider than they are; tokens of longer sequences, and
    tokens that see a page outside the cache (others of that sequence may be), are not a number.

    Logits, sums and ``lse`` in 32 bits.  16-bit types: the weights are multiplied with the values in two halves of 16 bits where a call has few rows, and rounded to
    the type once where it has many (results are then 1.4 times as far from 64 bits as by their own rounding).  No gradient.  On the CPU: the same in plain
    torch operations."""
    from .. import _C

    out = _C._N.cached_attention(q, k_cache, v_cache, block_table, lengths, q_starts, scale, prefix_table, prefix_length, return_lse, max_length)
    if out is not None:
        return out
    _refuse_gradients(q, k_cache, v_cache)
    if q.is_cuda:
        return _C.cached_attention(q, k_cache, v_cache, block_table, lengths, q_starts, scale, prefix_table, prefix_length, return_lse, max_length)
    scale, longest = _C.attention_args(q, k_cache, v_cache, block_table, lengths, q_starts, scale, prefix_table, prefix_length, max_length)
    (tokens, heads, dim), (pages, kv_heads, page, _) = q.shape, k_cache.shape
    out, lse = torch.zeros(q.shape, dtype=q.dtype), torch.full((tokens, heads), -math.inf)
    for s, begin, n, length in _tokens_of(lengths, q_starts, tokens):
        kept = min(max(length, 0), longest)
        used = block_table[s, :(kept + page - 1) // page]
        shared = prefix_table[:(prefix_length + page - 1) // page] if prefix_length else used[:0]
        if length > longest:
            out[begin:begin + n], lse[begin:begin + n] = math.nan, math.nan
            continue
        bad = bool(((used < 0) | (used >= pages)).any() or ((shared < 0) | (shared >= pages)).any())
        own = cache_read(k_cache, v_cache, used.clamp(0, pages - 1), kept, dim)
        if prefix_length:
            own = [torch.cat(t) for t in zip(cache_read(k_cache, v_cache, shared.clamp(0, pages - 1), prefix_length, dim), own)]
        for i in range(n):
            seen = prefix_length + max(min(length - n + 1 + i, kept), 0)
            if seen == 0:
                continue
            k, v = (t[:seen].float().repeat_interleave(heads // kv_heads, 1) for t in own)
            x = torch.einsum("hd,khd->hk", q[begin + i].float(), k) * scale
            sums = x.logsumexp(-1).masked_fill((x == math.inf).any(-1), math.nan)
            weights = x.softmax(-1).masked_fill((sums == -math.inf)[:, None], 0.0)
            lse[begin + i] = math.nan if bad else sums
            out[begin + i] = math.nan if bad else torch.einsum("hk,khd->hd", weights, v).to(q.dtype)
    return (out, lse) if return_lse else out
