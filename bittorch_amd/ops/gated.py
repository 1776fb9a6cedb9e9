"""``ternary_gated_linear``: the gated pair of a feed-forward block on full-precision masters, ``silu(gate(x)) * up(x)``, with its
gradient.

No counterpart in ``bittorch.ops``; the arithmetic is that of two ``TernaryLinear`` layers (``bittorch/nn/ternary_linear_cuda.py:23-111``)
and of the SwiGLU between them (``js/src/models/TernaryTransformer.ts:366-423``).  Both masters are ternarised as they are read, one
product forms both projections with ``silu(g) * u`` in its output stage, and one pass over the kept projections feeds both products
of the gradient.
"""

from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch import Tensor

from ..quant.ternary import ternary_quantize_ste
from ._autograd import differentiated


def _half(t: Optional[Tensor]) -> Optional[Tensor]:
    """What autocast does with an argument of a ternary layer: GPU floating-point tensors become fp16."""
    return None if t is None else t.half()


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, gate: Tensor, up: Tensor, gate_bias: Optional[Tensor], up_bias: Optional[Tensor],
                threshold_factor: float, per_channel: bool, keep: bool) -> Tensor:
        ctx.masters = gate.dtype, None if gate_bias is None else gate_bias.dtype, None if up_bias is None else up_bias.dtype
        ctx.x_dtype = x.dtype
        if not torch.is_autocast_enabled("cuda"):
            return _GatedLinear._forward(ctx, x, gate, up, gate_bias, up_bias, threshold_factor, per_channel, keep, False)
        with torch.autocast("cuda", enabled=False):  # (as TernaryLinear: fp32 masters are rounded as the quantizer reads them)
            as_half = gate.dtype == torch.float32
            return _GatedLinear._forward(ctx, _half(x), gate if as_half else _half(gate), up if as_half else _half(up), _half(gate_bias),
                                         _half(up_bias), threshold_factor, per_channel, keep, as_half)

    @staticmethod
    def _forward(ctx, x, gate, up, gate_bias, up_bias, threshold_factor, per_channel, keep, as_half) -> Tensor:
        from .. import _C

        f, k = gate.shape
        x2 = x.reshape(-1, k)
        if not keep and _C.gated_masters_serves(x2.shape[0], gate, per_channel, as_half):
            h = _C.gated_masters_forward(x2, gate, up, gate_bias, up_bias, threshold_factor, as_half)
            return h.reshape(*x.shape[:-1], f)
        w, w_back, scale, bias = _C.gated_weights(gate, up, gate_bias, up_bias, threshold_factor, per_channel, as_half,
                                                  back=keep and ctx.needs_input_grad[0])
        if x.dtype == torch.float32:
            # (the fp32 kernel of the masters' gradient takes four columns and more)
            x2 = F.pad(x2, (0, 4 - k)) if k < 4 else x2.contiguous()
            fp = scale.numel() // 2
            pre = _C.ternary_linear_tiled_forward(x2, w, scale[:2 * fp], bias, x2.shape[1], 2 * fp, natural_from_pairs=True)
            h = _C.swiglu(pre[:, :f], pre[:, fp:fp + f])
        else:
            h, pre, x2 = _C.ternary_gated_forward(x2, w, scale, bias, f, keep)
        if keep:
            ctx.save_for_backward(x2, pre, w_back, _C.gated_split(scale, f) if x.dtype == torch.float16 else scale)
            ctx.shape = f, k
        return h.reshape(*x.shape[:-1], f)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh: Tensor):
        with torch.autocast("cuda", enabled=False):  # (as the forward)
            return _GatedLinear._backward(ctx, dh)

    @staticmethod
    def _backward(ctx, dh: Tensor):
        from .. import _C

        x2, pre, w_back, scale = ctx.saved_tensors
        (f, k), (w_dtype, gb_dtype, ub_dtype) = ctx.shape, ctx.masters
        want_x, want_g, want_u, want_gb, want_ub = ctx.needs_input_grad[:5]
        lead, dh = dh.shape[:-1], dh.reshape(-1, f).contiguous()
        dx = dg = du = dgb = dub = None
        want_w, want_b = want_g or want_u, want_gb or want_ub
        b_dtype = (gb_dtype if gb_dtype == ub_dtype or not want_ub else ub_dtype if not want_gb else torch.float32) if want_b else None
        fp, split = (f + 15) // 16 * 16, dh.dtype == torch.float16  # (split: scale is that of gated_split)
        g, db = _C.gated_grad(dh, pre, scale[:2 * fp + 1], b_dtype)
        one = scale[2 * fp:2 * fp + 1]
        if want_x and split:
            dx = _C.gated_grad_input(g, w_back, scale, f, k).reshape(*lead, k).to(ctx.x_dtype)
        elif want_x:
            dx = _C.ternary_linear_tiled_forward(g, w_back, one, None, 2 * fp, k).reshape(*lead, k).to(ctx.x_dtype)
        if want_w and dh.dtype == torch.float32:
            dw, _ = _C.linear_grad_weight(g, x2, one)
            dg, du = (t.to(w_dtype).contiguous() for t in (dw[:f, :k], dw[fp:fp + f, :k]))
        elif want_w:
            dw = _C.gated_grad_masters(g, x2, scale[2 * fp + 16:4 * fp + 16] if split else one, f, k, dh.dtype if w_dtype == dh.dtype else torch.float32)
            dg, du = dw[:f].to(w_dtype), dw[f:].to(w_dtype)
        if want_b:
            dgb, dub = db[:f].to(gb_dtype) if want_gb else None, db[f:].to(ub_dtype) if want_ub else None
        return dx, dg if want_g else None, du if want_u else None, dgb, dub, None, None, None


def _check_gated(x: Tensor, gate: Tensor, up: Tensor, gate_bias: Optional[Tensor], up_bias: Optional[Tensor]) -> None:
    def check(cond: bool, msg: str) -> None:
        if not cond:
            raise RuntimeError(msg)

    check(gate.dim() == 2 and gate.shape == up.shape and gate.dtype == up.dtype, "gate and up weights must match, 2D [F, K]")
    check(gate.numel() > 0, "weight is empty")
    check(x.dim() >= 1 and x.numel() > 0, "x is empty")
    check(x.shape[-1] == gate.shape[1], "input K doesn't match weight K")
    for b in (gate_bias, up_bias):
        check(b is None or (b.dim() == 1 and b.shape[0] == gate.shape[0]), "bias shape mismatch")
    check(all(t is None or t.device == x.device for t in (gate, up, gate_bias, up_bias)), "All tensors must be on one device")


def _one_by_one(x, gate, up, gate_bias, up_bias, threshold_factor, per_channel) -> Tensor:
    from ..nn.ternary_linear_cuda import TernaryLinearCUDAFunction

    _check_gated(x, gate, up, gate_bias, up_bias)
    g, u = (TernaryLinearCUDAFunction.apply(x, w, b, threshold_factor, per_channel, None) for w, b in ((gate, gate_bias), (up, up_bias)))
    return F.silu(g) * u


def ternary_gated_linear(x: Tensor, gate_weight: Tensor, up_weight: Tensor, gate_bias: Optional[Tensor] = None,
                         up_bias: Optional[Tensor] = None, threshold_factor: float = 0.05, per_channel: bool = True) -> Tensor:
    """``silu(linear(x, T(gate_weight), gate_bias)) * linear(x, T(up_weight), up_bias)`` with ``T(w) = ternary_quantize(w)`` times its
    scale: ``x`` ``(*, K)``, masters ``(F, K)``, result ``(*, F)`` in ``x``'s dtype.

    On the GPU ``x`` and the masters are fp32, fp16 or bf16, in any combination; 16-bit results are rounded once, from fp32 projections.
    Differentiable (once) in all five tensors with the straight-through gradient of ``TernaryLinear``; the gradients of the masters and
    biases have their dtype.  Forward-mode derivatives are refused on the GPU.  Under autocast it runs in fp16, as ``TernaryLinear``.  On the CPU: the same in plain torch operations."""
    if x.is_cuda:
        from .. import _C

        if _C._N.generic_kernel_asked():  # (BITTORCH_KERNEL=generic: the layers one by one, which know that switch)
            return _one_by_one(x, gate_weight, up_weight, gate_bias, up_bias, threshold_factor, per_channel)
        h = _C._N.gated_linear(x, gate_weight, up_weight, gate_bias, up_bias, threshold_factor, per_channel)
        if h is not None:
            return h
    _check_gated(x, gate_weight, up_weight, gate_bias, up_bias)
    if not x.is_cuda:
        g, u = (F.linear(x, (q * s.reshape(-1, 1)).to(x.dtype), None if b is None else b.to(x.dtype))
                for (q, s), b in ((ternary_quantize_ste(w, threshold_factor, per_channel), b)
                                  for w, b in ((gate_weight, gate_bias), (up_weight, up_bias))))
        return F.silu(g) * u
    kinds = (torch.float32, torch.float16, torch.bfloat16)
    if x.dtype not in kinds or gate_weight.dtype not in kinds or any(b is not None and b.dtype not in kinds for b in (gate_bias, up_bias)):
        raise RuntimeError("x, weights and biases must be float32, float16 or bfloat16")
    keep = differentiated(x, gate_weight, up_weight, gate_bias, up_bias)
    return _GatedLinear.apply(x, gate_weight, up_weight, gate_bias, up_bias, threshold_factor, per_channel, keep)
