"""``bittorch._C`` look-alike over the C-ABI HIP library.

Same four entry points, argument order and keyword names as the reference's
pybind11 module (``csrc/bindings/bittorch_bindings.cpp:34-88``) with the host
checks of ``csrc/core/dispatch.cpp:52-142``; additional entry points expose
the fused quantize+pack kernel and the int8 pipeline stages.  Tensors are
passed to the library as raw device pointers; outputs and scratch are
allocated here with torch so the library itself never allocates.

The functions of small calls first ask ``_calls`` (``csrc/calls.cpp``), which does the same in native code for
an ordinary call and returns None for any other.

Importing this module raises ``ImportError`` when the library is not built.
"""

from __future__ import annotations

import contextlib
import os

from typing import Optional, Tuple

import torch
from torch import Tensor

from . import _lib

_L = _lib.load()  # ImportError here == "extension not available"
_N = _lib.load_calls()

_DT = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_INT8_OUT = 3
_F32_AS_F16 = 4  # bt_quantize_pack: fp32 weights quantized as their fp16 copy


def _check(cond: bool, msg: str) -> None:
    if not cond:
        raise RuntimeError(msg)


def _status(rc: int) -> None:
    if rc != 0:
        raise RuntimeError(_lib.last_error() or f"libbittorch_hip call failed ({rc})")


# A call's host time is most of a small launch's (one fp16 row through 4096 x 4096: 4.6 us on the GPU, 14 us a call).  The public
# forms of the next two build a stream object and enter a context, 3 us a call: the handle and the device are asked for instead.
_HERE = contextlib.nullcontext()


def _stream(t: Tensor) -> int:
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _on(t: Tensor):
    """Context in which ``t``'s device is the current one."""
    return _HERE if torch._C._cuda_getDevice() == t.get_device() else torch.cuda.device(t.device)


def _ptr(t: Optional[Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dt(t: Tensor, what: str) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise RuntimeError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}") from None


def _workspace(nbytes: int, device) -> Optional[Tensor]:
    """Scratch of one library call (the library needs no initialisation of it), its own: a call makes several launches and
    ctypes lets go of the interpreter lock, so calls of other host threads can come between them on the same stream; and a
    captured graph's launches keep addressing theirs, which the graph's pool then holds."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes > 0 else None


def _all_cuda(*ts: Optional[Tensor]) -> bool:
    for t in ts:
        if t is not None and not t.is_cuda:
            return False
    return True


def _flat_rows(X: Tensor, K: int) -> Tensor:
    """``X`` as contiguous ``[rows, K]``; most calls' already are."""
    return X if X.dim() == 2 and X.stride(0) == K and X.is_contiguous() else X.contiguous().reshape(-1, K)


def _unflat(y: Tensor, X: Tensor, N: int) -> Tensor:
    return y if X.dim() == 2 else y.reshape(*X.shape[:-1], N)


def _prep_vec(v: Tensor, x: Tensor) -> Tensor:
    """scale / bias operand: contiguous, in a dtype the kernels read (fp32 or 16-bit)."""
    if v.dtype not in _DT:
        v = v.to(x.dtype if x.dtype in _DT else torch.float32)
    return v.contiguous()


def dummy(input: Tensor) -> Tensor:
    """Copy of the input (reference ``dispatch.cpp:7-9``)."""
    return input.clone()


def _float64_packed(X, W_T, scale, bias, in_features):
    from .quant.ternary_packed import unpack_ternary_transposed
    w = unpack_ternary_transposed(W_T, in_features).to(X.dtype) * scale.to(X.dtype).unsqueeze(1)
    return torch.nn.functional.linear(X, w, None if bias is None else bias.to(X.dtype))


def pack_ternary_int8(W_tern: Tensor) -> Tensor:
    """Dense ternary ``[N, K]`` int8 on the GPU -> packed transposed ``[ceil(K/4), N]`` uint8
    (the bytes of ``quant.pack_ternary_transposed``)."""
    _check(W_tern.dim() == 2 and W_tern.dtype == torch.int8, "W_tern must be 2D int8")
    _check(W_tern.is_cuda, "All tensors must be CUDA")
    W_tern = W_tern.contiguous()
    N, K = W_tern.shape
    packed = torch.empty(((K + 3) // 4, N), dtype=torch.uint8, device=W_tern.device)
    with _on(W_tern):
        _status(_L.bt_pack_ternary_i8(W_tern.data_ptr(), N, K, packed.data_ptr(), _stream(W_tern)))
    return packed


def ternary_linear_forward(X: Tensor, W_tern: Tensor, scale: Tensor,
                           bias: Optional[Tensor] = None) -> Tensor:
    """``Y = X @ (W_tern * scale).T + bias`` with dense int8 ternary weights ``[N, K]``.

    Reference: ``bittorch_bindings.cpp:41-46``, ``dispatch.cpp:52-87``.
    """
    _check(X.dim() >= 1, "X must have at least 1 dimension")
    _check(X.numel() > 0, "X is empty")
    _check(W_tern.dim() == 2, "W_tern must be 2D [N, K]")
    _check(W_tern.dtype == torch.int8, "W_tern must be int8")
    _check(scale.dim() == 1, "scale must be 1D [N]")
    K = X.shape[-1]
    N, WK = W_tern.shape
    _check(K == WK, "input K doesn't match weight K")
    _check(scale.shape[0] in (N, 1), "scale size doesn't match N")
    if bias is not None:
        _check(bias.dim() == 1 and bias.shape[0] == N, "bias shape mismatch")
    _check(_all_cuda(X, W_tern, scale, bias), "All tensors must be CUDA")
    if X.dtype == torch.float64:
        w = W_tern.to(X.dtype) * scale.to(X.dtype).unsqueeze(1)
        return torch.nn.functional.linear(X, w, None if bias is None else bias.to(X.dtype))
    W_tern = W_tern.contiguous()
    if os.environ.get("BITTORCH_KERNEL", "auto") != "generic":
        # the weights are packed on the device (one read of N*K bytes) and the call joins the
        # packed matrix-core path; entries are taken as ternary (sign of anything non-zero)
        return ternary_linear_packed_forward(X, pack_ternary_int8(W_tern), scale, bias, K)
    x2 = _flat_rows(X, K)
    scale = _prep_vec(scale, x2)
    bias = None if bias is None else _prep_vec(bias, x2)
    B = x2.shape[0]
    y = torch.empty((B, N), dtype=X.dtype, device=X.device)
    with _on(X):
        _status(_L.bt_ternary_linear_forward(
            x2.data_ptr(), _dt(x2, "X"), W_tern.data_ptr(), scale.data_ptr(), _dt(scale, "scale"),
            scale.numel(), _ptr(bias), 0 if bias is None else _dt(bias, "bias"), y.data_ptr(),
            B, N, K, _stream(X)))
    return _unflat(y, X, N)


def _packed_checks(X, W_T, scale, bias, in_features, flatten: bool = True):
    _check(X.dim() >= 1, "X must have at least 1 dimension")
    _check(X.numel() > 0, "X is empty")
    _check(W_T.dim() == 2, "W_T must be 2D [K_bytes, N]")
    _check(W_T.dtype == torch.uint8, "W_T must be uint8")
    _check(scale.dim() == 1, "scale must be 1D [N]")
    K = X.shape[-1]
    K_bytes, N = W_T.shape
    _check(K == in_features, "input K doesn't match in_features")
    _check(K_bytes == (in_features + 3) // 4, "K_bytes doesn't match ceil(K/4)")
    _check(scale.shape[0] in (N, 1), "scale size doesn't match N")
    if bias is not None:
        _check(bias.dim() == 1 and bias.shape[0] == N, "bias shape mismatch")
    _check(_all_cuda(X, W_T, scale, bias), "All tensors must be CUDA")
    return K, N


def _residual_2d(residual: Tensor, like: Tensor, lead_shape, N: int) -> Tensor:
    _check(residual.shape == (*lead_shape, N), "residual shape doesn't match the output")
    _check(residual.dtype == like.dtype, "residual must have the output's dtype")
    _check(residual.device == like.device, "All tensors must be CUDA")
    r = residual.contiguous()
    if r.data_ptr() % 16:  # a view that starts inside a buffer: the epilogues read the residual in 16-byte pieces
        r = r.clone()
    return r.reshape(-1, N)


def ternary_linear_packed_forward(X: Tensor, W_T: Tensor, scale: Tensor,
                                  bias: Optional[Tensor] = None, in_features: int = -1,
                                  residual: Optional[Tensor] = None) -> Tensor:
    """Packed-weight forward, fp32 accumulation; ``W_T`` is ``[ceil(K/4), N]`` uint8.

    Reference: ``bittorch_bindings.cpp:48-63``, ``dispatch.cpp:105-142``.  ``scale``
    may be fp32 or the activation dtype and may have one entry (per-tensor scale).
    ``residual`` (additive, not in the reference): a tensor of the output's shape and dtype
    added in the kernel's epilogue with the two roundings of ``linear(x) + residual``.
    """
    if residual is None:
        y = _N.packed_forward(X, W_T, scale, bias, X.shape[-1] if in_features < 0 and X.dim() > 0 else in_features)
        if y is not None:
            return y
    if in_features < 0:
        in_features = X.shape[-1]
    K, N = _packed_checks(X, W_T, scale, bias, in_features)
    if X.dtype == torch.float64:
        y = _float64_packed(X, W_T, scale, bias, in_features)
        return y if residual is None else y + residual
    x2 = _flat_rows(X, K)
    W_T = W_T.contiguous()
    scale = _prep_vec(scale, x2)
    bias = None if bias is None else _prep_vec(bias, x2)
    B = x2.shape[0]
    xdt = _dt(x2, "X")
    y = torch.empty((B, N), dtype=X.dtype, device=X.device)
    with _on(X):
        ws_bytes = _L.bt_packed_forward_workspace_bytes(B, N, K, xdt)
        ws = _workspace(ws_bytes, X.device)
        if residual is None:
            _status(_L.bt_ternary_linear_packed_forward(
                x2.data_ptr(), xdt, W_T.data_ptr(), scale.data_ptr(), _dt(scale, "scale"), scale.numel(),
                _ptr(bias), 0 if bias is None else _dt(bias, "bias"), y.data_ptr(), B, N, K,
                _ptr(ws), 0 if ws is None else ws.numel(), _stream(X)))
        else:
            res = _residual_2d(residual, X, X.shape[:-1], N)
            _status(_L.bt_ternary_linear_packed_forward_res(
                x2.data_ptr(), xdt, W_T.data_ptr(), scale.data_ptr(), _dt(scale, "scale"), scale.numel(),
                _ptr(bias), 0 if bias is None else _dt(bias, "bias"), res.data_ptr(), y.data_ptr(), B, N, K,
                _ptr(ws), 0 if ws is None else ws.numel(), _stream(X)))
    return _unflat(y, X, N)


def ternary_linear_packed_forward_fused(X: Tensor, W_T: Tensor, scale: Tensor, bias: Optional[Tensor] = None,
                                        in_features: int = -1, residual: Optional[Tensor] = None,
                                        norm: Optional[Tuple[Optional[Tensor], float]] = None,
                                        swiglu_up: Optional[Tensor] = None) -> Tensor:
    """``linear(pro(X)) [+ residual]`` with ``pro`` = RMSNorm (``norm=(weight or None, eps)``) or
    SwiGLU (``X`` is the gate, ``swiglu_up`` the other factor): the values :func:`rmsnorm` /
    :func:`swiglu` would store, without the extra launch when ``X`` is one 16-bit row (a decode token)."""
    _check((norm is None) != (swiglu_up is None), "exactly one of norm and swiglu_up must be given")
    if in_features < 0:
        in_features = X.shape[-1]
    K, N = _packed_checks(X, W_T, scale, bias, in_features)
    _check(X.dtype in _DT, "X must be float32, float16 or bfloat16")
    x2 = _rows_2d(X, K)
    W_T = W_T.contiguous()
    scale = _prep_vec(scale, x2)
    bias = None if bias is None else _prep_vec(bias, x2)
    B = x2.shape[0]
    if norm is not None:
        w, eps = norm
        if w is not None:
            _check(w.dim() == 1 and w.shape[0] == K, "norm weight must be 1D [K]")
            w = w.to(X.dtype).contiguous()
        op, pb, ldb = 1, w, 0
    else:
        _check(swiglu_up.shape == X.shape and swiglu_up.dtype == X.dtype, "gate and up must match in shape and dtype")
        u2 = _rows_2d(swiglu_up, K)
        op, pb, ldb, eps = 2, u2, u2.stride(0), 0.0
    _check(_all_cuda(pb), "All tensors must be CUDA")
    xdt = _dt(x2, "X")
    y = torch.empty((B, N), dtype=X.dtype, device=X.device)
    res = None if residual is None else _residual_2d(residual, X, X.shape[:-1], N)
    with _on(X):
        ws = _workspace(_L.bt_packed_forward_fused_workspace_bytes(B, N, K, xdt), X.device)
        _status(_L.bt_ternary_linear_packed_forward_fused(
            x2.data_ptr(), x2.stride(0), xdt, op, _ptr(pb), ldb, float(eps), W_T.data_ptr(), scale.data_ptr(),
            _dt(scale, "scale"), scale.numel(), _ptr(bias), 0 if bias is None else _dt(bias, "bias"), _ptr(res),
            y.data_ptr(), B, N, K, _ptr(ws), 0 if ws is None else ws.numel(), _stream(X)))
    return _unflat(y, X, N)


def retile_weights(W_T: Tensor, in_features: int, gate_up_pairs: bool = False) -> Tensor:
    """Decode-tiled copy of ``W_T [ceil(K/4), N]`` (flat uint8 tensor): per 16-column tile and 16-row step
    the 64 dwords a wave of the decode kernel loads, contiguous.  Built once; :func:`untile_weights` inverts it.
    ``gate_up_pairs`` (N % 32 == 0): the tiles of the two column halves alternate, for the SwiGLU output stage
    of :func:`ternary_linear_tiled_forward` (such a copy serves only that)."""
    _check(W_T.dim() == 2 and W_T.dtype == torch.uint8, "W_T must be 2D uint8 [K_bytes, N]")
    _check(not gate_up_pairs or W_T.shape[1] % 32 == 0, "gate/up pair order needs N % 32 == 0")
    _check(W_T.shape[0] == (in_features + 3) // 4, "K_bytes doesn't match ceil(K/4)")
    _check(_all_cuda(W_T), "All tensors must be CUDA")
    W_T = W_T.contiguous()
    N = W_T.shape[1]
    with _on(W_T):
        out = torch.empty((_L.bt_tiled_weights_bytes(N, in_features),), dtype=torch.uint8, device=W_T.device)
        _status(_L.bt_retile_weights(W_T.data_ptr(), N, in_features, 1 if gate_up_pairs else 0, out.data_ptr(),
                                     _stream(W_T)))
    return out


def _tiled_checks(W_tiled: Tensor, N: int, K: int):
    _check(W_tiled.dtype == torch.uint8 and W_tiled.dim() == 1 and W_tiled.is_contiguous(),
           "W_tiled must be the flat uint8 tensor retile_weights returned")
    _check(N > 0 and K > 0 and W_tiled.numel() == _L.bt_tiled_weights_bytes(N, K),
           "W_tiled size doesn't match out_features x in_features")


def untile_weights(W_tiled: Tensor, out_features: int, in_features: int, gate_up_pairs: bool = False) -> Tensor:
    """``W_T [ceil(K/4), N]`` back from its decode-tiled copy (exact inverse of :func:`retile_weights`)."""
    _tiled_checks(W_tiled, out_features, in_features)
    _check(_all_cuda(W_tiled), "All tensors must be CUDA")
    with _on(W_tiled):
        out = torch.empty(((in_features + 3) // 4, out_features), dtype=torch.uint8, device=W_tiled.device)
        _status(_L.bt_untile_weights(W_tiled.data_ptr(), out_features, in_features, 1 if gate_up_pairs else 0,
                                     out.data_ptr(), _stream(W_tiled)))
    return out


def ternary_linear_tiled_forward(X: Tensor, W_tiled: Tensor, scale: Tensor, bias: Optional[Tensor] = None,
                                 in_features: int = -1, out_features: int = -1, residual: Optional[Tensor] = None,
                                 norm: Optional[Tuple[Optional[Tensor], float]] = None,
                                 swiglu_up: Optional[Tensor] = None, swiglu_pairs: bool = False,
                                 natural_from_pairs: bool = False) -> Tensor:
    """:func:`ternary_linear_packed_forward` / ``_fused`` on the decode-tiled copy of the weights: the same results
    bit for bit up to 32 rows and in the tiled GEMMs; a larger batch on the streaming kernel may split K among its waves
    differently on the two layouts, and the kernel for a few tens of 16-bit rows, priced for each layout by itself, may serve one
    alone: fp32 sums that differ in their last bits.
    ``swiglu_pairs`` (copy built with ``gate_up_pairs=True``): the layer's columns are ``[gate | up]`` and the
    output is the MLP's hidden vector ``swiglu(gate(x), up(x))`` ``[*, N/2]``, formed in the kernel's output stage.
    ``natural_from_pairs``: the same pair-ordered copy read as an ordinary linear layer (output ``[*, N]`` in natural
    column order, bit-identical to a natural-order copy's)."""
    y = _N.tiled_forward(X, W_tiled, scale, bias, in_features, out_features, residual, norm, swiglu_up, swiglu_pairs, natural_from_pairs)
    if y is not None:
        return y
    _check(not (swiglu_pairs and natural_from_pairs), "swiglu_pairs and natural_from_pairs exclude each other")
    _check(not natural_from_pairs or out_features % 32 == 0, "a pair-ordered copy has N % 32 == 0")
    _check(not swiglu_pairs or (residual is None and swiglu_up is None and out_features % 32 == 0),
           "swiglu_pairs needs N % 32 == 0 and takes neither a residual nor a SwiGLU prologue")
    _check(norm is None or swiglu_up is None, "at most one of norm and swiglu_up may be given")
    _check(X.dim() >= 1 and X.numel() > 0, "X is empty")
    K, N = X.shape[-1], out_features
    _check(K == in_features, "input K doesn't match in_features")
    _tiled_checks(W_tiled, N, K)
    _check(scale.dim() == 1 and scale.shape[0] in (N, 1), "scale size doesn't match N")
    _check(bias is None or (bias.dim() == 1 and bias.shape[0] == N), "bias shape mismatch")
    _check(_all_cuda(X, W_tiled, scale, bias), "All tensors must be CUDA")
    _check(X.dtype in _DT, "X must be float32, float16 or bfloat16")
    x2 = _rows_2d(X, K) if (norm is not None or swiglu_up is not None) else _flat_rows(X, K)
    scale = _prep_vec(scale, x2)
    bias = None if bias is None else _prep_vec(bias, x2)
    B = x2.shape[0]
    op, pb, ldb, eps = 0, None, 0, 0.0
    if norm is not None:
        w, eps = norm
        if w is not None:
            _check(w.dim() == 1 and w.shape[0] == K, "norm weight must be 1D [K]")
            w = w.to(X.dtype).contiguous()
        op, pb = 1, w
    elif swiglu_up is not None:
        _check(swiglu_up.shape == X.shape and swiglu_up.dtype == X.dtype, "gate and up must match in shape and dtype")
        pb = _rows_2d(swiglu_up, K)
        op, ldb = 2, pb.stride(0)
    _check(_all_cuda(pb), "All tensors must be CUDA")
    xdt = _dt(x2, "X")
    Ny = N // 2 if swiglu_pairs else N
    y = torch.empty((B, Ny), dtype=X.dtype, device=X.device)
    res = None if residual is None else _residual_2d(residual, X, X.shape[:-1], N)
    with _on(X):
        query = _L.bt_tiled_forward_workspace_bytes if op == 0 and not swiglu_pairs else _L.bt_packed_forward_fused_workspace_bytes
        ws = _workspace(query(B, N, K, xdt), X.device)
        _status(_L.bt_ternary_linear_tiled_forward(
            x2.data_ptr(), x2.stride(0), xdt, op, _ptr(pb), ldb, float(eps), W_tiled.data_ptr(), scale.data_ptr(),
            _dt(scale, "scale"), scale.numel(), _ptr(bias), 0 if bias is None else _dt(bias, "bias"), _ptr(res),
            1 if swiglu_pairs else 2 if natural_from_pairs else 0, y.data_ptr(), B, N, K, _ptr(ws), 0 if ws is None else ws.numel(), _stream(X)))
    return _unflat(y, X, Ny)


def pointer_table(tensors) -> Tensor:
    """Device array of the tensors' device addresses (int64), the form :func:`ternary_gemv_grouped` takes its
    operands in.  The caller keeps the tensors alive for as long as the table is used."""
    tensors = list(tensors)
    _check(len(tensors) > 0 and _all_cuda(*tensors), "All tensors must be CUDA")
    return torch.tensor([t.data_ptr() for t in tensors], dtype=torch.int64, device=tensors[0].device)


def ternary_gemv_grouped(x_tab: Tensor, w_tiled_tab: Tensor, scale_tab: Tensor, bias_tab: Optional[Tensor],
                         y_tab: Tensor, in_features: int, out_features: int, scale_len: int = -1,
                         scale_dtype: torch.dtype = torch.float32, bias_dtype: torch.dtype = torch.float16,
                         x_dtype: torch.dtype = torch.float16) -> None:
    """``G`` independent decode GEMVs in one launch: unit ``u`` multiplies the fp16 row at ``x_tab[u]`` with the
    decode-tiled weights at ``w_tiled_tab[u]`` into the fp16 row at ``y_tab[u]``, exactly as
    :func:`ternary_linear_tiled_forward` would on that row (same bits).  The tables are int64 device tensors of
    ``G`` device addresses (:func:`pointer_table`); nothing is allocated or returned.
    ``x_dtype=torch.bfloat16``: bf16 rows and outputs; each row is scaled by its own largest exponent and summed
    exactly on the int8 matrix cores."""
    G = x_tab.numel()
    tabs = (x_tab, w_tiled_tab, scale_tab, y_tab) + (() if bias_tab is None else (bias_tab,))
    for t in tabs:
        _check(t.dtype == torch.int64 and t.dim() == 1 and t.numel() == G and t.is_contiguous(),
               "pointer tables must be contiguous int64 tensors of one length")
    _check(_all_cuda(*tabs), "All tensors must be CUDA")
    _check(scale_dtype in _DT and bias_dtype in _DT, "scale / bias dtype must be float32, float16 or bfloat16")
    _check(x_dtype in (torch.float16, torch.bfloat16), "x_dtype must be float16 or bfloat16")
    with _on(x_tab):
        _status(_L.bt_ternary_gemv_grouped(
            x_tab.data_ptr(), _DT[x_dtype], w_tiled_tab.data_ptr(), scale_tab.data_ptr(), _DT[scale_dtype],
            out_features if scale_len < 0 else scale_len, _ptr(bias_tab), _DT[bias_dtype], y_tab.data_ptr(), G,
            out_features, in_features, _stream(x_tab)))


def ternary_gemm_int8_grouped(q_tab: Tensor, sx_tab: Tensor, w_tiled_tab: Tensor, scale_tab: Tensor,
                              bias_tab: Optional[Tensor], y_tab: Tensor, rows: int, in_features: int, out_features: int,
                              scale_len: int = -1, scale_dtype: torch.dtype = torch.float32,
                              bias_dtype: torch.dtype = torch.float32, out_dtype: torch.dtype = torch.bfloat16,
                              q_operand_order: bool = False, acc_tab: Optional[Tensor] = None) -> None:
    """``G`` independent int8 units of ``rows`` (at most 16) activation rows each in one launch: unit ``u`` multiplies
    the int8 rows at ``q_tab[u]`` (row scales at ``sx_tab[u]``) with the decode-tiled weights at ``w_tiled_tab[u]``
    into ``y_tab[u]`` ``[rows, N]``, exactly as :func:`ternary_gemm_int8_tiled` would (same accumulators, same bits).
    The tables are int64 device tensors of ``G`` device addresses (:func:`pointer_table`); ``acc_tab`` optionally
    receives the int32 accumulators; nothing is allocated or returned."""
    G = q_tab.numel()
    tabs = (q_tab, sx_tab, w_tiled_tab, scale_tab, y_tab) + tuple(t for t in (bias_tab, acc_tab) if t is not None)
    for t in tabs:
        _check(t.dtype == torch.int64 and t.dim() == 1 and t.numel() == G and t.is_contiguous(),
               "pointer tables must be contiguous int64 tensors of one length")
    _check(_all_cuda(*tabs), "All tensors must be CUDA")
    _check(scale_dtype in _DT and bias_dtype in _DT and out_dtype in _DT,
           "scale / bias / output dtype must be float32, float16 or bfloat16")
    with _on(q_tab):
        _status(_L.bt_ternary_gemm_i8_grouped(
            q_tab.data_ptr(), 1 if q_operand_order else 0, sx_tab.data_ptr(), w_tiled_tab.data_ptr(), scale_tab.data_ptr(),
            _DT[scale_dtype], out_features if scale_len < 0 else scale_len, _ptr(bias_tab), _DT[bias_dtype],
            y_tab.data_ptr(), _DT[out_dtype], _ptr(acc_tab), G, rows, out_features, in_features, _stream(q_tab)))


def retile_fields(W_tiled: Tensor, in_features: int, out_features: int) -> Tensor:
    """The prefill-only field layout of a decode-tiled copy (same size; natural or pair-ordered tiles are kept in
    their order): what :func:`ternary_gemm_int8_fields` reads."""
    _tiled_checks(W_tiled, out_features, in_features)
    _check(W_tiled.is_cuda, "All tensors must be CUDA")
    with _on(W_tiled):
        out = torch.empty_like(W_tiled)
        _status(_L.bt_retile_fields(W_tiled.data_ptr(), out_features, in_features, out.data_ptr(), _stream(W_tiled)))
    return out


def ternary_gemm_int8_fields(Q: Tensor, s_x: Tensor, q_rowsum: Tensor, W_fields: Tensor, scale: Tensor,
                             bias: Optional[Tensor] = None, in_features: int = -1, out_features: int = -1,
                             out_dtype: torch.dtype = torch.float32, return_acc: bool = False,
                             residual: Optional[Tensor] = None, q_operand_order: bool = False,
                             natural_from_pairs: bool = False):
    """:func:`ternary_gemm_int8_tiled` on the field layout (:func:`retile_fields`) with the rows' sums of ``Q``
    (``act_quant_int8(..., return_rowsum=True)``): the same results bit for bit through a cheaper weight decode.
    Always the tiled matrix-core GEMM (prefill batches); ``in_features`` a multiple of 128."""
    _check(Q.dim() == 2 and Q.dtype == torch.int8 and Q.numel() > 0, "Q must be 2D int8")
    K, N = Q.shape[-1], out_features
    _check(K == in_features, "input K doesn't match in_features")
    _tiled_checks(W_fields, N, K)
    _check(scale.dim() == 1 and scale.shape[0] in (N, 1), "scale size doesn't match N")
    _check(bias is None or (bias.dim() == 1 and bias.shape[0] == N), "bias shape mismatch")
    _check(s_x.dtype == torch.float32 and s_x.numel() == Q.shape[0], "s_x must be fp32 [B]")
    _check(q_rowsum.dtype == torch.int32 and q_rowsum.numel() == Q.shape[0], "q_rowsum must be int32 [B]")
    _check(_all_cuda(Q, s_x, q_rowsum, W_fields, scale, bias), "All tensors must be CUDA")
    _check(out_dtype in _DT, "out_dtype must be float32, float16 or bfloat16")
    q = Q.contiguous()
    s_x = s_x.contiguous()
    q_rowsum = q_rowsum.contiguous()
    scale = _prep_vec(scale, s_x)
    bias = None if bias is None else _prep_vec(bias, s_x)
    B = q.shape[0]
    y = torch.empty((B, N), dtype=out_dtype, device=q.device)
    acc = torch.empty((B, N), dtype=torch.int32, device=q.device) if return_acc else None
    res = None if residual is None else _residual_2d(residual, y, (B,), N)
    with _on(q):
        _status(_L.bt_ternary_gemm_i8_fields(
            q.data_ptr(), 1 if q_operand_order else 0, s_x.data_ptr(), q_rowsum.data_ptr(), W_fields.data_ptr(),
            1 if natural_from_pairs else 0, scale.data_ptr(), _dt(scale, "scale"), scale.numel(), _ptr(bias),
            0 if bias is None else _dt(bias, "bias"), _ptr(res), y.data_ptr(), _DT[out_dtype], _ptr(acc), B, N, K,
            _stream(q)))
    return (y, acc) if return_acc else y


def ternary_gemm_int8_tiled(Q: Tensor, s_x: Tensor, W_tiled: Tensor, scale: Tensor, bias: Optional[Tensor] = None,
                            in_features: int = -1, out_features: int = -1,
                            out_dtype: torch.dtype = torch.float32, return_acc: bool = False,
                            residual: Optional[Tensor] = None, q_operand_order: bool = False):
    """:func:`ternary_gemm_int8` on the decode-tiled copy of the weights (same results bit for bit)."""
    if not return_acc:
        y = _N.gemm_i8_tiled(Q, s_x, W_tiled, scale, bias, in_features, out_features, out_dtype, residual, q_operand_order)
        if y is not None:
            return y
    _check(Q.dim() == 2 and Q.dtype == torch.int8 and Q.numel() > 0, "Q must be 2D int8")
    K, N = Q.shape[-1], out_features
    _check(K == in_features, "input K doesn't match in_features")
    _tiled_checks(W_tiled, N, K)
    _check(scale.dim() == 1 and scale.shape[0] in (N, 1), "scale size doesn't match N")
    _check(bias is None or (bias.dim() == 1 and bias.shape[0] == N), "bias shape mismatch")
    _check(s_x.dtype == torch.float32 and s_x.numel() == Q.shape[0], "s_x must be fp32 [B]")
    _check(_all_cuda(Q, s_x, W_tiled, scale, bias), "All tensors must be CUDA")
    _check(out_dtype in _DT, "out_dtype must be float32, float16 or bfloat16")
    q = Q.contiguous()
    s_x = s_x.contiguous()
    scale = _prep_vec(scale, s_x)
    bias = None if bias is None else _prep_vec(bias, s_x)
    B = q.shape[0]
    y = torch.empty((B, N), dtype=out_dtype, device=q.device)
    acc = torch.empty((B, N), dtype=torch.int32, device=q.device) if return_acc else None
    res = None if residual is None else _residual_2d(residual, y, (B,), N)
    with _on(q):
        _status(_L.bt_ternary_gemm_i8_tiled(
            q.data_ptr(), 1 if q_operand_order else 0, s_x.data_ptr(), W_tiled.data_ptr(), scale.data_ptr(),
            _dt(scale, "scale"), scale.numel(), _ptr(bias), 0 if bias is None else _dt(bias, "bias"), _ptr(res),
            y.data_ptr(), _DT[out_dtype], _ptr(acc), B, N, K, _stream(q)))
    return (y, acc) if return_acc else y


def swiglu_int8_tiled_pays(rows: int, in_features: int, out_features: int) -> bool:
    """Whether :func:`ternary_swiglu_int8_tiled` is the faster way for this size."""
    return bool(_L.bt_swiglu_i8_tiled_pays(rows, out_features, in_features))


def ternary_swiglu_int8_tiled(Q: Tensor, s_x: Tensor, W_tiled: Tensor, scale: Tensor, bias: Optional[Tensor],
                              in_features: int, out_features: int, out_dtype: torch.dtype) -> Tensor:
    """``silu(gate) * up`` ``[B, N / 2]`` of the projections ``[gate | up]`` that :func:`ternary_gemm_int8_tiled` makes of the
    same arguments, bit for bit what :func:`swiglu` makes of its output: the product is formed in the GEMM's output stage.
    ``Q`` in operand order, a copy in natural order, ``N % 32 == 0`` and a 16-bit ``out_dtype``."""
    h = _N.swiglu_i8_tiled(Q, s_x, W_tiled, scale, bias, in_features, out_features, out_dtype)
    if h is not None:
        return h
    _check(Q.dim() == 2 and Q.dtype == torch.int8 and Q.numel() > 0, "Q must be 2D int8")
    K, N = Q.shape[-1], out_features
    _check(K == in_features, "input K doesn't match in_features")
    _tiled_checks(W_tiled, N, K)
    _check(scale.dim() == 1 and scale.shape[0] in (N, 1), "scale size doesn't match N")
    _check(bias is None or (bias.dim() == 1 and bias.shape[0] == N), "bias shape mismatch")
    _check(s_x.dtype == torch.float32 and s_x.numel() == Q.shape[0], "s_x must be fp32 [B]")
    _check(_all_cuda(Q, s_x, W_tiled, scale, bias), "All tensors must be CUDA")
    _check(out_dtype in (torch.float16, torch.bfloat16) and N % 32 == 0, "out_dtype must be float16 or bfloat16, and N a multiple of 32")
    q = Q.contiguous()
    s_x = s_x.contiguous()
    scale = _prep_vec(scale, s_x)
    bias = None if bias is None else _prep_vec(bias, s_x)
    B = q.shape[0]
    h = torch.empty((B, N // 2), dtype=out_dtype, device=q.device)
    with _on(q):
        _status(_L.bt_ternary_swiglu_i8_tiled(
            q.data_ptr(), s_x.data_ptr(), W_tiled.data_ptr(), scale.data_ptr(), _dt(scale, "scale"), scale.numel(), _ptr(bias),
            0 if bias is None else _dt(bias, "bias"), h.data_ptr(), _DT[out_dtype], B, N, K, _stream(q)))
    return h


def ternary_linear_tensor_core_forward(X: Tensor, W_T: Tensor, scale: Tensor,
                                       bias: Optional[Tensor] = None, in_features: int = -1,
                                       version: int = 1) -> Tensor:
    """Matrix-core forward; ``X`` must be 2-D as in the reference.

    version 1: float compute (the reference's validation kernel,
    ``ternary_gemm_tensor_core.cu:120-271``) -- served by the fp32-accumulate
    packed kernel.  version 2: per-row int8 activations, int8 MFMA, int32
    accumulators (``:349-657`` with the whole-row activation scale).
    """
    if version == 2:
        y = _N.tensor_core_forward(X, W_T, scale, bias, X.shape[-1] if in_features < 0 and X.dim() > 0 else in_features)
        if y is not None:
            return y
    _check(X.dim() == 2, "X must be 2D")
    _check(version in (1, 2), "version must be 1 (V1 float) or 2 (V2 mma.sync)")
    if in_features < 0:
        in_features = X.shape[-1]
    K, N = _packed_checks(X, W_T, scale, bias, in_features)
    if version == 1:
        return ternary_linear_packed_forward(X, W_T, scale, bias, in_features)
    _check(X.dtype in _DT, "X must be float32, float16 or bfloat16 for version 2")
    x2 = X.contiguous()
    W_T = W_T.contiguous()
    scale = _prep_vec(scale, x2)
    bias = None if bias is None else _prep_vec(bias, x2)
    B = x2.shape[0]
    y = torch.empty((B, N), dtype=X.dtype, device=X.device)
    with _on(X):
        ws_bytes = _L.bt_tensor_core_workspace_bytes(B, N, K)
        ws = _workspace(ws_bytes, X.device)
        _status(_L.bt_ternary_linear_tensor_core_forward(
            x2.data_ptr(), _dt(x2, "X"), W_T.data_ptr(), scale.data_ptr(), _dt(scale, "scale"),
            scale.numel(), _ptr(bias), 0 if bias is None else _dt(bias, "bias"), y.data_ptr(),
            B, N, K, _ptr(ws), 0 if ws is None else ws.numel(), _stream(X)))
    return y


# ---- additive entry points (no counterpart in the reference module) ----------------------


def ternary_quantize_pack(weight: Tensor, threshold_factor: float = 0.05, per_channel: bool = True,
                          want_packed: bool = True, want_tern: bool = False, as_half: bool = False
                          ) -> Tuple[Optional[Tensor], Tensor, Optional[Tensor]]:
    """Fused quantize + pack of master weights ``[N, K]`` on the GPU.

    Returns ``(packed_T uint8 [ceil(K/4), N] | None, scale, w_tern int8 [N, K] | None)``;
    ``scale`` has the weight dtype and shape ``(N,)`` (per channel) or ``()`` (per tensor),
    exactly what ``quant.ternary_quantize`` returns.  ``as_half=True`` (fp32 weights): the results for ``weight.half()``,
    rounded as the weights are read.
    """
    if want_packed and not want_tern:
        out = _N.quantize_pack(weight, threshold_factor, per_channel, as_half)
        if out is not None:
            return out
    _check(weight.dim() == 2, "weight must be 2D [N, K]")
    _check(not as_half or weight.dtype == torch.float32, "as_half takes fp32 weights")
    _check(weight.is_cuda, "All tensors must be CUDA")
    w = weight.detach().contiguous()
    N, K = w.shape
    _check(N > 0 and K > 0, "weight is empty")
    wdt = _F32_AS_F16 if as_half else _dt(w, "weight")
    dev = w.device
    packed = torch.empty(((K + 3) // 4, N), dtype=torch.uint8, device=dev) if want_packed else None
    tern = torch.empty((N, K), dtype=torch.int8, device=dev) if want_tern else None
    scale = torch.empty((N if per_channel else 1,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        _status(_L.bt_quantize_pack(w.data_ptr(), wdt, N, K, float(threshold_factor),
                                    int(bool(per_channel)), _ptr(packed), scale.data_ptr(),
                                    _ptr(tern), _stream(w)))
    scale = scale.to(torch.float16 if as_half else weight.dtype)
    if not per_channel:
        scale = scale.squeeze(0)
    return packed, scale, tern


def act_quant_int8(X: Tensor, operand_order: bool = False, return_rowsum: bool = False):
    """Per-row int8 activation quantization: ``(Q int8 [B,K], s_x fp32 [B])``.

    ``operand_order=True`` (K % 16 == 0) writes every 16-byte group of ``Q`` in the order the
    int8 GEMMs feed the matrix cores; such a ``Q`` must go to :func:`ternary_gemm_int8` with
    ``q_operand_order=True``.  ``return_rowsum=True`` adds the rows' sums of ``Q`` (int32 ``[B]``), which
    :func:`ternary_gemm_int8_fields` needs."""
    if not return_rowsum:
        out = _N.act_quant_int8(X, operand_order)
        if out is not None:
            return out
    _check(X.dim() == 2 and X.numel() > 0, "X must be 2D and non-empty")
    _check(X.is_cuda, "All tensors must be CUDA")
    x = X.contiguous()
    B, K = x.shape
    q = torch.empty((B, K), dtype=torch.int8, device=x.device)
    s = torch.empty((B,), dtype=torch.float32, device=x.device)
    with _on(x):
        if return_rowsum:
            rs = torch.empty((B,), dtype=torch.int32, device=x.device)
            _status(_L.bt_act_quant_i8_rowsum(x.data_ptr(), _dt(x, "X"), B, K, q.data_ptr(), s.data_ptr(), rs.data_ptr(),
                                              1 if operand_order else 0, _stream(x)))
            return q, s, rs
        _status(_L.bt_act_quant_i8_layout(x.data_ptr(), _dt(x, "X"), B, K, q.data_ptr(), s.data_ptr(),
                                          1 if operand_order else 0, _stream(x)))
    return q, s


def ternary_gemm_int8(Q: Tensor, s_x: Tensor, W_T: Tensor, scale: Tensor,
                      bias: Optional[Tensor] = None, in_features: int = -1,
                      out_dtype: torch.dtype = torch.float32, return_acc: bool = False,
                      residual: Optional[Tensor] = None, q_operand_order: bool = False):
    """int8 activations x packed ternary weights; optionally also the int32 accumulators.
    ``residual`` ``[B, N]`` in ``out_dtype`` is added in the epilogue (``linear + residual``);
    ``q_operand_order`` says that ``Q`` was written with ``operand_order=True``."""
    _check(Q.dim() == 2 and Q.dtype == torch.int8, "Q must be 2D int8")
    if in_features < 0:
        in_features = Q.shape[-1]
    K, N = _packed_checks(Q, W_T, scale, bias, in_features)
    _check(s_x.dtype == torch.float32 and s_x.numel() == Q.shape[0], "s_x must be fp32 [B]")
    _check(_all_cuda(s_x), "All tensors must be CUDA")
    _check(out_dtype in _DT, "out_dtype must be float32, float16 or bfloat16")
    q = Q.contiguous()
    W_T = W_T.contiguous()
    s_x = s_x.contiguous()
    scale = _prep_vec(scale, s_x)
    bias = None if bias is None else _prep_vec(bias, s_x)
    B = q.shape[0]
    y = torch.empty((B, N), dtype=out_dtype, device=q.device)
    acc = torch.empty((B, N), dtype=torch.int32, device=q.device) if return_acc else None
    with _on(q):
        ws_bytes = _L.bt_gemm_i8_workspace_bytes(B, N, K)
        ws = _workspace(ws_bytes, q.device)
        if residual is None and not q_operand_order:
            _status(_L.bt_ternary_gemm_i8(
                q.data_ptr(), s_x.data_ptr(), W_T.data_ptr(), scale.data_ptr(), _dt(scale, "scale"),
                scale.numel(), _ptr(bias), 0 if bias is None else _dt(bias, "bias"), y.data_ptr(),
                _DT[out_dtype], _ptr(acc), B, N, K, _ptr(ws), 0 if ws is None else ws.numel(), _stream(q)))
        else:
            res = None if residual is None else _residual_2d(residual, y, (B,), N)
            _status(_L.bt_ternary_gemm_i8_res(
                q.data_ptr(), 1 if q_operand_order else 0, s_x.data_ptr(), W_T.data_ptr(), scale.data_ptr(),
                _dt(scale, "scale"), scale.numel(), _ptr(bias), 0 if bias is None else _dt(bias, "bias"), _ptr(res),
                y.data_ptr(), _DT[out_dtype], _ptr(acc), B, N, K, _stream(q)))
    return (y, acc) if return_acc else y


def _row_op_outputs(x2: Tensor, store: bool, quantize: bool):
    _check(store or quantize, "nothing to compute: store and quantize are both False")
    B, K = x2.shape
    h = torch.empty((B, K), dtype=x2.dtype, device=x2.device) if store else None
    q = torch.empty((B, K), dtype=torch.int8, device=x2.device) if quantize else None
    s = torch.empty((B,), dtype=torch.float32, device=x2.device) if quantize else None
    return h, q, s


def _row_op_result(h, q, s, lead_shape, K):
    if h is not None:
        h = h.reshape(*lead_shape, K)
    if q is None:
        return h
    return (q, s) if h is None else (h, q, s)


def _rows_2d(t: Tensor, K: int) -> Tensor:
    """A 2-D view with unit inner stride (row stride kept: slices of a wider matrix stay in place)."""
    if t.stride(-1) == 1 and t.dim() >= 2 and t.stride(-2) >= K:
        lead_ok = all(t.stride(i) == t.stride(i + 1) * t.shape[i + 1] for i in range(t.dim() - 2))
        if lead_ok:  # the leading dimensions collapse into one row index with a single stride
            rows = t.numel() // K
            return t if t.dim() == 2 else t.as_strided((rows, K), (t.stride(-2), 1), t.storage_offset())
    return t.contiguous().reshape(-1, K)


def swiglu(gate: Tensor, up: Tensor, store: bool = True, quantize: bool = False, operand_order: bool = False,
           return_rowsum: bool = False):
    """``silu(gate) * up`` in one pass, rounded as the two separate torch ops round it.

    Returns the product (``store``), or with ``quantize`` its per-row int8 form ``(Q, s_x)`` for
    :func:`ternary_gemm_int8` -- ``(h, Q, s_x)`` when both are asked for.  ``gate`` and ``up`` may
    be column slices of one wider matrix (the output of a fused gate/up projection).  ``return_rowsum`` (with
    ``quantize``) appends the rows' sums of ``Q`` (int32), which :func:`ternary_gemm_int8_fields` needs."""
    if quantize and not store and not return_rowsum:
        out = _N.swiglu_int8(gate, up, operand_order)
        if out is not None:
            return out
    _check(gate.shape == up.shape and gate.dtype == up.dtype, "gate and up must match in shape and dtype")
    _check(gate.dim() >= 1 and gate.numel() > 0, "gate is empty")
    _check(gate.dtype in _DT, "gate must be float32, float16 or bfloat16")
    _check(_all_cuda(gate, up), "All tensors must be CUDA")
    K = gate.shape[-1]
    g2, u2 = _rows_2d(gate, K), _rows_2d(up, K)
    h, q, s = _row_op_outputs(g2, store, quantize)
    rs = None
    with _on(gate):
        if return_rowsum:
            _check(q is not None, "return_rowsum needs quantize=True")
            rs = torch.empty((g2.shape[0],), dtype=torch.int32, device=gate.device)
            _status(_L.bt_swiglu_rowsum(g2.data_ptr(), g2.stride(0), u2.data_ptr(), u2.stride(0), _dt(g2, "gate"),
                                        g2.shape[0], K, _ptr(h), _ptr(q), _ptr(s), rs.data_ptr(),
                                        1 if operand_order else 0, _stream(gate)))
        else:
            _status(_L.bt_swiglu(g2.data_ptr(), g2.stride(0), u2.data_ptr(), u2.stride(0), _dt(g2, "gate"),
                                 g2.shape[0], K, _ptr(h), _ptr(q), _ptr(s), 1 if operand_order else 0, _stream(gate)))
    if q is not None and gate.dim() != 2:
        q = q.reshape(*gate.shape[:-1], K)
        s = s.reshape(gate.shape[:-1])
    out = _row_op_result(h, q, s, gate.shape[:-1], K)
    return out if rs is None else (*out, rs.reshape(gate.shape[:-1]))


def rmsnorm(x: Tensor, weight: Optional[Tensor] = None, eps: float = 1e-6, store: bool = True,
            quantize: bool = False, operand_order: bool = False, return_rowsum: bool = False):
    """RMSNorm over the last dimension, ``(x * rsqrt(mean(x^2) + eps)) * weight``; with
    ``quantize`` also (or only, ``store=False``) the per-row int8 form of the result, and with ``return_rowsum``
    the rows' sums of that form appended (int32)."""
    if quantize and not store and not return_rowsum:
        out = _N.rmsnorm_int8(x, weight, eps, operand_order)
        if out is not None:
            return out
    _check(x.dim() >= 1 and x.numel() > 0, "x is empty")
    _check(x.dtype in _DT, "x must be float32, float16 or bfloat16")
    K = x.shape[-1]
    if weight is not None:
        _check(weight.dim() == 1 and weight.shape[0] == K, "weight must be 1D [K]")
        weight = weight.to(x.dtype).contiguous()
    _check(_all_cuda(x, weight), "All tensors must be CUDA")
    x2 = _rows_2d(x, K)
    h, q, s = _row_op_outputs(x2, store, quantize)
    rs = None
    with _on(x):
        if return_rowsum:
            _check(q is not None, "return_rowsum needs quantize=True")
            rs = torch.empty((x2.shape[0],), dtype=torch.int32, device=x.device)
            _status(_L.bt_rmsnorm_rowsum(x2.data_ptr(), x2.stride(0), _ptr(weight), float(eps), _dt(x2, "x"),
                                         x2.shape[0], K, _ptr(h), _ptr(q), _ptr(s), rs.data_ptr(),
                                         1 if operand_order else 0, _stream(x)))
        else:
            _status(_L.bt_rmsnorm(x2.data_ptr(), x2.stride(0), _ptr(weight), float(eps), _dt(x2, "x"),
                                  x2.shape[0], K, _ptr(h), _ptr(q), _ptr(s), 1 if operand_order else 0, _stream(x)))
    if q is not None and x.dim() != 2:
        q = q.reshape(*x.shape[:-1], K)
        s = s.reshape(x.shape[:-1])
    out = _row_op_result(h, q, s, x.shape[:-1], K)
    return out if rs is None else (*out, rs.reshape(x.shape[:-1]))


def _add_rmsnorm_checks(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor]) -> int:
    _check(x.dim() >= 1 and x.numel() > 0, "x is empty")
    _check(x.dtype in _DT, "x must be float32, float16 or bfloat16")
    K = x.shape[-1]
    if residual is not None:
        _check(residual.shape == x.shape, "residual shape doesn't match x")
        _check(residual.dtype in (x.dtype, torch.float32), "residual must have x's dtype or be float32")
        _check(residual.device == x.device, "All tensors must be CUDA")
    if weight is not None:
        _check(weight.dim() == 1 and weight.shape[0] == K, "weight must be 1D [K]")
        _check(weight.dtype in (x.dtype, torch.float32), "weight must have x's dtype or be float32")
        _check(weight.device == x.device, "All tensors must be CUDA")
    _check(x.is_cuda, "All tensors must be CUDA")
    return K


def add_rmsnorm(x: Tensor, residual: Optional[Tensor], weight: Optional[Tensor] = None, eps: float = 1e-6, store: bool = True,
                quantize: bool = False, operand_order: bool = False, return_rowsum: bool = False, return_rstd: bool = False):
    """``s = x + residual`` and its RMSNorm in one pass: ``(s, y)``, with ``quantize`` ``(s, y, Q, s_x)`` or, ``store=False``,
    ``(s, Q, s_x)``; ``return_rowsum`` and ``return_rstd`` append the rows' sums of ``Q`` and their reciprocal root mean squares.
    ``s`` has the residual's dtype (``x``'s or fp32) and is ``x`` itself without a residual."""
    K = _add_rmsnorm_checks(x, residual, weight)
    _check(store or quantize, "nothing to compute: store and quantize are both False")
    _check(quantize or not return_rowsum, "return_rowsum needs quantize=True")
    x2 = _rows_2d(x, K)
    r2 = None if residual is None else _rows_2d(residual, K)
    w = None if weight is None else weight.contiguous()
    B, dev, lead = x2.shape[0], x.device, x.shape[:-1]
    s = x if residual is None else torch.empty(x.shape, dtype=residual.dtype, device=dev)
    y = torch.empty(x.shape, dtype=x.dtype, device=dev) if store else None
    q = torch.empty(x.shape, dtype=torch.int8, device=dev) if quantize else None
    s_x = torch.empty(lead, dtype=torch.float32, device=dev) if quantize else None
    rs = torch.empty(lead, dtype=torch.int32, device=dev) if return_rowsum else None
    rstd = torch.empty((B,), dtype=torch.float32, device=dev) if return_rstd else None
    with _on(x):
        _status(_L.bt_add_rmsnorm(
            x2.data_ptr(), x2.stride(0), _DT[x.dtype], _ptr(r2), 0 if r2 is None else r2.stride(0), 0 if r2 is None else _DT[r2.dtype],
            _ptr(w), 0 if w is None else _DT[w.dtype], float(eps), B, K, None if residual is None else s.data_ptr(), _ptr(y), _ptr(rstd),
            _ptr(q), _ptr(s_x), _ptr(rs), 1 if operand_order else 0, _stream(x)))
    return tuple(t for t in (s, y, q, s_x, rs, rstd) if t is not None)


def add_rmsnorm_backward(s: Tensor, rstd: Tensor, weight: Optional[Tensor], d_sum: Optional[Tensor], d_norm: Tensor,
                         want_x: bool = True, want_residual: bool = True, want_weight: bool = True
                         ) -> Tuple[Optional[Tensor], Optional[Tensor], Optional[Tensor]]:
    """Gradients ``(x, residual, weight)`` of :func:`add_rmsnorm`'s ``s`` and ``y`` from the stored ``s`` and ``rstd``; those of
    ``x`` and ``residual`` are one tensor where their dtypes are the same."""
    K = _add_rmsnorm_checks(d_norm, s, weight)
    _check(d_sum is None or (d_sum.shape == s.shape and d_sum.dtype == s.dtype and d_sum.device == s.device),
           "the sum's gradient must match the sum")
    B = s.numel() // K
    _check(rstd.dtype == torch.float32 and rstd.numel() == B and rstd.device == s.device, "rstd must be fp32 [B]")
    _check(not want_weight or weight is not None, "no weight to differentiate")
    _check(want_x or want_residual or want_weight, "no gradient requested")
    s, rstd, d_norm = s.contiguous(), rstd.contiguous(), d_norm.contiguous()
    d_sum = None if d_sum is None else d_sum.contiguous()
    weight = None if weight is None else weight.contiguous()
    dev, one = s.device, s.dtype == d_norm.dtype
    dr = torch.empty(s.shape, dtype=s.dtype, device=dev) if want_residual or (one and want_x) else None
    dx = torch.empty(s.shape, dtype=d_norm.dtype, device=dev) if want_x and not one else None
    dw = torch.empty((K,), dtype=weight.dtype, device=dev) if want_weight else None
    with _on(s):
        ws = _workspace(_L.bt_add_rmsnorm_backward_workspace_bytes(B, K), dev) if want_weight else None
        _status(_L.bt_add_rmsnorm_backward(
            s.data_ptr(), _DT[s.dtype], rstd.data_ptr(), _ptr(weight), 0 if weight is None else _DT[weight.dtype], d_norm.data_ptr(),
            _DT[d_norm.dtype], _ptr(d_sum), B, K, _ptr(dx), _ptr(dr), _ptr(dw), _ptr(ws), 0 if ws is None else ws.numel(), _stream(s)))
    return (dr if one and want_x else dx), (dr if want_residual else None), dw


def _gated_operands(gate: Tensor, up: Tensor, gate_bias: Optional[Tensor], up_bias: Optional[Tensor], as_half: bool):
    """The checked masters and biases as the kernels read them: ``(masters, their tag, biases, their tag)``."""
    _check(gate.dim() == 2 and gate.shape == up.shape and gate.dtype == up.dtype, "gate and up weights must match, 2D [F, K]")
    _check(gate.numel() > 0, "weight is empty")
    _check(not as_half or gate.dtype == torch.float32, "as_half takes fp32 weights")
    biases = [None if b is None else b.detach() for b in (gate_bias, up_bias)]
    given = [b for b in biases if b is not None]
    for b in given:
        _check(b.dim() == 1 and b.shape[0] == gate.shape[0], "bias shape mismatch")
    _check(_all_cuda(gate, up, *biases), "All tensors must be CUDA")
    b_dtype = given[0].dtype if given and given[0].dtype in _DT and all(b.dtype == given[0].dtype for b in given) else torch.float32
    return ([t.detach().contiguous() for t in (gate, up)], _F32_AS_F16 if as_half else _dt(gate, "weight"),
            [None if b is None else b.to(b_dtype).contiguous() for b in biases], _DT[b_dtype])


def gated_masters_forward(X: Tensor, gate: Tensor, up: Tensor, gate_bias: Optional[Tensor] = None, up_bias: Optional[Tensor] = None,
                          threshold_factor: float = 0.05, as_half: bool = False) -> Tensor:
    """``silu(gate) * up`` ``[1, F]`` of one row ``[1, K]`` (:func:`gated_masters_serves`) straight from the masters ``[F, K]``, each
    quantized per feature as it is read."""
    _check(X.dim() == 2 and X.shape[0] == 1 and X.numel() > 0 and X.dtype in _DT, "X must be one row, float32, float16 or bfloat16")
    masters, wdt, biases, bdt = _gated_operands(gate, up, gate_bias, up_bias, as_half)
    F, K = gate.shape
    _check(K == X.shape[1], "input K doesn't match weight K")
    _check(X.device == gate.device, "All tensors must be CUDA")
    X = X.contiguous()
    h = torch.empty((1, F), dtype=X.dtype, device=X.device)
    with _on(X):
        _status(_L.bt_gated_masters_forward(X.data_ptr(), _DT[X.dtype], masters[0].data_ptr(), masters[1].data_ptr(), wdt, float(threshold_factor),
                                            _ptr(biases[0]), _ptr(biases[1]), bdt, h.data_ptr(), F, K, _stream(X)))
    return h


def gated_masters_serves(rows: int, masters: Tensor, per_channel: bool = True, as_half: bool = False) -> bool:
    """Whether :func:`gated_masters_forward` takes a call of so many rows on such masters."""
    wdt = _F32_AS_F16 if as_half else _dt(masters, "weight")
    return bool(_L.bt_gated_masters_serves(rows, masters.shape[1], wdt, int(bool(per_channel))))


def gated_weights(gate: Tensor, up: Tensor, gate_bias: Optional[Tensor] = None, up_bias: Optional[Tensor] = None,
                  threshold_factor: float = 0.05, per_channel: bool = True, as_half: bool = False, back: bool = False):
    """The operands of the gated pair, of two masters ``[F, K]`` quantized as :func:`ternary_quantize_pack` does: ``(W_pairs, W_back,
    scale, bias)`` as ``bt_gated_quantize`` makes them; ``back``: with the copy for the input's gradient (otherwise None)."""
    masters, wdt, biases, bdt = _gated_operands(gate, up, gate_bias, up_bias, as_half)
    (F, K), dev = gate.shape, gate.device
    Fp = (F + 15) // 16 * 16
    w = torch.empty((_L.bt_tiled_weights_bytes(2 * Fp, K),), dtype=torch.uint8, device=dev)
    w_back = torch.empty((_L.bt_tiled_weights_bytes(K, 2 * Fp),), dtype=torch.uint8, device=dev) if back else None
    scale = torch.empty((2 * Fp + 1,), dtype=torch.float32, device=dev)
    bias = torch.empty((2 * Fp,), dtype=torch.float32, device=dev) if any(b is not None for b in biases) else None
    with _on(gate):
        ws = _workspace(_L.bt_gated_quantize_workspace_bytes(F, K, int(bool(per_channel))), dev)
        _status(_L.bt_gated_quantize(masters[0].data_ptr(), masters[1].data_ptr(), wdt, F, K, float(threshold_factor), int(bool(per_channel)),
                                     _ptr(biases[0]), _ptr(biases[1]), bdt, w.data_ptr(), _ptr(w_back), scale.data_ptr(), _ptr(bias), _ptr(ws),
                                     0 if ws is None else ws.numel(), _stream(gate)))
    return w, w_back, scale, bias


def gated_split(scale: Tensor, out_features: int) -> Tensor:
    """The scales of :func:`gated_weights` taken apart for the gradient of fp16 rows, as ``bt_gated_split`` lays them out (fp32 and, at the end,
    fp16); ``scale``'s last entry becomes the power of two above all of them."""
    n = 2 * ((out_features + 15) // 16 * 16)
    _check(scale.is_cuda and scale.dtype == torch.float32 and scale.numel() == n + 1 and scale.is_contiguous(), "scale must be that of gated_weights")
    split = torch.empty((_L.bt_gated_split_bytes(out_features) // 4,), dtype=torch.float32, device=scale.device)
    with _on(scale):
        _status(_L.bt_gated_split(scale.data_ptr(), out_features, split.data_ptr(), _stream(scale)))
    return split


def gated_grad_input(G: Tensor, W_back: Tensor, split: Tensor, out_features: int, in_features: int) -> Tensor:
    """``[B, K]``: the gradient of fp16 rows, of :func:`gated_grad`'s ``G`` with ``split[:2 Fp + 1]`` in the place of the scales."""
    F, K, Fp = out_features, in_features, (out_features + 15) // 16 * 16
    _check(G.dim() == 2 and G.dtype == torch.float16 and G.shape[1] == 2 * Fp and G.numel() > 0, "G must be fp16, [B, 2 F] as gated_grad pads it")
    _check(W_back.dtype == torch.uint8 and W_back.dim() == 1 and W_back.is_contiguous() and W_back.numel() == _L.bt_tiled_weights_bytes(K, 2 * Fp),
           "W_back size doesn't match in_features x out_features")
    _check(split.dtype == torch.float32 and split.is_contiguous() and 4 * split.numel() == _L.bt_gated_split_bytes(F), "split must be that of gated_split")
    _check(_all_cuda(G, W_back, split), "All tensors must be CUDA")
    G = G.contiguous()
    out = torch.empty((G.shape[0], K), dtype=G.dtype, device=G.device)
    with _on(G):
        ws = _workspace(_L.bt_gated_grad_input_workspace_bytes(G.shape[0], F, K), G.device)
        _status(_L.bt_gated_grad_input(G.data_ptr(), W_back.data_ptr(), split.data_ptr(), out.data_ptr(), G.shape[0], F, K, _ptr(ws),
                                       0 if ws is None else ws.numel(), _stream(G)))
    return out


def ternary_gated_forward(X: Tensor, W_pairs: Tensor, scale: Tensor, bias: Optional[Tensor], out_features: int,
                          want_pre: bool = False) -> Tuple[Tensor, Optional[Tensor], Tensor]:
    """``silu(gate) * up`` ``[B, F]`` of 16-bit rows ``[B, K]`` on the operands of :func:`gated_weights`; with ``want_pre`` the two
    projections (int32 ``[B, 3 Fp / 2]``, 24 bits each) as :func:`gated_grad` reads them; and the rows as the kernels read them (a padded copy of ``X`` where
    K is no multiple of 8 or it is not 16-byte aligned)."""
    _check(X.dim() == 2 and X.numel() > 0 and X.dtype in (torch.float16, torch.bfloat16), "X must be 2D fp16 or bf16")
    B, K = X.shape
    F, Fp = out_features, (out_features + 15) // 16 * 16
    _check(W_pairs.dtype == torch.uint8 and W_pairs.dim() == 1 and W_pairs.is_contiguous()
           and W_pairs.numel() == _L.bt_tiled_weights_bytes(2 * Fp, K), "W_pairs size doesn't match out_features x in_features")
    _check(scale.dtype == torch.float32 and scale.numel() >= 2 * Fp and (bias is None or (bias.dtype == torch.float32 and bias.numel() >= 2 * Fp)),
           "scale and bias must be fp32 with an entry for each padded feature")
    _check(_all_cuda(X, W_pairs, scale, bias), "All tensors must be CUDA")
    X, scale, bias = X.contiguous(), scale.contiguous(), None if bias is None else bias.contiguous()
    rows = X if K % 8 == 0 and X.data_ptr() % 16 == 0 else torch.empty((B, (K + 7) // 8 * 8), dtype=X.dtype, device=X.device)
    h = torch.empty((B, F), dtype=X.dtype, device=X.device)
    pre = torch.empty((B, Fp // 2 * 3), dtype=torch.int32, device=X.device) if want_pre else None
    with _on(X):
        _status(_L.bt_ternary_gated_forward(X.data_ptr(), _DT[X.dtype], None if rows is X else rows.data_ptr(), W_pairs.data_ptr(),
                                            scale.data_ptr(), _ptr(bias), h.data_ptr(), _ptr(pre), B, F, K, _stream(X)))
    return h, pre, rows


def gated_grad(dH: Tensor, pre: Tensor, scale: Tensor, bias_dtype: Optional[torch.dtype] = None) -> Tuple[Tensor, Optional[Tensor]]:
    """Gradient of ``silu(gate) * up`` in both projections times their scales over ``scale``'s last entry, ``[B, 2 Fp]`` (``pre`` as :func:`ternary_gated_forward` kept
    it, or for fp32 rows ``[gate | up]`` ``[B, 2 Fp]``); with ``bias_dtype`` also its sums over the rows ``[2 F]``, without scales."""
    _check(dH.dim() == 2 and dH.numel() > 0 and dH.dtype in _DT, "dH must be 2D float32, float16 or bfloat16")
    B, F = dH.shape
    Fp = (F + 15) // 16 * 16
    kept = (torch.float32, (B, 2 * Fp)) if dH.dtype == torch.float32 else (torch.int32, (B, Fp // 2 * 3))
    _check((pre.dtype, pre.shape) == kept and pre.is_contiguous(), "the projections must be those that the forward kept")
    _check(scale.dtype == torch.float32 and scale.numel() == 2 * Fp + 1 and scale.is_contiguous(), "scale must be that of gated_weights")
    _check(_all_cuda(dH, pre, scale), "All tensors must be CUDA")
    dH = dH.contiguous()
    G = torch.empty((B, 2 * Fp), dtype=dH.dtype, device=dH.device)
    db = None if bias_dtype is None else torch.empty((2 * F,), dtype=bias_dtype, device=dH.device)
    with _on(dH):
        ws = None if db is None else _workspace(_L.bt_gated_grad_workspace_bytes(B, F), dH.device)
        _status(_L.bt_gated_grad(dH.data_ptr(), _DT[dH.dtype], pre.data_ptr(), scale.data_ptr(), G.data_ptr(), _ptr(db),
                                 0 if db is None else _DT[bias_dtype], B, F, _ptr(ws), 0 if ws is None else ws.numel(), _stream(dH)))
    return G, db


def _gated_grad_operands(G: Tensor, X: Tensor, scale: Tensor, F: int, K: int, out_dtype: torch.dtype):
    Fp, Kr = (F + 15) // 16 * 16, (K + 7) // 8 * 8
    _check(G.dim() == 2 and G.dtype in (torch.float16, torch.bfloat16) and X.dtype == G.dtype and G.shape[1] == 2 * Fp
           and X.shape == (G.shape[0], Kr), "G and X must be 16-bit, [B, 2 F] and [B, K] as the other calls pad them")
    _check(out_dtype in (G.dtype, torch.float32), "out_dtype must be G's or float32")
    _check(_all_cuda(G, X, scale), "All tensors must be CUDA")
    return G.contiguous(), X.contiguous(), torch.empty((2 * F, K), dtype=out_dtype, device=G.device), 2 * Fp, Kr


def gated_grad_weight(G: Tensor, X: Tensor, scale: Tensor, out_features: int, in_features: int, out_dtype: torch.dtype) -> Tensor:
    """``[2 F, K]``: the gradients of both 16-bit masters, ``G^T X`` times ``scale``'s last entry, of :func:`gated_grad`'s ``G`` and the rows
    that :func:`ternary_gated_forward` read; each sum is rounded to 16 bits before the factor and after it."""
    F, K = out_features, in_features
    G, X, out, n, Kr = _gated_grad_operands(G, X, scale, F, K, out_dtype)
    _check(scale.dtype == torch.float32 and scale.numel() == n + 1 and scale.is_contiguous(), "scale must be that of gated_weights")
    with _on(G):
        ws = _workspace(_L.bt_linear_grad_weight_16_workspace_bytes(G.shape[0], n, Kr), G.device)
        _status(_L.bt_gated_grad_weight(G.data_ptr(), X.data_ptr(), _DT[G.dtype], scale[n:].data_ptr(), out.data_ptr(), _DT[out_dtype],
                                        G.shape[0], F, K, _ptr(ws), 0 if ws is None else ws.numel(), _stream(G)))
    return out


def gated_grad_masters(G: Tensor, X: Tensor, scale: Tensor, out_features: int, in_features: int, out_dtype: torch.dtype) -> Tensor:
    """As :func:`gated_grad_weight`, with a scale for each padded feature (``[2 Fp]``) or one (``[1]``), and the scaled fp32 sums rounded once."""
    F, K = out_features, in_features
    G, X, out, n, Kr = _gated_grad_operands(G, X, scale, F, K, out_dtype)
    _check(scale.dtype == torch.float32 and scale.dim() == 1 and scale.numel() in (1, n) and scale.is_contiguous(),
           "scale must be fp32 with an entry for each padded feature, or one")
    with _on(G):
        ws = _workspace(_L.bt_linear_grad_weight_16_workspace_bytes(G.shape[0], n, Kr), G.device)
        _status(_L.bt_gated_grad_masters(G.data_ptr(), X.data_ptr(), _DT[G.dtype], scale.data_ptr(), scale.numel(), out.data_ptr(), _DT[out_dtype],
                                         G.shape[0], F, K, _ptr(ws), 0 if ws is None else ws.numel(), _stream(G)))
    return out


def unpack_dequant(W_T: Tensor, in_features: int, scale: Optional[Tensor] = None,
                   out_dtype: torch.dtype = torch.float32) -> Tensor:
    """Dense ``[N, K]`` weights from packed ``W_T``: ``decode * scale[:, None]``
    (``out_dtype`` float) or the plain ternary values (``out_dtype=torch.int8``)."""
    if scale is not None and out_dtype != torch.int8:
        out = _N.unpack_dequant(W_T, in_features, scale, out_dtype)
        if out is not None:
            return out
    _check(W_T.dim() == 2 and W_T.dtype == torch.uint8, "W_T must be 2D uint8")
    _check(W_T.shape[0] == (in_features + 3) // 4, "K_bytes doesn't match ceil(K/4)")
    _check(_all_cuda(W_T, scale), "All tensors must be CUDA")
    W_T = W_T.contiguous()
    N = W_T.shape[1]
    if out_dtype == torch.int8:
        odt, scale_f = _INT8_OUT, None
    else:
        _check(out_dtype in _DT, "out_dtype must be float32, float16, bfloat16 or int8")
        odt = _DT[out_dtype]
        scale_f = None if scale is None else scale.reshape(-1).to(torch.float32).contiguous()
        if scale_f is not None:
            _check(scale_f.numel() in (N, 1), "scale size doesn't match N")
    out = torch.empty((N, in_features), dtype=out_dtype, device=W_T.device)
    with _on(W_T):
        _status(_L.bt_unpack_dequant(W_T.data_ptr(), _ptr(scale_f),
                                     0 if scale_f is None else scale_f.numel(), out.data_ptr(), odt,
                                     N, in_features, _stream(W_T)))
    return out


def linear_grad_input(dY: Tensor, W_T: Tensor, scale: Tensor, in_features: int) -> Tensor:
    """Input gradient of an fp32 packed layer, ``(dY * scale) @ decode(W_T)`` ``[M, K]`` (``dY`` ``[M, N]`` fp32,
    ``scale`` fp32 ``[N]`` or one entry)."""
    out = _N.grad_input(dY, W_T, scale, in_features)
    if out is not None:
        return out
    _check(dY.dim() == 2 and dY.dtype == torch.float32 and dY.numel() > 0, "dY must be 2D fp32")
    _check(W_T.dim() == 2 and W_T.dtype == torch.uint8 and W_T.shape[0] == (in_features + 3) // 4
           and W_T.shape[1] == dY.shape[1], "W_T must be uint8 [ceil(K/4), N]")
    _check(scale.dtype == torch.float32 and scale.numel() in (dY.shape[1], 1), "scale must be fp32 [N] or one entry")
    _check(_all_cuda(dY, W_T, scale), "All tensors must be CUDA")
    dY, W_T, scale = dY.contiguous(), W_T.contiguous(), scale.contiguous()
    M, N = dY.shape
    out = torch.empty((M, in_features), dtype=torch.float32, device=dY.device)
    with _on(dY):
        _status(_L.bt_ternary_linear_grad_input(dY.data_ptr(), W_T.data_ptr(), scale.data_ptr(), scale.numel(),
                                                out.data_ptr(), M, N, in_features, _stream(dY)))
    return out


def linear_grad_weight(dY: Tensor, X: Tensor, scale: Tensor, want_bias: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """Weight gradient under the straight-through estimator, ``scale[:, None] * (dY.T @ X)`` ``[N, K]``, and with
    ``want_bias`` the bias gradient ``dY.sum(0)`` from the same pass (all fp32, N and K at least 4)."""
    out = _N.grad_weight(dY, X, scale, want_bias)
    if out is not None:
        return out
    _check(dY.dim() == 2 and X.dim() == 2 and dY.shape[0] == X.shape[0] and dY.numel() > 0 and X.numel() > 0,
           "dY [M, N] and X [M, K] must be 2D with the same rows")
    _check(dY.dtype == X.dtype == scale.dtype == torch.float32, "dY, X and scale must be fp32")
    _check(scale.numel() in (dY.shape[1], 1), "scale size doesn't match N")
    _check(_all_cuda(dY, X, scale), "All tensors must be CUDA")
    dY, X, scale = dY.contiguous(), X.contiguous(), scale.contiguous()
    (M, N), K = dY.shape, X.shape[1]
    dW = torch.empty((N, K), dtype=torch.float32, device=dY.device)
    dB = torch.empty((N,), dtype=torch.float32, device=dY.device) if want_bias else None
    with _on(dY):
        ws = _workspace(_L.bt_linear_grad_weight_workspace_bytes(M, N, K), dY.device)
        _status(_L.bt_linear_grad_weight(dY.data_ptr(), X.data_ptr(), scale.data_ptr(), scale.numel(), dW.data_ptr(), _ptr(dB),
                                         M, N, K, _ptr(ws), 0 if ws is None else ws.numel(), _stream(dY)))
    return dW, dB


def linear_grad_weight_16(dY: Tensor, X: Tensor, scale: Tensor, out_dtype: torch.dtype) -> Tensor:
    """Weight gradient of a 16-bit layer, ``scale[:, None] * (dY.T @ X)`` ``[N, K]`` in their dtype or fp32, with the roundings
    of the unfused operations (``dY`` ``[M, N]``, ``X`` ``[M, K]``, N and K multiples of 8)."""
    out = _N.grad_weight_16(dY, X, scale, out_dtype)
    if out is not None:
        return out
    _check(dY.dim() == 2 and X.dim() == 2 and dY.shape[0] == X.shape[0] and dY.numel() > 0 and X.numel() > 0,
           "dY [M, N] and X [M, K] must be 2D with the same rows")
    _check(dY.dtype == X.dtype and dY.dtype in (torch.float16, torch.bfloat16), "dY and X must be fp16 or bf16")
    _check(out_dtype in (dY.dtype, torch.float32), "the gradient is of the operands' dtype or fp32")
    _check(scale.dtype in _DT and scale.numel() in (dY.shape[1], 1), "scale must be fp32 or 16-bit, [N] or one entry")
    _check(_all_cuda(dY, X, scale), "All tensors must be CUDA")
    dY, X, scale = dY.contiguous(), X.contiguous(), scale.reshape(-1).contiguous()
    (M, N), K = dY.shape, X.shape[1]
    out = torch.empty((N, K), dtype=out_dtype, device=dY.device)
    with _on(dY):
        ws = _workspace(_L.bt_linear_grad_weight_16_workspace_bytes(M, N, K), dY.device)
        _status(_L.bt_linear_grad_weight_16(dY.data_ptr(), X.data_ptr(), _DT[dY.dtype], scale.data_ptr(), _DT[scale.dtype],
                                            scale.numel(), out.data_ptr(), _DT[out_dtype], M, N, K, _ptr(ws), 0 if ws is None else ws.numel(),
                                            _stream(dY)))
    return out


def scale_grad_weight(G: Tensor, scale: Tensor) -> Tensor:
    """``(G * scale[:, None].to(G.dtype)).float()`` in one pass (``G`` ``[N, K]`` fp16 or bf16, ``scale`` ``[N]`` or one entry)."""
    _check(G.dim() == 2 and G.dtype in (torch.float16, torch.bfloat16) and G.numel() > 0, "G must be 2D fp16 or bf16")
    _check(scale.numel() in (G.shape[0], 1), "scale size doesn't match N")
    _check(_all_cuda(G, scale), "All tensors must be CUDA")
    G, scale = G.contiguous(), scale.reshape(-1).to(torch.float32).contiguous()
    out = torch.empty(G.shape, dtype=torch.float32, device=G.device)
    with _on(G):
        _status(_L.bt_scale_grad_weight(G.data_ptr(), _DT[G.dtype], scale.data_ptr(), scale.numel(), out.data_ptr(),
                                        G.shape[0], G.shape[1], _stream(G)))
    return out


def _token_rows(x: Tensor) -> Tensor:
    """``(*, heads, D)`` as ``[tokens, heads, D]`` whose last dimension is contiguous: a view wherever one stride fits all tokens."""
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        x = x.contiguous()
    return x if x.dim() == 3 else x.flatten(0, -3) if x.dim() > 3 else x.unsqueeze(0)


def _rotary_checks(dim: int, inv_freq: Optional[Tensor], device) -> int:
    if inv_freq is None:
        return 0
    _check(inv_freq.dim() == 1 and inv_freq.dtype in (torch.float32, torch.float64), "inv_freq must be 1D, float32 or float64")
    _check(2 * inv_freq.shape[0] <= dim, f"inv_freq turns {2 * inv_freq.shape[0]} features, a head has {dim}")
    _check(inv_freq.device == device, "All tensors must be on one device")
    return 2 * inv_freq.shape[0]


def rotary_args(q: Tensor, k: Optional[Tensor], positions: Tensor, inv_freq: Tensor) -> None:
    _check(q.dim() >= 2, "q must be (*, heads, head_dim)")
    _check(q.is_floating_point(), "q must be a floating-point tensor")
    if k is not None:
        _check(k.dim() == q.dim() and k.shape[:-2] == q.shape[:-2] and k.shape[-1] == q.shape[-1], "k must be (*, kv_heads, head_dim) of q's tokens")
        _check(k.dtype == q.dtype and k.device == q.device, "k must match q's dtype and device")
    _check(positions.dtype in (torch.int32, torch.int64), "positions must be int32 or int64")
    _check(positions.device == q.device, "All tensors must be on one device")
    _rotary_checks(q.shape[-1], inv_freq, q.device)


def rotary(q: Tensor, k: Optional[Tensor], positions: Tensor, inv_freq: Tensor, interleaved: bool = False, amplitude: float = 1.0,
           backward: bool = False) -> Tuple[Tensor, Optional[Tensor]]:
    """``q`` and ``k`` ``(*, heads, D)`` turned by their positions (any shape that broadcasts to ``*``); ``backward``: by the opposite angles."""
    rotary_args(q, k, positions, inv_freq)
    _check(q.is_cuda, "All tensors must be CUDA")
    dt = _dt(q, "q")
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device), None if k is None else torch.empty(k.shape, dtype=k.dtype, device=k.device)
    if k is not None and k.numel() == 0:
        return rotary(q, None, positions, inv_freq, interleaved, amplitude, backward)[0], out[1]
    if q.numel() == 0:
        return out if k is None else (out[0], rotary(k, None, positions, inv_freq, interleaved, amplitude, backward)[0])
    lead = q.shape[:-2]
    pos = positions if positions.shape == lead else positions.expand(lead)
    pos, freq = pos.contiguous(), inv_freq.contiguous()
    q3, k3 = _token_rows(q), None if k is None else _token_rows(k)
    with _on(q):
        _status(_L.bt_rotary(
            q3.data_ptr(), q3.stride(0), q3.stride(1), _ptr(k3), 0 if k3 is None else k3.stride(0), 0 if k3 is None else k3.stride(1), dt,
            pos.data_ptr(), int(pos.dtype == torch.int64), _ptr(freq), int(freq.dtype == torch.float64), int(interleaved), float(amplitude),
            int(backward), q3.shape[0], q3.shape[1], 0 if k3 is None else k3.shape[1], q3.shape[2], 2 * freq.shape[0], out[0].data_ptr(),
            _ptr(out[1]), _stream(q)))
    return out


def cache_head_dim(dtype: torch.dtype, head_dim: int) -> int:
    """Features that a cache keeps of a head: ``head_dim`` rounded up to 64 bytes."""
    _check(dtype in _DT, "the cache must be float32, float16 or bfloat16")
    _check(0 < head_dim <= 256, f"head_dim must be 1 .. 256, got {head_dim}")
    return _L.bt_cache_head_dim(_DT[dtype], head_dim)


def cache_args(rows: Tensor, kv_heads: Optional[int], k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor,
               q_starts: Optional[Tensor]) -> None:
    """What every call on the cache has to hold; ``rows``: the new tokens' ``[tokens, heads, D]``."""
    _check(rows.dim() == 3, "k, v and q must be 3D [tokens, heads, head_dim]")
    _check(k_cache.dim() == 4 and k_cache.shape == v_cache.shape, "the caches must match, 4D [pages, kv_heads, page_size, features]")
    _check(k_cache.dtype == rows.dtype == v_cache.dtype, "the caches must have the rows' dtype")
    _check(k_cache.is_contiguous() and v_cache.is_contiguous(), "the caches must be contiguous")
    _check(k_cache.shape[3] == cache_head_dim(rows.dtype, rows.shape[2]),
           f"the caches keep {k_cache.shape[3]} features, a head of {rows.shape[2]} wants {cache_head_dim(rows.dtype, rows.shape[2])}")
    _check(kv_heads is None or k_cache.shape[1] == kv_heads, "kv_heads don't match the caches")
    page = k_cache.shape[2]
    _check(page >= 32 and page & (page - 1) == 0 and k_cache.shape[0] > 0, "page_size must be a power of two from 32 on")
    index = [t for t in (block_table, lengths, q_starts) if t is not None]
    _check(all(t.dtype == torch.int32 for t in index), "block_table, lengths and q_starts must be int32")
    _check(block_table.dim() == 2 and lengths.dim() == 1 and block_table.shape[0] == lengths.shape[0], "block_table must be 2D [sequences, width], lengths 1D")
    _check(q_starts is None or (q_starts.dim() == 1 and q_starts.shape[0] == lengths.shape[0] + 1), "q_starts must be 1D [sequences + 1]")
    _check(q_starts is not None or lengths.shape[0] == rows.shape[0], "without q_starts every sequence has one token")
    _check(all(t.device == rows.device for t in (k_cache, v_cache, *index)), "All tensors must be on one device")
    _check(rows.shape[0] == 0 or (lengths.shape[0] > 0 and block_table.shape[1] > 0), "there are tokens and no sequences")


def append_args(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor, q_starts: Optional[Tensor],
                q: Optional[Tensor], inv_freq: Optional[Tensor]) -> None:
    cache_args(k, k.shape[1] if k.dim() == 3 else None, k_cache, v_cache, block_table, lengths, q_starts)
    _check(v.shape == k.shape and v.dtype == k.dtype and v.device == k.device, "k and v must match")
    if q is not None:
        _check(q.dim() == 3 and q.shape[0] == k.shape[0] and q.shape[2] == k.shape[2] and q.dtype == k.dtype and q.device == k.device,
               "q must be [tokens, heads, head_dim] of k's tokens and dtype")
        _check(inv_freq is not None, "q is turned by inv_freq, which is not given")
    _rotary_checks(k.shape[2], inv_freq, k.device)
    a, b, size = k_cache.data_ptr(), v_cache.data_ptr(), k_cache.numel() * k_cache.element_size()
    _check(a + size <= b or b + size <= a, "the caches share memory")


def cache_append(k: Tensor, v: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor, q_starts: Optional[Tensor],
                 q: Optional[Tensor], inv_freq: Optional[Tensor], interleaved: bool, amplitude: float, first_position: int) -> Optional[Tensor]:
    """The new tokens' keys (turned) and values to their pages; ``q`` turned, or None."""
    append_args(k, v, k_cache, v_cache, block_table, lengths, q_starts, q, inv_freq)
    _check(k.is_cuda, "All tensors must be CUDA")
    dt = _dt(k, "k")
    out = None if q is None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if k.numel() == 0:
        return out
    if q is not None and q.numel() == 0:
        q = None
    k, v = _token_rows(k), _token_rows(v)
    q = None if q is None else _token_rows(q)
    table, lengths = block_table.contiguous(), lengths.contiguous()
    starts = None if q_starts is None else q_starts.contiguous()
    freq = None if inv_freq is None else inv_freq.contiguous()
    for cache in (k_cache, v_cache):
        if not cache.is_inference():
            torch.autograd.graph.increment_version(cache)
    with _on(k):
        _status(_L.bt_cache_append(
            k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1), _ptr(q), 0 if q is None else q.stride(0),
            0 if q is None else q.stride(1), dt, _ptr(freq), int(freq is not None and freq.dtype == torch.float64), int(interleaved), float(amplitude),
            int(first_position), k.shape[0], 0 if q is None else q.shape[1], k.shape[1], k.shape[2], 0 if freq is None else 2 * freq.shape[0],
            k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0], k_cache.shape[2], table.data_ptr(), table.shape[1], lengths.data_ptr(),
            _ptr(starts), lengths.shape[0], _ptr(out), _stream(k)))
    return out


def attention_args(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor, q_starts: Optional[Tensor],
                   scale: Optional[float], prefix_table: Optional[Tensor], prefix_length: int, max_length: Optional[int]) -> Tuple[float, int]:
    """The checked call's scale and its bound of a sequence's length."""
    cache_args(q, None, k_cache, v_cache, block_table, lengths, q_starts)
    _check(k_cache.shape[1] > 0 and q.shape[1] % k_cache.shape[1] == 0, "heads must be a multiple of kv_heads")
    page, most = k_cache.shape[2], block_table.shape[1] * k_cache.shape[2]
    _check(prefix_length >= 0, "prefix_length is negative")
    if prefix_length:
        _check(prefix_table is not None and prefix_table.dim() == 1 and prefix_table.dtype == torch.int32 and prefix_table.device == q.device,
               "prefix_table must be 1D int32 on q's device")
        _check(prefix_length <= prefix_table.shape[0] * page, "prefix_length is beyond prefix_table")
    if max_length is None:
        max_length = most
    _check(0 <= max_length <= most, f"max_length must be 0 .. {most}, what block_table holds")
    scale = q.shape[2] ** -0.5 if scale is None else float(scale)
    _check(0.0 < scale < 3.0e38, "scale must be a positive number")
    return scale, max_length


def cached_attention(q: Tensor, k_cache: Tensor, v_cache: Tensor, block_table: Tensor, lengths: Tensor, q_starts: Optional[Tensor],
                     scale: Optional[float], prefix_table: Optional[Tensor], prefix_length: int, return_lse: bool, max_length: Optional[int]):
    """``out`` ``[tokens, heads, D]``, with ``return_lse`` also fp32 ``[tokens, heads]``."""
    scale, longest = attention_args(q, k_cache, v_cache, block_table, lengths, q_starts, scale, prefix_table, prefix_length, max_length)
    _check(q.is_cuda, "All tensors must be CUDA")
    dt = _dt(q, "q")
    (tokens, heads, dim), (pages, kv_heads, page, _), (n_seq, width) = q.shape, k_cache.shape, block_table.shape
    out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=q.device) if return_lse else None
    if q.numel():
        q, table, lengths = _token_rows(q), block_table.contiguous(), lengths.contiguous()
        starts = None if q_starts is None else q_starts.contiguous()
        prefix = prefix_table.contiguous() if prefix_length else None
        with _on(q):
            per = 16 // q.element_size()
            in_place = all(n % per == 0 for n in (dim, q.stride(0), q.stride(1))) and q.data_ptr() % 16 == 0
            ws = _workspace(_L.bt_cached_attention_workspace_bytes(dt, int(in_place), tokens, heads, kv_heads, dim, page, width, longest, int(starts is not None), n_seq,
                                                                   prefix_length), q.device)
            _status(_L.bt_cached_attention(
                q.data_ptr(), q.stride(0), q.stride(1), dt, k_cache.data_ptr(), v_cache.data_ptr(), pages, page, table.data_ptr(), width, longest,
                lengths.data_ptr(), _ptr(starts), n_seq, _ptr(prefix), prefix_length, scale, tokens, heads, kv_heads, dim, out.data_ptr(), _ptr(lse),
                _ptr(ws), 0 if ws is None else ws.numel(), _stream(q)))
    return (out, lse) if return_lse else out
