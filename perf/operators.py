"""The feed-forward half of a pre-norm block, in training and ahead of int8 layers, as cases that can be timed.

A case is a dict of plain values; its ``kind`` names the operator:

* ``norm``   ``ops.add_rmsnorm``: a branch is added to the residual stream and the sum is normalised, with the int8 rows that
             the int8 layers read (``int8``) or with the gradients of a training step (``train``);
* ``gated``  ``ops.ternary_gated_linear``: ``silu(gate(x)) * up(x)`` with both projections ternarised from full-precision masters
             as they are read, forward alone (evaluation while training) or with the gradients (``train``).

``own`` false: the operators in elementary torch operations, in 32 bits; true: the framework's kernels.
"""

import math

import torch

own = False

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"fp32": 4, "fp16": 2, "bf16": 2}
_EPS = 1e-5
_THRESHOLD = 0.05


def _norm_case(name, rows, k, dtype, stream="same", int8=False, train=False):
    return dict(name=name, kind="norm", rows=rows, k=k, dtype=dtype, stream=stream, int8=int8, train=train)


def _gated_case(name, rows, d, ffn, dtype, bias=False, train=True):
    return dict(name=name, kind="gated", rows=rows, d=d, ffn=ffn, dtype=dtype, bias=bias, train=train)


def listed():
    return [
        # One decoded token between two layers of the 2B-parameter stack: the smallest call, launch and host latency.
        _norm_case("norm_token", 1, 2560, "bf16"),
        # A batched decode step (16 sequences) ahead of int8 layers.
        _norm_case("norm_batch_int8", 16, 4096, "fp16", int8=True),
        # A prefill of 8 x 512 tokens ahead of the int8 layers of the 2B-parameter stack.
        _norm_case("norm_prefill_int8", 4096, 2560, "bf16", int8=True),
        # Training on rows that fill no vector, half-precision branches on a residual stream kept in fp32.
        _norm_case("norm_ragged", 777, 1001, "fp16", stream="fp32", train=True),
        # A training step's share of one norm of the 2B-parameter stack over 8 x 512 tokens.
        _norm_case("norm_train", 4096, 2560, "bf16", train=True),
        # Training in the layers' default dtype on many short rows.
        _norm_case("norm_train_fp32", 16384, 768, "fp32", train=True),
        # A small network in training: the plumbing sizes, all launches.
        _gated_case("gated_small", 32, 512, 256, "fp32", bias=True),
        # One token evaluated on the masters: the bytes of the masters.
        _gated_case("gated_token", 1, 2560, 6912, "bf16", train=False),
        # A validation prompt of a thousand tokens between two training steps.
        _gated_case("gated_prompt", 1000, 2560, 6912, "bf16", train=False),
        # Training with dimensions that are no multiple of a vector, biases, half precision.
        _gated_case("gated_ragged", 500, 1100, 2730, "fp16", bias=True),
        # Training in the layers' default dtype.
        _gated_case("gated_train_fp32", 4096, 768, 2048, "fp32"),
        # A training step's share of one block of the 2B-parameter stack over 8 x 512 tokens.
        _gated_case("gated_train", 4096, 2560, 6912, "bf16"),
    ]


# ---- draws -----------------------------------------------------------------------------------------------------------

_MAX_ELEMENTS = 16384 * 768         # norm_train_fp32's
_MAX_WEIGHTS = 2560 * 6912          # of a projection: gated_train's
_MAX_FLOPS = 12.0 * 4096 * 2560 * 6912
_MAX_FLOPS_FP32 = 12.0 * 4096 * 768 * 2048


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _features(rng, lo, hi):
    """A dimension: mostly a multiple of 256 or of 16 as layers have them, now and then any number."""
    v = _log_uniform(rng, lo, hi)
    step = rng.choice((256, 256, 64, 16, 1))
    return max(lo, v // step * step)


def _rows(rng, hi):
    return rng.choice((_log_uniform(rng, 1, 64), _log_uniform(rng, 64, hi), _log_uniform(rng, 64, hi)))


def draw(rng):
    while True:
        dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
        if rng.random() < 0.5:
            train = rng.random() < 0.5
            case = dict(kind="norm", rows=_rows(rng, 16384), k=_features(rng, 64, 16384), dtype=dtype,
                        stream=rng.choice(("same", "same", "fp32")), int8=not train and rng.random() < 0.5, train=train)
            if case["rows"] * case["k"] <= _MAX_ELEMENTS:
                return case
        else:
            case = dict(kind="gated", rows=_rows(rng, 8192), d=_features(rng, 64, 8192), ffn=_features(rng, 64, 12288), dtype=dtype,
                        bias=rng.random() < 0.3, train=rng.random() < 0.7)
            if case["d"] * case["ffn"] <= _MAX_WEIGHTS and work(case)["flops"] <= (_MAX_FLOPS_FP32 if dtype == "fp32" else _MAX_FLOPS):
                return case


# ---- what a program holds before the call ----------------------------------------------------------------------------

def _normal(g, shape, std, dtype=torch.float32):
    return torch.randn(shape, generator=g, device=g.device).mul_(std).to(dtype)


def _hidden(g, shape, dtype):
    """N(0, 1) with a thousandth of the entries twenty times as large, as hidden states have them."""
    x = torch.randn(shape, generator=g, device=g.device)
    return torch.where(torch.rand(shape, generator=g, device=g.device) < 1e-3, x * 20, x).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 29)
    dt, rows, train = _DTYPES[case["dtype"]], case["rows"], case["train"]
    state = dict(kind=case["kind"], train=train)
    if case["kind"] == "norm":
        k, sdt = case["k"], torch.float32 if case["stream"] == "fp32" else dt
        state.update(int8=case["int8"], x=_normal(g, (rows, k), 1.0, dt), residual=_hidden(g, (rows, k), sdt),
                     weight=(1 + _normal(g, (k,), 0.1)).to(dt))
        if train:
            state.update(dsum=_normal(g, (rows, k), 0.01, sdt), dnorm=_normal(g, (rows, k), 0.01, dt))
        leaves = ("x", "residual", "weight")
    else:
        d, ffn = case["d"], case["ffn"]
        state.update(x=_normal(g, (rows, d), 1.0, dt), gate=_normal(g, (ffn, d), 0.02, dt), up=_normal(g, (ffn, d), 0.02, dt),
                     gate_bias=_normal(g, (ffn,), 0.1, dt) if case["bias"] else None,
                     up_bias=_normal(g, (ffn,), 0.1, dt) if case["bias"] else None)
        if train:
            state["dh"] = _normal(g, (rows, ffn), 0.05, dt)
        leaves = ("x", "gate", "up", "gate_bias", "up_bias")
    if train:
        for name in leaves:
            if state[name] is not None:
                state[name].requires_grad_()
    return state


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    if own:
        return _norm_own(state) if state["kind"] == "norm" else _gated_own(state)
    with torch.no_grad():
        return _norm_plain(state) if state["kind"] == "norm" else _gated_plain(state)


def _codes(q, scale, dtype):
    """What int8 rows stand for, in the activations' type."""
    return q * scale.to(dtype).unsqueeze(-1)


def _norm_own(st):
    from bittorch_amd import ops

    x, residual, weight = st["x"], st["residual"], st["weight"]
    if st["train"]:
        total, norm = ops.add_rmsnorm(x, residual, weight, _EPS)
        dx, dresidual, dweight = torch.autograd.grad((total, norm), (x, residual, weight), (st["dsum"], st["dnorm"]))
        return dict(sum=total.detach(), norm=norm.detach(), dx=dx, dresidual=dresidual, dweight=dweight)
    if st["int8"]:
        total, q, scale = ops.add_rmsnorm(x, residual, weight, _EPS, store=False, quantize=True)
        return dict(sum=total, codes=_codes(q, scale, x.dtype), scale=scale)
    total, norm = ops.add_rmsnorm(x, residual, weight, _EPS)
    return dict(sum=total, norm=norm)


def _norm_plain(st):
    dt, w = st["x"].dtype, st["weight"].float()
    total = (st["x"].float() + st["residual"].float()).to(st["residual"].dtype)
    s = total.float()  # (the norm is that of the sum as the stream keeps it)
    r = 1.0 / torch.sqrt(s.double().square().sum(-1, keepdim=True).float() / s.shape[-1] + _EPS)
    norm = ((s * r) * w).to(dt)
    out = dict(sum=total)
    if st["int8"]:
        # (values next to a border between two codes: every step is one rounding in 32 bits, as the quantizer is defined)
        amax = norm.float().abs().amax(-1, keepdim=True)
        scale = torch.where(amax > 1e-6, amax / 127.0, torch.ones_like(amax))
        v = norm.float() * (1.0 / scale)
        q = (torch.sign(v) * torch.floor(v.abs().double() + 0.5)).clamp(-127, 127).to(torch.int8)
        out.update(codes=_codes(q, scale.squeeze(-1), dt), scale=scale.squeeze(-1))
        return out
    out["norm"] = norm
    if st["train"]:
        dy, xhat = st["dnorm"].float(), s * r
        dyw = dy * w
        ds = st["dsum"].float() + r * (dyw - xhat * (dyw * xhat).mean(-1, keepdim=True))
        out.update(dx=ds.to(dt), dresidual=ds.to(total.dtype), dweight=(dy * xhat).sum(0).to(dt))
    return out


def _gated_own(st):
    from bittorch_amd import ops

    leaves = [st[n] for n in ("x", "gate", "up", "gate_bias", "up_bias") if st[n] is not None]
    if not st["train"]:
        with torch.no_grad():
            return dict(h=ops.ternary_gated_linear(st["x"], st["gate"], st["up"], st["gate_bias"], st["up_bias"]))
    h = ops.ternary_gated_linear(st["x"], st["gate"], st["up"], st["gate_bias"], st["up_bias"])
    return dict(h=h.detach(), grads=torch.autograd.grad(h, leaves, st["dh"]))


def _ternary(w):
    """The ternary values and the rows' scales in 32 bits; the threshold is rounded to the masters' type, as it is defined."""
    mag = w.abs()
    scale = mag.amax(1, keepdim=True).clamp(min=1e-8)
    keep = mag > (scale.float() * _THRESHOLD).to(w.dtype)
    return torch.where(keep, torch.sign(w), torch.zeros_like(w)).float(), scale.float()


def _gated_plain(st):
    dt, x = st["x"].dtype, st["x"].float()
    (tg, ag), (tu, au) = _ternary(st["gate"]), _ternary(st["up"])
    wg, wu = tg * ag, tu * au
    g, u = x @ wg.t(), x @ wu.t()
    if st["gate_bias"] is not None:
        g, u = g + st["gate_bias"].float(), u + st["up_bias"].float()
    sig = 1.0 / (1.0 + torch.exp(-g))
    silu = g * sig
    out = dict(h=(silu * u).to(dt))
    if st["train"]:
        dh = st["dh"].float()
        dg, du = dh * u * (sig * (1.0 + g * (1.0 - sig))), dh * silu
        grads = [(dg @ wg + du @ wu).to(dt), (ag * (dg.t() @ x)).to(dt), (au * (du.t() @ x)).to(dt)]
        if st["gate_bias"] is not None:
            grads += [dg.sum(0).to(dt), du.sum(0).to(dt)]
        out["grads"] = grads
    return out


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    size, rows, train = _SIZE[case["dtype"]], case["rows"], case["train"]
    if case["kind"] == "norm":
        k, stream = case["k"], 4 if case["stream"] == "fp32" else size
        # x, the stream in and out, and the norm or its codes
        nbytes = rows * k * (size + 2 * stream + (1 if case["int8"] else size)) + size * k + (4 * rows if case["int8"] else 0)
        if train:  # both incoming gradients and both outgoing ones (one tensor where their type is the same)
            nbytes += rows * k * (stream + size + stream + (size if stream != size else 0)) + size * k
        return {"bytes": nbytes, "flops": (14.0 if train else 5.0) * rows * k}
    d, ffn = case["d"], case["ffn"]
    nbytes = size * (rows * d + 2 * ffn * d + rows * ffn + (2 * ffn if case["bias"] else 0))
    if train:
        nbytes += size * (rows * ffn + rows * d + 2 * ffn * d + (2 * ffn if case["bias"] else 0))
    return {"bytes": nbytes, "flops": (12.0 if train else 4.0) * rows * d * ffn}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    dt, train = _DTYPES[case["dtype"]], case["train"]

    def leaf(t):
        return None if t is None else t.detach().double().requires_grad_(train)

    with torch.enable_grad():
        if case["kind"] == "norm":
            x, residual, weight = leaf(st["x"]), leaf(st["residual"]), leaf(st["weight"])
            total = x + residual
            # the norm of the sum as it is stored; its gradient passes through the rounding
            stored = total + (total.detach().to(st["residual"].dtype).double() - total.detach())
            norm = stored / (stored.pow(2).mean(dim=-1, keepdim=True) + _EPS).pow(0.5) * weight
            out = dict(sum=total.detach())
            if case["int8"]:
                y = norm.to(dt).double()
                scale = y.abs().max(dim=-1).values / 127
                scale = torch.where(scale * 127 > 1e-6, scale, torch.ones_like(scale))
                code = torch.floor((y / scale[:, None]).abs() + 0.5).clamp(max=127) * y.sign()
                # (32-bit rows come to a border between two codes by the last bit of their norm: no code has a value of its own there)
                out.update(codes=None if dt == torch.float32 else code * scale[:, None], scale=scale)
                return out
            out["norm"] = norm.detach()
            if train:
                grads = torch.autograd.grad((total, norm), (x, residual, weight), (st["dsum"].double(), st["dnorm"].double()))
                out.update(zip(("dx", "dresidual", "dweight"), grads))
            return out
        x, gate_bias, up_bias = leaf(st["x"]), leaf(st["gate_bias"]), leaf(st["up_bias"])
        scales, dense = [], []
        for master in (st["gate"].detach(), st["up"].detach()):
            top = master.abs().max(dim=1).values.double()
            border = (top * torch.tensor(_THRESHOLD, dtype=torch.float32).double()).float().to(master.dtype).double()
            m = master.double()
            ternary = (m > border[:, None]).double() - (m < -border[:, None]).double()
            scales.append(top)
            dense.append((ternary * top[:, None]).requires_grad_(train))
        gate, up = torch.matmul(x, dense[0].T), torch.matmul(x, dense[1].T)
        if case["bias"]:
            gate, up = gate + gate_bias, up + up_bias
        h = gate / (1 + (-gate).exp()) * up
        out = dict(h=h.detach())
        if train:
            leaves = [x] + dense + ([gate_bias, up_bias] if case["bias"] else [])
            grads = list(torch.autograd.grad(h, leaves, st["dh"].double()))
            for i, top in enumerate(scales):  # straight through: the gradient of the effective weights times their row's scale
                grads[1 + i] = grads[1 + i] * top[:, None]
            out["grads"] = grads
        return out
