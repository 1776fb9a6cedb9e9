"""``nn.TernaryGatedMLP`` and the operators of a pre-norm block's feed-forward half together, as a training program uses them."""
import copy

import pytest
import torch
import torch.nn.functional as F

import bittorch_amd as bt
from conftest import announce

EPS = 1e-5


def _mlp(d, ffn, seed=0, **kwargs):
    torch.manual_seed(seed)
    return bt.nn.TernaryGatedMLP(d, ffn, **kwargs)


def _norm_error(got, want):
    got, want = got.detach().double().cpu(), want.detach().double().cpu()
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("bias", [False, True])
def test_on_the_cpu_it_is_the_three_layers(bias):
    mlp = _mlp(24, 40, bias=bias)
    assert sorted(mlp.state_dict()) == sorted(f"{m}.{p}" for m in ("gate", "up", "down") for p in (("weight", "bias") if bias else ("weight",)))
    x, res = torch.randn(2, 5, 24), torch.randn(2, 5, 24)
    want = mlp.down(F.silu(mlp.gate(x)) * mlp.up(x))
    assert torch.equal(mlp(x), want) and torch.equal(mlp(x, residual=res), want + res)
    w = 1 + 0.1 * torch.randn(24)
    h = F.rms_norm(x, (24,), w, EPS)
    assert torch.equal(mlp(x, w, EPS, res), mlp.down(F.silu(mlp.gate(h)) * mlp.up(h)) + res)
    other = copy.deepcopy(mlp)
    other.load_state_dict(mlp.state_dict())
    assert torch.equal(other(x), want)
    with torch.no_grad():
        assert torch.allclose(mlp.to_inference()(x), want, rtol=1e-5, atol=1e-6)
        assert torch.allclose(bt.utils.convert_linear_layers(torch.nn.Sequential(mlp))[0](x), want, rtol=1e-5, atol=1e-6)
    mlp.gate.quantize = False
    assert torch.equal(mlp(x), mlp.down(F.silu(F.linear(x, mlp.gate.weight, mlp.gate.bias)) * mlp.up(x)))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d,ffn,bias", [(96, 160, False), (100, 70, True)])
def test_training_step_and_evaluation(d, ffn, bias, dt):
    announce("gated mlp", d, ffn, bias, dt)
    mlp = _mlp(d, ffn, seed=1, bias=bias).cuda()
    ref = copy.deepcopy(mlp).double().cpu()
    g = torch.Generator().manual_seed(2)
    x, dy = torch.randn(3, 21, d, generator=g).to(dt), torch.randn(3, 21, d, generator=g).to(dt)
    xc, xr = x.cuda().requires_grad_(), x.double().requires_grad_()
    y = mlp(xc)
    y.backward(dy.cuda())
    want = ref(xr)
    want.backward(dy.double())
    # half a step each: h, the down projection's output and, backward, its gradient, G and the products; TernaryLinear rounds its scale too
    half = torch.finfo(dt).eps / 2
    tol = 3 * half + 1e-5
    assert y.dtype == dt and _norm_error(y, want) <= tol
    assert _norm_error(xc.grad, xr.grad) <= tol
    for (name, p), q in zip(mlp.named_parameters(), ref.parameters()):
        assert p.grad.dtype == p.dtype and _norm_error(p.grad, q.grad) <= tol, name
    with torch.no_grad():
        kept = mlp(xc)
        assert _norm_error(kept, want) <= tol + 2 * half  # (the projections rounded, and silu, as the converted module rounds them)
        assert mlp._packed.key is not None
        fused = mlp.to_inference(fuse_gate_up=True)
        assert torch.equal(mlp.hidden(xc), fused.gate_up.forward_swiglu(xc) if ffn % 16 == 0 else bt.ops.swiglu(fused.gate_up(xc)[..., :ffn], fused.gate_up(xc)[..., ffn:]))
        for p in mlp.parameters():
            p.mul_(-1.5)
        assert torch.equal(mlp.hidden(xc), copy.deepcopy(mlp).hidden(xc)) and not torch.equal(mlp(xc), kept)
        mlp.gate.weight.data.zero_()  # (unseen by the version counter)
        mlp.invalidate_packed_cache()
        if not bias:
            assert not mlp.hidden(xc).any()
        one = mlp.hidden(xc[0, 0])
        assert one.shape == (ffn,)
    frozen = _mlp(d, ffn, seed=1, bias=bias).cuda().requires_grad_(False)
    z = x.cuda().requires_grad_()
    frozen(z).backward(dy.cuda())
    assert _norm_error(z.grad, xr.grad) <= tol


@pytest.mark.gpu
@pytest.mark.parametrize("dt,stream", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32),
                                       (torch.float16, torch.float32)])
@pytest.mark.parametrize("rows,d,ffn", [(1, 64, 48), (130, 264, 176), (77, 129, 90)])
def test_feed_forward_half_of_a_block(rows, d, ffn, dt, stream):
    """A branch is added to the stream and normed, the gated pair and the down projection follow, and their sum is normed again: forward and
    every gradient against the same in 64 bits."""
    announce("block half", rows, d, ffn, dt, stream)
    g = torch.Generator().manual_seed(rows + d)
    mk = lambda std, *shape: torch.randn(*shape, generator=g) * std
    branch, x, ds, dy = mk(1, rows, d).to(dt), mk(2, rows, d).to(stream), mk(1, rows, d).to(stream), mk(1, rows, d).to(dt)
    n1, n2 = (1 + mk(0.1, d)).to(dt), (1 + mk(0.1, d)).to(dt)
    mlp = _mlp(d, ffn, seed=3).to(dt)
    ref = copy.deepcopy(mlp).double()
    # (a 16-bit master's threshold is rounded to 16 bits: the codes are taken from the masters as they are trained)
    for layer, trained in ((ref.gate, mlp.gate), (ref.up, mlp.up), (ref.down, mlp.down)):
        q, s = trained.get_quantized_weight()
        with torch.no_grad():
            layer.weight.copy_(q.double() * s.double().reshape(-1, 1))
    mlp = mlp.cuda()
    leaves = [t.cuda().requires_grad_() for t in (branch, x, n1, n2)]
    s1, h = bt.ops.add_rmsnorm(leaves[0], leaves[1], leaves[2], EPS)
    out = bt.ops.add_rmsnorm(mlp(h), s1, leaves[3], EPS)
    got = torch.autograd.grad(out, [*leaves, *mlp.parameters()], (ds.cuda(), dy.cuda()))

    refs = [t.double().requires_grad_() for t in (branch, x, n1, n2)]
    t1 = refs[0] + refs[1]
    t1 = t1 + (t1.detach().to(stream).double() - t1.detach())  # (the stream as it is stored)
    hr = F.rms_norm(t1, (d,), refs[2], EPS)
    t2 = t1 + ref(hr)
    nr = F.rms_norm(t2, (d,), refs[3], EPS)
    want = torch.autograd.grad((t2, nr), [*refs, *ref.parameters()], (ds.double(), dy.double()))
    # forward: at most five roundings to 16 bits one after the other (the sum, the norm, h, the down projection and its scale), backward
    # five more; independent of each other, so their root of squares and not their sum: sqrt(10) halves of a step
    tol = 3.2 * torch.finfo(dt).eps / 2 + 1e-5
    for a, b in zip(out, (t2, nr)):
        assert _norm_error(a, b) <= tol
    for a, b in zip(got, want):
        assert _norm_error(a, b) <= tol


@pytest.mark.gpu
def test_block_stack_training_forward_and_gradient():
    """Two blocks, fused glue and unfused modules: the same loss and gradients up to fp32's sums."""
    from bittorch_amd.utils.block_stack import BlockStack
    std = dict(q=0.02, k=0.02, v=0.02, o=0.01, gate=0.01, up=0.01, down=0.005)
    stack = BlockStack("cuda", layers=2, d_model=128, heads=4, ffn=208, batch=2, seq=24, vocab=64, act_dtype=torch.float32, master_std=std)
    params = [*stack.emb.parameters(), *stack.blocks.parameters(), *stack.final.parameters()]
    dy = torch.randn(2, 24, 128, generator=torch.Generator().manual_seed(1)).cuda()
    fused = stack.forward_train()
    got = torch.autograd.grad(fused, params, dy)
    x = stack.emb(stack.tokens)
    for blk in stack.blocks:
        x = blk(x)
    plain = stack.final(x)
    want = torch.autograd.grad(plain, params, dy)
    # fp32 sums of up to 208 terms in another order, through two blocks
    assert _norm_error(fused, plain) <= 1e-5
    for a, b in zip(got, want):
        assert _norm_error(a, b) <= 2e-5


@pytest.mark.gpu
def test_training_step_captured_and_replayed():
    """A step on fresh leaves in a graph, replayed between eager steps of the same module."""
    mlp = _mlp(136, 80, seed=4).to(torch.bfloat16).cuda()
    x, dy = torch.randn(40, 136, device="cuda").bfloat16(), torch.randn(40, 136, device="cuda").bfloat16()
    n = torch.ones(136, device="cuda", dtype=torch.bfloat16)

    def step(x, dy):
        leaves = [t.detach().requires_grad_() for t in (x, n, mlp.gate.weight, mlp.up.weight)]
        s, h = bt.ops.add_rmsnorm(leaves[0], x, leaves[1], EPS)
        out = bt.ops.ternary_gated_linear(h, *leaves[2:])
        return (out.detach(), *torch.autograd.grad((s, out), leaves, (dy, out.detach())))

    static = [x.clone(), dy.clone()]
    expect = [t.clone() for t in step(*static)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*static)
    for k in range(3):
        new = x * (k + 1)
        static[0].copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step(new, dy)))
    static[0].copy_(x)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, expect))


@pytest.mark.gpu
@pytest.mark.parametrize("learns", ["gate.bias", "up.bias", "down.weight", "x"])
def test_frozen_weights_with_something_else_that_learns(learns):
    announce("gated mlp, frozen but for", learns)
    mlp = _mlp(64, 48, seed=5, bias=True).cuda()
    x = torch.randn(9, 64, generator=torch.Generator().manual_seed(6)).cuda()
    want = {n: torch.autograd.grad(mlp(x.requires_grad_()).square().sum(), t)[0] for n, t in (*mlp.named_parameters(), ("x", x)) if n == learns}[learns]
    x = x.detach().requires_grad_(learns == "x")
    for n, p in mlp.named_parameters():
        p.requires_grad_(n == learns)
    leaf = x if learns == "x" else dict(mlp.named_parameters())[learns]
    got, = torch.autograd.grad(mlp(x).square().sum(), leaf)
    # (down.weight: the pair's hidden values come from the kept copy, as those of the converted module, rounded to fp32 at other places)
    assert _norm_error(got, want) <= 1e-5


@pytest.mark.gpu
def test_kept_weights_on_other_streams_and_in_graphs():
    announce("gated mlp, kept weights")
    mlp = _mlp(512, 768, seed=7).cuda().bfloat16()
    x = torch.randn(33, 512, generator=torch.Generator().manual_seed(8)).cuda().bfloat16()
    busy = torch.randn(4096, 4096, device="cuda")
    with torch.no_grad():
        want = mlp(x).clone()
        mlp.gate.weight.mul_(1.0)  # (the same values, packed anew)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                busy = busy @ busy * 1e-3
            first = mlp(x)  # packs behind all of that
        second = mlp(x)  # this stream has not waited for it
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want)
        copied = copy.deepcopy(mlp)
        assert copied._packed.key is None and torch.equal(copied(x), want)
        mlp.invalidate_packed_cache()
        for layer in (mlp.gate, mlp.up, mlp.down):
            layer(torch.zeros(1, layer.in_features, dtype=x.dtype, device="cuda"))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mlp(x)
        assert mlp._packed.key is None  # (what the capture packed is written by each replay only)
        assert torch.equal(mlp(x), want)
        for _ in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(mlp(x), want)


def _rewritten(device):
    """Memory that was given back, taken again and overwritten."""
    torch.cuda.synchronize()
    return [torch.full((n,), 255, dtype=torch.uint8, device=device) for n in (512, 4096, 1 << 16, 1 << 18, 1 << 20, 3 << 20, 1 << 22) for _ in range(8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bias", [False, True])
def test_a_graph_captured_on_kept_weights_follows_the_masters(bias, dt):
    """Evaluated, captured, the masters changed, evaluated again and the memory of the first packing written over: the graph's replays are
    the module's values."""
    announce("gated mlp, captured warm", bias, dt)
    mlp = _mlp(512, 768, seed=9, bias=bias).to(dt).cuda()
    x = torch.randn(33, 512, generator=torch.Generator().manual_seed(8)).cuda().to(dt)
    with torch.no_grad():
        mlp.hidden(x)
        assert mlp._packed.key is not None
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mlp.hidden(x)
        for n in range(3):
            for p in mlp.parameters():
                p.mul_(-1.25)
            if n == 1:
                mlp.invalidate_packed_cache()
            want = mlp.hidden(x).clone()
            held = _rewritten(x.device)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(mlp.hidden(x), want)
            del held


@pytest.mark.gpu
@pytest.mark.parametrize("warm", [False, True])
@pytest.mark.parametrize("cls", [bt.nn.TernaryLinear, bt.nn.TernaryLinearCUDA])
def test_a_layer_captured_in_evaluation_follows_its_master(cls, warm):
    """As above for a single layer, captured with its packed weights kept and without: what the capture packed is written by its replays
    only, so an evaluation behind the capture does not read it."""
    announce("layer captured", cls.__name__, warm)
    torch.manual_seed(10)
    layer = cls(512, 768).bfloat16().cuda()
    x = torch.randn(40, 512, generator=torch.Generator().manual_seed(8)).cuda().bfloat16()
    with torch.no_grad():
        want = layer(x).clone()
        if not warm:
            layer.invalidate_packed_cache()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(x)
        assert (layer._packed.key is not None) == warm and torch.equal(layer(x), want)
        for n in range(3):
            layer.weight.mul_(-1.25)
            want = layer(x).clone()
            held = _rewritten(x.device)
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(layer(x), want)
            del held


@pytest.mark.gpu
def test_a_layers_kept_weights_on_another_stream():
    announce("layer, kept weights on another stream")
    torch.manual_seed(11)
    layer = bt.nn.TernaryLinear(512, 768).bfloat16().cuda()
    x = torch.randn(40, 512, generator=torch.Generator().manual_seed(8)).cuda().bfloat16()
    busy = torch.randn(4096, 4096, device="cuda")
    with torch.no_grad():
        want = layer(x).clone()
        layer.weight.mul_(1.0)  # (the same values, packed anew)
        side = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for _ in range(20):
                busy = busy @ busy * 1e-3
            first = layer(x)  # packs behind all of that
        second = layer(x)  # this stream has not waited for it
        torch.cuda.synchronize()
        assert torch.equal(first, want) and torch.equal(second, want)
        copied = copy.deepcopy(layer)
        assert copied._packed.key is None and torch.equal(copied(x), want)


class _Sign(torch.nn.Module):
    """A parametrization with a state of its own: the weight is a new tensor, without a history, at every reading."""

    def __init__(self):
        super().__init__()
        self.by = torch.nn.Parameter(torch.ones(()))

    def forward(self, w):
        return w * self.by


@pytest.mark.gpu
@pytest.mark.parametrize("cls", [bt.nn.TernaryLinear, bt.nn.TernaryLinearCUDA])
def test_kept_weights_of_a_weight_that_is_computed(cls):
    """A new tensor at the address of one that is gone, of the same version, is not what was packed."""
    announce("kept weights, computed weight", cls.__name__)
    torch.manual_seed(12)
    layer = cls(64, 48, bias=False).cuda()
    torch.nn.utils.parametrize.register_parametrization(layer, "weight", _Sign())
    x = torch.randn(5, 64, device="cuda")
    with torch.no_grad():
        for _ in range(3):
            before = layer(x).clone()
            layer.parametrizations.weight[0].by.neg_()
            assert torch.equal(layer(x), -before) and before.any()


@pytest.mark.gpu
def test_kept_weights_of_a_parameter_put_in_the_place_of_another():
    announce("kept weights, parameter replaced")
    torch.manual_seed(13)
    mlp, other = _mlp(512, 768).cuda(), None
    x = torch.randn(33, 512, device="cuda")
    with torch.no_grad():
        for layer in (mlp.gate, mlp.down):
            mlp(x)
            at, version, values = layer.weight.data_ptr(), layer.weight._version, -layer.weight.cpu()
            del layer.weight
            layer.weight = torch.nn.Parameter(values.cuda())
            while layer.weight._version < version:
                layer.weight.mul_(1.0)
            assert torch.equal(mlp(x), copy.deepcopy(mlp)(x)), (at == layer.weight.data_ptr(), version)


@pytest.mark.gpu
def test_modules_made_in_inference_mode():
    """Their parameters have no version counter: nothing is kept, and they are evaluated all the same."""
    announce("kept weights, inference tensors")
    with torch.inference_mode():
        mlp = _mlp(64, 48, seed=14, bias=True).cuda()
        x = torch.randn(5, 64, generator=torch.Generator().manual_seed(8)).cuda()
        got = mlp(x)
    other = _mlp(64, 48, seed=14, bias=True).cuda()
    with torch.no_grad():
        # (the pair without kept weights: silu and the projections rounded to fp32 at other places)
        assert _norm_error(got, other(x.clone())) <= 1e-6
    assert mlp._packed.key is None and mlp.down._packed.key is None


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(grad):
    """A tangent is refused, whichever argument has it and whatever the gradient mode; it is never dropped.  Calls without one go on."""
    announce("forward mode", grad)
    import torch.autograd.forward_ad as fa
    mk = lambda *shape: torch.randn(*shape, device="cuda")
    x, r, w, wg, wu, bg, bu = mk(4, 64), mk(4, 64), mk(64), mk(48, 64), mk(48, 64), mk(48), mk(48)
    mlp = _mlp(64, 48, seed=15, bias=True).cuda().requires_grad_(False)
    norm = lambda *a: bt.ops.add_rmsnorm(*a)
    codes = lambda *a: bt.ops.add_rmsnorm(*a, store=False, quantize=True)
    pair = lambda *a: bt.ops.ternary_gated_linear(*a)
    biases = lambda a, g, u, b, c: torch.func.functional_call(mlp, {"gate.weight": g, "up.weight": u, "gate.bias": b, "up.bias": c}, (a,))
    with fa.dual_level(), torch.set_grad_enabled(grad):
        for call, args in ((norm, (x, r, w)), (norm, (x, None, w)), (codes, (x, r, w)), (pair, (x, wg, wu, bg, bu)), (pair, (x[:1], wg, wu)), (mlp, (x,)),
                           (biases, (x, wg, wu, bg, bu))):
            call(*args)
            for n, t in enumerate(args):
                if t is not None:
                    with pytest.raises((NotImplementedError, RuntimeError), match="jvp"):
                        call(*args[:n], fa.make_dual(t, torch.ones_like(t)), *args[n + 1:])
            call(*args)


def _layer_by_layer(mlp, h):
    return F.silu(mlp.gate(h)) * mlp.up(h)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("kind", ["forward", "pre", "backward", "backward pre", "global", "instance"])
def test_hooks_of_both_layers_run(kind, grad):
    """A layer with a hook is called, not read: the pair is then the two layers, as on the CPU."""
    announce("gated mlp, hooks", kind, grad)
    for which in ("gate", "up"):
        mlp, seen = _mlp(64, 48, seed=16, bias=True).cuda(), []
        layer, x = getattr(mlp, which), torch.randn(9, 64, device="cuda", requires_grad=True)
        note = lambda m, *rest: seen.append(m)
        handle = None
        if kind == "forward":
            handle = layer.register_forward_hook(lambda m, args, out: note(m) or out * 0)
        elif kind == "pre":
            handle = layer.register_forward_pre_hook(lambda m, args: note(m) or (args[0] * 2,))
        elif kind == "backward":
            handle = layer.register_full_backward_hook(note)
        elif kind == "backward pre":
            handle = layer.register_full_backward_pre_hook(note)
        elif kind == "global":
            handle = torch.nn.modules.module.register_module_forward_hook(note)
        else:
            inner = layer.forward
            layer.forward = lambda h: note(layer) or inner(h) * 3
        try:
            with torch.set_grad_enabled(grad):
                want = _layer_by_layer(mlp, x)
                seen.clear()
                got = mlp.hidden(x)
                if grad:
                    got.sum().backward()
            assert torch.equal(got, want)
            assert layer in seen or (not grad and kind.startswith("backward"))
        finally:
            if handle is not None:
                handle.remove()


@pytest.mark.gpu
def test_weights_that_a_hook_computes():
    """weight_norm and pruning set the weight in front of each call: two training steps, and an evaluation behind each."""
    announce("gated mlp, weights computed in front of the call")
    import torch.nn.utils.prune as prune
    for change in (lambda m: torch.nn.utils.weight_norm(m), lambda m: prune.random_unstructured(m, "weight", 0.5)):
        torch.manual_seed(17)
        mlp = _mlp(64, 48, seed=17).cuda()
        change(mlp.gate)
        change(mlp.up)
        x = torch.randn(9, 64, device="cuda")
        opt = torch.optim.SGD(mlp.parameters(), lr=1.0)
        for _ in range(2):
            opt.zero_grad()
            got, want = mlp.hidden(x), _layer_by_layer(mlp, x)
            assert torch.equal(got, want)
            got.square().sum().backward()
            assert all(p.grad is not None for n, p in mlp.named_parameters() if not n.startswith("down"))
            opt.step()
            with torch.no_grad():
                assert torch.equal(mlp.hidden(x), _layer_by_layer(mlp, x))


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["gate", "up"])
def test_layers_that_differ_in_backend_or_dtype(which):
    announce("gated mlp, layers that differ", which)
    x = torch.randn(9, 64, device="cuda")
    mlp = _mlp(64, 48, seed=18, bias=True).cuda()
    getattr(mlp, which).backend = "python"
    assert torch.equal(mlp.hidden(x), _layer_by_layer(mlp, x))
    with torch.no_grad():
        assert torch.equal(mlp.hidden(x), _layer_by_layer(mlp, x))
    for part, dtype in (("weight", torch.bfloat16), ("bias", torch.float64)):
        mlp = _mlp(64, 48, seed=18, bias=True).cuda()
        layer = getattr(mlp, which)
        setattr(layer, part, torch.nn.Parameter(getattr(layer, part).detach().to(dtype)))
        y = x.clone().requires_grad_()
        out = mlp.hidden(y)
        assert torch.equal(out, _layer_by_layer(mlp, y))
        out.square().sum().backward()
        assert getattr(layer, part).grad.dtype == dtype and y.grad is not None
        with torch.no_grad():
            assert torch.equal(mlp.hidden(x), _layer_by_layer(mlp, x))


@pytest.mark.gpu
@pytest.mark.parametrize("dt,wt", [(torch.float64, torch.float64), (torch.float64, None), (torch.float32, torch.bfloat16), (torch.float32, torch.float64)])
def test_norms_that_the_kernel_does_not_take(dt, wt):
    announce("gated mlp, norm", dt, wt)
    mlp = _mlp(64, 48, seed=19).cuda()
    x = torch.randn(5, 64, device="cuda", dtype=dt)
    w = None if wt is None else (1 + 0.1 * torch.randn(64, device="cuda")).to(wt)
    assert torch.equal(mlp(x, w, EPS), mlp(F.rms_norm(x, (64,), w, EPS)))


@pytest.mark.gpu
def test_generic_kernels_in_evaluation(monkeypatch):
    """BITTORCH_KERNEL=generic: the layers one by one, kept weights or not."""
    announce("gated mlp, generic kernels")
    mlp = _mlp(64, 48, seed=20, bias=True).cuda()
    x = torch.randn(5, 64, device="cuda")
    with torch.no_grad():
        kept = mlp.hidden(x)
        monkeypatch.setenv("BITTORCH_KERNEL", "generic")
        from bittorch_amd import _C
        monkeypatch.setattr(_C, "ternary_linear_tiled_forward", None)
        got = mlp.hidden(x)
        assert torch.equal(got, F.silu(mlp.gate(x)) * mlp.up(x)) and _norm_error(got, kept) <= 1e-5


@pytest.mark.gpu
def test_kept_weights_are_replaced_as_one():
    """Whatever another thread reads in between, the weights it finds kept are those that the key beside them stands for."""
    announce("kept weights, replaced as one")
    from bittorch_amd.nn._packed_cache import PackedWeightCache
    values = {}

    class Watched(PackedWeightCache):
        __slots__ = ()

        def __setattr__(self, name, value):
            super().__setattr__(name, value)
            if getattr(self, "key", None) is not None:
                assert self.value is values[self.key[0]]  # (by the weight's version)

        def _pack(self, weight, *settings):
            values[weight._version] = super()._pack(weight, *settings)
            return values[weight._version]

    cache, weight = Watched(), torch.nn.Parameter(torch.randn(48, 64, device="cuda"))
    for n in range(3):
        with torch.no_grad():
            weight.mul_(-1.0)
        assert cache.get(weight, 0.05, True) is cache.get(weight, 0.05, True) is values[weight._version]
