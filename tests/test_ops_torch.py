"""The policy-head operators (factory_marl_amd/ops.py) as torch reaches them other than by a plain call, on the CPU backend:
hooks on what a graph keeps, tracing, direct calls of the registered operators."""
import pytest
import torch

import ops_cases as cases
from factory_marl_amd import ops

CPU = torch.device("cpu")


def inputs(device=CPU):
    x, w, b, dy = cases.norm_inputs(4, 6, torch.float32, torch.float32, device)
    z, at, t, g = cases.distill_inputs(4, 6, 3, torch.float32, device)
    return x, w, b, dy, z, at, t, g


def gradients(x, w, b, dy, z, at, t, g):
    """(dx, dweight, dbias) of the layer norm, (dlogits) of the distillation"""
    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    y = ops.layer_norm(*leaves)
    leaf = z.clone().requires_grad_()
    loss = ops.distill_loss(leaf, at, t, temperature=1.5)
    return [*torch.autograd.grad(y, leaves, dy), *torch.autograd.grad(loss, leaf, g)]


# ------------------------------------------------------------------ hooks on saved tensors
def transposed(t):
    """the same values, columns not adjacent"""
    return t.t().contiguous().t() if t.dim() == 2 else torch.stack([t, t], 1)[:, 0]


@pytest.mark.parametrize("layout", [transposed, lambda t: t.clone(), lambda t: torch.stack([t] * 3, -1)[..., 1]])
def test_unpacked_tensors_may_have_any_layout(layout):
    want = gradients(*inputs())
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), layout):
        got = gradients(*inputs())
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_unpacked_tensors_of_equal_values_may_be_expanded():
    x, w, b, dy, z, at, t, g = inputs()
    args = (torch.full_like(x, 0.5), torch.full_like(w, 2.0), b, dy, torch.full_like(z, 0.25), torch.full_like(at, 1), torch.full_like(t, 3.0), g)
    want = gradients(*args)
    with torch.autograd.graph.saved_tensors_hooks(lambda v: v.detach(), lambda v: v.reshape(-1)[0].clone().expand(v.shape) if v.unique().numel() == 1 else v):
        got = gradients(*args)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("change", [lambda t: t[:-1], lambda t: t[..., :-1], lambda t: t.double(), lambda t: t.to("meta"), lambda t: t.new_empty(0)])
def test_other_tensors_unpacked_are_refused(change):
    x, w, b, dy, z, at, t, g = inputs()
    for which in range(7):  # each kept tensor in turn: x, weight, statistics; logits, indices, teacher's logits, statistics
        seen = []

        def unpack(v):
            seen.append(v)
            return change(v) if len(seen) - 1 == which else v

        with torch.autograd.graph.saved_tensors_hooks(lambda v: v, unpack):
            y = ops.layer_norm(x.clone().requires_grad_(), w, b)
            loss = ops.distill_loss(z.clone().requires_grad_(), at, t)
            with pytest.raises(RuntimeError, match="kept for the backward pass"):
                y.backward(dy)
                loss.backward(g)


# ------------------------------------------------------------------ tracing
def _bias_gradient(x, w, b, dy, z, at, t, g):
    leaf = b.clone().requires_grad_()
    return torch.autograd.grad(ops.layer_norm(x, None, leaf), leaf, dy)


CALLS = {
    "layer_norm": lambda x, w, b, dy, z, at, t, g: ops.layer_norm(x, w, b),
    "layer_norm without parameters": lambda x, w, b, dy, z, at, t, g: ops.layer_norm(x[:, None, 1:]),
    "sample_logits": lambda x, w, b, dy, z, at, t, g: ops.sample_logits(z, g.abs() % 1, top_p=0.9, top_k=g.long().abs() + 1),
    "sample_logits, mask": lambda x, w, b, dy, z, at, t, g: ops.sample_logits(z, g.abs() % 1, mask=b > 0),
    "distill_loss": lambda x, w, b, dy, z, at, t, g: ops.distill_loss(z, at, t, temperature=2.0),
    "gradients": gradients,
    "bias only": _bias_gradient,
}


def same(a, b):
    a, b = ([v] if torch.is_tensor(v) else list(v) for v in (a, b))
    return len(a) == len(b) and all(p.dtype == q.dtype and torch.equal(p, q) for p, q in zip(a, b))


def other_inputs(device=CPU):
    x, w, b, dy, z, at, t, g = inputs(device)
    return x.flip(0) + 1, w.flip(0), b.flip(0) - 0.1, dy.flip(1), z.flip(1) * 2, at.flip(0), t.flip(1), g.flip(0)


@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
@pytest.mark.parametrize("call", list(CALLS))
def test_traced_calls_compute_what_they_recorded(call, mode):
    """a recorded graph holds the operators: on new inputs it gives what a call gives"""
    from torch.fx.experimental.proxy_tensor import make_fx

    graph = make_fx(CALLS[call], tracing_mode=mode)(*inputs())
    assert any("factorysim" in str(n.target) for n in graph.graph.nodes)
    for args in (inputs(), other_inputs()):
        assert same(graph(*args), CALLS[call](*args))


@pytest.mark.parametrize("call", ["layer_norm", "layer_norm without parameters", "distill_loss"])
def test_traced_graphs_are_differentiable_again(call):
    from torch.fx.experimental.proxy_tensor import make_fx

    graph = make_fx(CALLS[call])(*inputs())
    args, again = list(inputs()), list(inputs())
    for a in (args, again):
        for i in (0, 1, 2, 4):
            a[i].requires_grad_()
    out, want = graph(*args), CALLS[call](*again)
    out.sum().backward(), want.sum().backward()
    for a, b in zip(args, again):
        assert (a.grad is None) == (b.grad is None) and (a.grad is None or torch.equal(a.grad, b.grad))


@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_calls(dynamic):
    torch._dynamo.reset()

    def step(x, w, b, z, at, t, u):
        y = ops.layer_norm(x, w, b)
        return y.tanh(), ops.distill_loss(z + y, at, t, temperature=2.0), ops.sample_logits(z, u, top_p=0.9)

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    for rows in (4, 3):
        results = []
        for f in (step, compiled):
            x, w, b, _, z, at, t, g = inputs()
            leaves = [v[:rows].clone().requires_grad_() for v in (x, z)] + [v.clone().requires_grad_() for v in (w, b)]
            y, loss, token = f(leaves[0], leaves[2], leaves[3], leaves[1], at[:rows], t[:rows], g[:rows].abs() % 1)
            results.append([y.detach(), loss.detach(), token, *torch.autograd.grad((y.sum(1) * loss).sum(), leaves)])
        assert same(*results)


def test_a_compiled_call_may_be_the_first_one(monkeypatch):
    torch._dynamo.reset()
    monkeypatch.setattr(ops, "_loaded", None)  # as before anything was called
    x = inputs()[0]
    assert torch.equal(torch.compile(lambda v: ops.layer_norm(v), backend="eager", fullgraph=True)(x), ops.layer_norm(x))


def test_registrations():
    """torch's own check of an operator: schema, gradients, shapes without data, tracing"""
    x, w, b, dy, z, at, t, g = inputs()
    ops._library()
    f = torch.ops.factorysim
    for grad in (False, True):
        xs, ws, bs, zs = (v.clone().requires_grad_(grad) for v in (x, w, b, z))
        torch.library.opcheck(f.layer_norm.default, (xs, ws, bs, 1e-5))
        torch.library.opcheck(f.layer_norm.default, (xs, None, None, 1e-5))
        torch.library.opcheck(f.distill_loss.default, (zs, at, t, 1.5))
        torch.library.opcheck(f.sample_logits.default, (zs, g.abs() % 1, None, 1.0, 0, 0.9, 0.0, None, None, None, None))


def test_function_transforms():
    x, w, b, dy, z, at, t, g = inputs()
    a = x.clone().requires_grad_()
    want, = torch.autograd.grad((ops.layer_norm(a, w, b) * dy).sum(), a)
    assert torch.equal(torch.func.grad(lambda v: (ops.layer_norm(v, w, b) * dy).sum())(x), want)
    stack = torch.stack([x, x + 1, 2 * x])
    assert torch.equal(torch.func.vmap(lambda v: ops.layer_norm(v, w, b))(stack), ops.layer_norm(stack, w, b))
    assert torch.equal(torch.func.vmap(lambda v: ops.distill_loss(v, at, t))(stack), torch.stack([ops.distill_loss(v, at, t) for v in stack]))


# ------------------------------------------------------------------ the registered operators, called directly
def test_direct_calls_are_checked():
    """whatever would be read or written past its end, or on another device, is refused"""
    x, w, b, dy, z, at, t, g = inputs()
    ops._library()
    f = torch.ops.factorysim
    u, stats, dstats = g.abs() % 1, torch.rand(2, 4), torch.rand(4, 2)
    calls = [
        (f.layer_norm, [x, w, b, 1e-5]), (f.layer_norm_stats, [x, w, b, 1e-5]),
        (f.layer_norm_backward, [dy, x, w, stats, torch.float32, [True] * 3]),
        (f.distill_loss, [z, at, t, 1.0]), (f.distill_loss_stats, [z, at, t, 1.0]), (f.distill_backward, [g, z, at, t, dstats, 1.0]),
        (f.sample_logits, [z, u, z > 0, 1.0, 0, 1.0, 0.0, u, at[:, 0].int(), u, u]),
    ]
    for op, args in calls:
        op(*args)
        for i, a in enumerate(args):
            if not torch.is_tensor(a):
                continue
            for bad in (a[:-1], a[..., :-1], a[None], a.reshape(-1), a.to(torch.float64 if a.dtype != torch.float64 else torch.float32),
                        a.to(torch.complex64), a.new_empty(0)):
                if bad.shape == a.shape and (bad.dtype == a.dtype or op is f.sample_logits and i == 1):
                    continue
                if op in (f.layer_norm, f.layer_norm_stats) and a is x and bad.shape == (3, 6) or \
                        op in (f.distill_loss, f.distill_loss_stats, f.distill_backward) and a is z and bad.shape == (4, 5):
                    continue  # fewer rows or columns: this argument alone says how many
                with pytest.raises((RuntimeError, TypeError)):
                    op(*args[:i], bad, *args[i + 1:])
    for args in ([x.half(), w, b.half(), 1e-5], [x.half(), w.bfloat16(), None, 1e-5], [x[:, :0], None, None, 1e-5]):
        with pytest.raises((RuntimeError, TypeError)):
            f.layer_norm(*args)
    with pytest.raises(TypeError):
        f.layer_norm_backward(dy, x, w, stats, torch.float16, [True] * 3)
    broad = f.sample_logits(z, u, (z > 0)[:1], 1.0, 0, 1.0, 0.0, None, None, None, None)  # one row of a mask for all
    assert torch.equal(broad, ops.sample_logits(z, u, mask=(z > 0)[0]))


def test_a_teacher_that_wants_a_gradient_is_refused_directly_too():
    ops._library()
    _, _, _, _, z, at, t, _ = inputs()
    for op in (torch.ops.factorysim.distill_loss, torch.ops.factorysim.distill_loss_stats):
        for leaf in (z.clone().requires_grad_(), z):
            with pytest.raises(RuntimeError, match="detach"):
                op(leaf, at, t.clone().requires_grad_(), 1.0)
        with torch.no_grad():
            op(z, at, t.clone().requires_grad_(), 1.0)


def test_the_entry_points_are_no_operator():
    ops._library()
    with pytest.raises(AttributeError):
        torch.ops.factorysim.bind


# ------------------------------------------------------------------ graphs used more than once
def test_graphs_kept_changed_and_differentiated_again():
    x, w, b, dy, z, at, t, g = inputs()
    for leaf, call, seed in ((x, lambda v: ops.layer_norm(v, w, b), dy), (z, lambda v: ops.distill_loss(v, at, t), g)):
        a = leaf.clone().requires_grad_()
        y = call(a)
        first, = torch.autograd.grad(y, a, seed, retain_graph=True)
        second, = torch.autograd.grad(y, a, seed)
        assert torch.equal(first, second)
        with pytest.raises(RuntimeError, match="second time"):
            torch.autograd.grad(y, a, seed)
        y = call(a)
        with torch.no_grad():
            a.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(y, a, seed)
        again, = torch.autograd.grad(call(a), a, seed, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            again.sum().backward()
