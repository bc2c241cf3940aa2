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
