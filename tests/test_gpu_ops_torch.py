"""The policy-head operators (factory_marl_amd/ops.py) on the GPU as torch reaches them other than by a plain call: hooks on
what a graph keeps, tracing, compiled calls (tests/test_ops_torch.py holds the CPU backend to the same and more)."""
import pytest

torch = pytest.importorskip("torch")
import test_ops_torch as plain  # noqa: E402
from factory_marl_amd import ops  # noqa: E402

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs an MI355X")]
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("layout", [plain.transposed, lambda t: torch.stack([t] * 3, -1)[..., 1]])
def test_unpacked_tensors_may_have_any_layout(layout):
    want = plain.gradients(*plain.inputs(DEV))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.detach(), layout):
        got = plain.gradients(*plain.inputs(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.autograd.graph.save_on_cpu():
        got = plain.gradients(*plain.inputs(DEV))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("mode", ["real", "symbolic"])
@pytest.mark.parametrize("call", list(plain.CALLS))
def test_traced_calls_compute_what_they_recorded(call, mode):
    from torch.fx.experimental.proxy_tensor import make_fx

    graph = make_fx(plain.CALLS[call], tracing_mode=mode)(*plain.inputs(DEV))
    for args in (plain.inputs(DEV), plain.other_inputs(DEV)):
        assert plain.same(graph(*args), plain.CALLS[call](*args))


def test_compiled_calls():
    torch._dynamo.reset()

    def step(x, w, b, z, at, t, u):
        y = ops.layer_norm(x, w, b)
        return y.tanh(), ops.distill_loss(z + y, at, t, temperature=2.0), ops.sample_logits(z, u, top_p=0.9)

    results = []
    for f in (step, torch.compile(step, backend="aot_eager", fullgraph=True)):
        x, w, b, _, z, at, t, g = plain.inputs(DEV)
        leaves = [v.clone().requires_grad_() for v in (x, z, w, b)]
        y, loss, token = f(leaves[0], leaves[2], leaves[3], leaves[1], at, t, g.abs() % 1)
        results.append([y.detach(), loss.detach(), token, *torch.autograd.grad((y.sum(1) * loss).sum(), leaves)])
    assert plain.same(*results)
