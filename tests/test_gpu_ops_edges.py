"""The policy-head operators (factory_marl_amd/ops.py) on the GPU at the ends of their ranges: the widest rows, block shapes
that go on to later rows, draws exactly on a border."""
import pytest

torch = pytest.importorskip("torch")
import ops_cases as cases  # noqa: E402
from factory_marl_amd import ops  # noqa: E402

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs an MI355X")]
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("cols", [2**27 + 5, 2**28])
def test_parameter_gradients_of_the_widest_rows(cols):
    """One row: dbias is dy, dweight is dy h.  A thread adds up cols / 1024 elements one after the other and 10 + 4 sums of
    those follow, so the mean is off by at most cols / 1024 + 14 roundings of mean |x|, the variance (and half of that 1 /
    deviation) by as many of itself; dy h is rounded to float16."""
    g = torch.Generator(device=DEV).manual_seed(cols)
    x, dy = (torch.randn(1, cols, device=DEV, dtype=torch.float16, generator=g) for _ in range(2))
    w, b = (torch.zeros(cols, device=DEV, dtype=torch.float16).requires_grad_() for _ in range(2))
    dw, db = torch.autograd.grad(ops.layer_norm(x, w, b), (w, b), dy)
    assert torch.equal(db, dy[0])
    var, mean = torch.var_mean(x.double(), unbiased=False)
    size = x.double().abs().mean() * torch.rsqrt(var + 1e-5)
    lost = (cols / 1024 + 14) * cases.E32
    for part in range(0, cols, 1 << 24):
        at = slice(part, min(part + (1 << 24), cols))
        h = (x[0, at].double() - mean) * torch.rsqrt(var + 1e-5)
        want, slack = dy[0, at].double() * h, dy[0, at].double().abs() * lost * (size + h.abs())
        assert ((dw[at].double() - want).abs() <= slack + 2.0**-11 * (want.abs() + slack) + 2.0**-25).all()
