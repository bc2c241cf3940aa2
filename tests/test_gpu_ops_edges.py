"""The policy-head operators (factory_marl_amd/ops.py) on the GPU at the ends of their ranges: the widest rows, block shapes
that go on to later rows, draws exactly on a border."""
import pytest

torch = pytest.importorskip("torch")
import ops_cases as cases  # noqa: E402
import test_ops_edges as plain  # noqa: E402
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


@pytest.mark.parametrize("kind,cols", [("f32", 4100), ("f32", 8192), ("f32", 16383), ("f16", 8200), ("bf16", 16384)])
def test_norm_blocks_of_512_and_1024_threads_go_on_to_later_rows(kind, cols):
    """a row a block of one CU: with 300 rows some blocks take two, one with and one without a row to follow"""
    t = cases.DTYPES[kind]
    cases.check_norm(*cases.norm_inputs(300, cols, t, t, DEV))


def test_norm_wide_rows_beyond_the_sums_of_one_stretch():
    """more than 16 rows a stretch of the parameters' sums, and more rows than one a block"""
    cases.check_norm(*cases.norm_inputs(600, 16400, torch.bfloat16, torch.float32, DEV))


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("rows,cols", [(200, 1500), (200, 2100), (200, 9001), (1100, 5003), (100, 70001)])
def test_draws_exactly_on_the_borders_of_equal_logits(rows, cols, kind):
    """256 equal logits, whatever they are, and nothing else that weighs: u = k / 256 draws the k-th of them, and of the half
    that top_p = 0.5 keeps u = k / 128 (the first up to which MORE than u of the weight lies); top_p = n / 256 keeps n"""
    g = torch.Generator().manual_seed(cols)
    for rest in (-float("inf"), -1e4):
        at = torch.stack([torch.randperm(cols, generator=g)[:256] for _ in range(rows)]).sort(1).values
        value = torch.cat([1e-3 * torch.randn(rows // 2, generator=g), 10 * torch.randn(rows - rows // 2, generator=g)])
        z = torch.full((rows, cols), rest).scatter_(1, at, value[:, None].expand(rows, 256)).to(DEV, cases.DTYPES[kind])
        k = torch.randint(0, 128, (rows,), generator=g)
        want = at.gather(1, k[:, None])[:, 0]
        for settings, parts in ((dict(), 256), (dict(top_p=0.5), 128), (dict(min_p=1.0), 256), (dict(top_k=128), 128), (dict(temperature=0.3), 256)):
            got = ops.sample_logits(z, (k / parts).to(DEV), **settings)
            assert torch.equal(got.cpu(), want), (rest, settings, int((got.cpu() != want).sum()))
        for p in (0.25, 0.5, 0.75):  # the last one kept
            got = ops.sample_logits(z, torch.full((rows,), 1 - 2.0**-24, device=DEV), top_p=p).cpu()
            assert torch.equal(got, at[:, int(256 * p) - 1]), (rest, p, int((got != at[:, int(256 * p) - 1]).sum()))
        mask = torch.zeros(rows, cols, dtype=torch.bool).scatter_(1, at, True)
        got = ops.sample_logits(value[:, None].expand(rows, cols).contiguous().to(DEV, cases.DTYPES[kind]), (k / 256).to(DEV), mask=mask.to(DEV))
        assert torch.equal(got.cpu(), want)


def milliseconds(call):
    """the shortest of several runs of 5"""
    call()
    times = []
    for _ in range(8):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(5):
            call()
        b.record()
        torch.cuda.synchronize(DEV)
        times.append(a.elapsed_time(b) / 5)
    return min(times)


@pytest.mark.parametrize("rows,cols,spread,settings", [(1, 32768, 1.0, dict(temperature=2.0, min_p=0.001)), (64, 131072, 0.2, dict(min_p=0.05)),
                                                       (64, 131072, 0.2, dict(min_p=0.05, top_p=0.9)), (64, 50021, 1.0, dict(min_p=1e-9, top_k=3000))])
def test_min_p_that_cuts_nothing_costs_little(rows, cols, spread, settings):
    """its border lies below every category: no list is made of it, let alone the search digit by digit that an endless list
    ends in (some ten times as long).  Draws are those without it."""
    g = torch.Generator().manual_seed(cols)
    z = (spread * torch.randn(rows, cols, generator=g)).to(DEV)
    u = torch.rand(rows, generator=g).to(DEV)
    without = {k: v for k, v in settings.items() if k != "min_p"}
    cases.check_sample(z[:4], u[:4], **settings)
    assert torch.equal(ops.sample_logits(z, u, **settings), ops.sample_logits(z, u, **without))
    slow, base = milliseconds(lambda: ops.sample_logits(z, u, **settings)), milliseconds(lambda: ops.sample_logits(z, u, **without))
    assert slow < 2 * base, (slow, base)


def test_draws_below_the_steps():
    """logits far apart after a stretch of close ones: borders and draws among those that lie below all steps, few (one list)
    or many of them"""
    g = torch.Generator().manual_seed(11)
    for cols, low in ((9001, 1500), (9001, 4500), (70001, 1900), (70001, 35000)):
        z = 1e-3 * torch.randn(6, cols, generator=g)
        z[:, cols - low:] -= 0.3 + 3 * torch.rand(6, low, generator=g)
        for t in (z, z.bfloat16()):
            for u in (0.3, 0.7, 0.95, 0.9999):
                for settings in (dict(), dict(top_p=0.9), dict(min_p=0.3), dict(min_p=0.3, top_p=0.8), dict(top_k=cols - 700), dict(top_k=cols - 700, min_p=0.01)):
                    cases.check_sample(t.to(DEV), torch.full((6,), u, device=DEV), **settings)


@pytest.mark.parametrize("cols", [2, 50, 700, 5003, 70001])
def test_settings_and_logits_that_are_no_numbers_leave_other_rows_alone(cols):
    """NaN and infinities among u, the settings and the logits, above and below the first vectors' largest"""
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(cols)
    z, u = 3 * torch.randn(40, cols, generator=g), torch.rand(40, generator=g)
    p = torch.full((40,), 0.9)
    z[1, -1], z[2, 0], z[3, cols // 2], z[4, -1], u[5], p[6] = nan, nan, inf, -inf, nan, nan
    z[7, 1:] = -inf
    z[8, -1] = 3e38
    z[9] = -3e38
    z[9, cols // 3] = 3e38
    barred = torch.ones(40, cols, dtype=torch.bool)
    barred[10, 0] = False
    z[10, 0] = nan
    got = cases.check_sample(z.to(DEV), u.to(DEV), mask=barred.to(DEV), top_p=p.to(DEV))
    assert got[1] == got[2] == got[5] == got[6] == -1 and (got[[3, 4, 7, 8, 9]] >= 0).all()


def test_rows_of_the_student_without_a_softmax():
    plain.check_softmaxless(DEV)


@pytest.mark.parametrize("rows,cols", [(300, 5), (300, 128), (50, 1001), (30, 9000), (20, 20000)])
def test_norm_gradients_wanted_in_part(rows, cols):
    """each gradient alone, or two of them, has the bits that it has among all three"""
    x, w, b, dy = cases.norm_inputs(rows, cols, torch.bfloat16, torch.float32, DEV)
    full = torch.autograd.grad(ops.layer_norm(*(leaves := [v.clone().requires_grad_() for v in (x, w, b)])), leaves, dy)
    for wanted in ((0,), (1,), (2,), (0, 1), (0, 2), (1, 2)):
        args = [v.clone().requires_grad_(i in wanted) for i, v in enumerate((x, w, b))]
        got = torch.autograd.grad(ops.layer_norm(*args), [args[i] for i in wanted], dy)
        assert all(torch.equal(a, full[i]) for a, i in zip(got, wanted)), wanted
