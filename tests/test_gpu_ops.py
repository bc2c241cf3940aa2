"""The policy-head operators (factory_marl_amd/ops.py) on the GPU, against the float64 statements of ops_reference.py:
sizes from one element up, odd and unaligned rows, long strides, masks, streams, graphs, and a run of them together."""
import json
import os

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import ops_cases as cases  # noqa: E402
from factory_marl_amd import _lib, ops  # noqa: E402

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs an MI355X")]
DEV = torch.device("cuda", 0)
KINDS = ["f32", "f16", "bf16"]


# ------------------------------------------------------------------ layer norm
@pytest.mark.parametrize("kind,param", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 2), (130, 5), (7, 16), (300, 63), (65, 64), (66, 65), (1000, 128), (37, 130), (9, 257),
                                       (33, 512), (5, 1001), (18, 1024), (4, 2047), (3, 4096), (5, 5003), (2, 8192), (3, 16384), (2, 16391), (3, 40001)])
def test_norm(rows, cols, kind, param):
    cases.check_norm(*cases.norm_inputs(rows, cols, cases.DTYPES[kind], cases.DTYPES[param], DEV))


@pytest.mark.parametrize("cols", [1, 2, 17, 128, 1000, 9000])
def test_norm_many_rows(cols):
    cases.check_norm(*cases.norm_inputs(max(3, 3_000_000 // cols // 8), cols, torch.float32, torch.float32, DEV))


@pytest.mark.parametrize("kind", KINDS)
def test_norm_optional_parameters_and_strided_rows(kind):
    t = cases.DTYPES[kind]
    for cols in (40, 128, 1001, 3000, 17000):
        x, w, b, dy = cases.norm_inputs(6, cols, t, t, DEV)
        cases.check_norm(x, None, None, dy)
        cases.check_norm(x, w, None, dy)
        cases.check_norm(x, None, b, dy)
        cases.check_norm(x.view(2, 3, cols), w, b, dy.view(2, 3, cols))
        wide = cases.norm_inputs(6, cols + 9, t, t, DEV, seed=1)
        for o in (1, 3, 8):  # rows at every alignment, parameters and gradients too
            cases.check_norm(wide[0][:, o:o + cols], wide[1][o:o + cols], wide[2][o:o + cols], wide[3][:, 9 - o:9 - o + cols])
        cases.check_norm(x[:1].expand(6, cols), w, b, dy[:1].expand(6, cols))  # every row the same memory
        cases.check_norm(x.t().contiguous().t(), w, b, dy)


def test_norm_large_mean_constant_rows_and_non_finite_values():
    x, w, b, dy = cases.norm_inputs(8, 512, torch.float32, torch.float32, DEV, offset=100.0)
    cases.check_norm(x, w, b, dy)
    x[2] = 3.0  # variance 0: rstd = 1 / sqrt(eps)
    cases.check_norm(x, w, b, dy)
    clean = ops.layer_norm(x, w, b)
    x[5, 7] = float("nan")
    x[6, 0] = float("inf")
    y = ops.layer_norm(x, w, b)
    others = [0, 1, 2, 3, 4, 7]
    assert y[5].isnan().all() and y[6].isnan().any() and torch.equal(y[others], clean[others])


def test_norm_rows_far_apart():
    """row offsets past 2^32 elements"""
    stride = 2**31 + 5
    big = torch.empty(2 * stride + 300, dtype=torch.float16, device=DEV)
    x = torch.as_strided(big, (3, 300), (stride, 1))
    small = cases.norm_inputs(3, 300, torch.float16, torch.float32, DEV)
    x.copy_(small[0])
    y, grads = cases.check_norm(x, *small[1:])
    y2, grads2 = cases.check_norm(*small)
    assert torch.equal(y, y2) and all(torch.equal(a, b) for a, b in zip(grads, grads2))


def test_norm_writes_its_rows_and_nothing_else():
    """guard elements before and behind every output of the C entry points"""
    L = _lib.load()
    for cols in (1, 5, 128, 1001, 4096, 20000):
        n = 5
        x, w, b, dy = cases.norm_inputs(n, cols, torch.bfloat16, torch.bfloat16, DEV)

        def guarded(count, dtype):
            return torch.full((count + 128,), 7.0, dtype=dtype, device=DEV)

        y, dx = guarded(n * cols, torch.bfloat16), guarded(n * cols, torch.bfloat16)
        dw, db = guarded(cols, torch.bfloat16), guarded(cols, torch.bfloat16)
        mean, rstd = guarded(n, torch.float32), guarded(n, torch.float32)
        need = L.fm_layer_norm_workspace(n, cols)
        work = torch.full((need + 256,), 9, dtype=torch.uint8, device=DEV)
        s = torch.cuda.current_stream(DEV).cuda_stream
        a = _lib.FmLayerNormArgs(0, 2, 2, 0, n, cols, x.data_ptr(), cols, w.data_ptr(), b.data_ptr(), 1e-5, y.data_ptr() + 128, mean.data_ptr() + 256,
                                 rstd.data_ptr() + 256, dy.data_ptr(), cols, dx.data_ptr() + 128, dw.data_ptr() + 128, db.data_ptr() + 128,
                                 work.data_ptr(), need, s)
        _lib.check(L.fm_layer_norm_forward(a), L)
        _lib.check(L.fm_layer_norm_backward(a), L)
        for t, count in ((y, n * cols), (dx, n * cols), (dw, cols), (db, cols), (mean, n), (rstd, n)):
            assert (t[:64] == 7).all() and (t[64 + count:] == 7).all()
        assert (work[need:] == 9).all()
        assert torch.equal(y[64:64 + n * cols].view(n, cols), ops.layer_norm(x, w, b))


def test_norm_same_bits_every_time():
    for rows, cols in ((8192, 128), (300, 5000), (77, 20000)):
        x, w, b, dy = cases.norm_inputs(rows, cols, torch.bfloat16, torch.float32, DEV)
        first = None
        for _ in range(3):
            leaves = [t.clone().requires_grad_() for t in (x, w, b)]
            got = torch.autograd.grad(ops.layer_norm(*leaves), leaves, dy)
            assert first is None or all(torch.equal(p, q) for p, q in zip(first, got))
            first = got


# ------------------------------------------------------------------ drawing categories
SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.0),
            dict(temperature=1.4, top_k=12, top_p=0.9, min_p=0.05), dict(top_k=2500), dict(top_k=2500, top_p=0.97), dict(top_p=0.0),
            dict(min_p=1.5), dict(temperature=1e-30), dict(temperature=float("inf")), dict(temperature=50.0, top_p=0.999, min_p=1e-4)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("settings", SETTINGS)
def test_sample(settings, kind):
    g = torch.Generator().manual_seed(1)
    for rows, cols in [(300, 1), (500, 2), (200, 3), (60, 7), (40, 33), (30, 64), (20, 65), (9, 129), (9, 600), (6, 1500), (5, 2048), (4, 2049), (3, 5003), (2, 20011)]:
        z = (torch.randn(rows, cols, generator=g) * 2).to(cases.DTYPES[kind]).to(DEV)
        cases.check_sample(z, torch.rand(rows, generator=g).to(DEV), **settings)
        cases.check_sample(z, torch.rand(rows, generator=g, dtype=torch.float64).to(DEV), mask=(torch.rand(rows, cols, generator=g) < 0.7).to(DEV), **settings)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("cols", [50021, 131072, 300007])
def test_sample_long_rows(cols, kind):
    """peaked, ordinary and flat rows, and rows of few distinct values"""
    g = torch.Generator().manual_seed(cols)
    for scale in (0.0, 0.02, 1.0, 3.0, 30.0):
        z = torch.randn(4, cols, generator=g) * scale
        if scale == 30.0:
            z = z.round()
        z = z.to(cases.DTYPES[kind]).to(DEV)
        u = torch.rand(4, generator=g).to(DEV)
        for settings in (dict(), dict(top_p=0.9), dict(top_k=50, top_p=0.95, temperature=0.7), dict(top_k=cols // 2, top_p=0.99), dict(min_p=0.01),
                         dict(top_k=7000), dict(temperature=0.0)):
            cases.check_sample(z, u, **settings)
        cases.check_sample(z, u, mask=(torch.rand(4, cols, generator=g) < 0.5).to(DEV), top_p=0.8)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols", [(5, 2500), (5, 9001), (1100, 5001), (4, 70003)])
def test_sample_rows_that_long_rows_kernels_treat_apart(rows, cols, kind):
    """where the first vectors of a row say little or the wrong thing about it: the largest logits at its end, nothing open at
    its start, few categories open at all, logits wider or closer than a step, one value throughout, infinities"""
    g = torch.Generator().manual_seed(cols)
    some = [0, rows // 2, rows - 1]

    def check(z, mask=None, settings=(dict(), dict(top_p=0.9), dict(top_k=30, top_p=0.8), dict(min_p=0.1), dict(top_k=3000, top_p=0.99, min_p=1e-5))):
        z, u = z.to(cases.DTYPES[kind]).to(DEV), torch.rand(rows, generator=g).to(DEV)
        mask = None if mask is None else mask.to(DEV)
        for s in settings:
            got = ops.sample_logits(z, u, mask=mask, **s)
            few = cases.check_sample(z[some], u[some], mask=None if mask is None else mask[some], **s)
            assert torch.equal(got[some], few)

    normal = torch.randn(rows, cols, generator=g)
    late = normal.clone()
    late[:, -7:] += 25
    check(late)
    late[:, -1] += 300
    check(late)
    bars = torch.ones(rows, cols, dtype=torch.bool)
    bars[:, : cols - 900] = False
    check(normal * 2, bars)  # nothing open where the steps begin
    check(normal * 2, torch.rand(rows, cols, generator=g) < 12 / cols)  # a handful of categories open
    one = torch.zeros(rows, cols, dtype=torch.bool)
    one[:, cols - 3] = True
    check(normal, one)
    check(normal * 60, settings=(dict(), dict(top_k=50, temperature=0.7), dict(top_k=2000), dict(temperature=1e-6)))
    check(normal * 1e-4, settings=(dict(), dict(top_p=0.5), dict(temperature=1e-4), dict(temperature=float("inf"), top_p=0.9)))
    check(normal * 1e-3 + 900)
    check(torch.full((rows, cols), -3.0))
    infinite = normal.clone()
    infinite[:, cols // 2] = float("inf")
    infinite[:, 5] = -float("inf")
    check(infinite)


def edge_rows():
    inf, nan, low = float("inf"), float("nan"), torch.finfo(torch.float32).min
    z = torch.tensor([[1, 2, 3, 4], [-inf, -inf, -inf, -inf], [nan, inf, 0, 1], [nan, 1, 2, 3], [low, low, low, low],
                      [inf, 0, inf, 1], [-inf, 5, -inf, -inf], [0.0, -0.0, 0.0, -0.0], [2, 2, 2, 2], [low, 0, low, 0],
                      [1, 2, 3, 4], [inf, inf, -inf, nan]])
    mask = torch.ones(12, 4, dtype=torch.bool)
    mask[2, :2] = False
    mask[10] = False
    mask[11, 3] = False
    return z, mask, torch.linspace(0, 0.99, 12)


@pytest.mark.parametrize("settings", SETTINGS)
@pytest.mark.parametrize("repeat", [1, 25, 700, 16400])
def test_sample_edge_rows(settings, repeat):
    """masks that empty a row, NaN and infinities in barred places, the type's lowest value, ties: in rows of every
    length (the four values repeated)"""
    z, mask, u = (t.to(DEV) for t in edge_rows())
    z, mask = z.repeat(1, repeat), mask.repeat(1, repeat)
    got = cases.check_sample(z, u, mask=mask, **settings)
    assert got[1] == got[3] == got[10] == -1


@pytest.mark.parametrize("cols", [2, 40, 1000, 3000, 60000])
def test_sample_settings_of_each_row(cols):
    g = torch.Generator().manual_seed(2)
    n = 24
    z = (torch.randn(n, cols, generator=g) * 2).to(DEV)
    sets = dict(temperature=torch.rand(n, generator=g) * 2, top_k=torch.randint(-1, 40, (n,), generator=g),
                top_p=torch.rand(n, generator=g) * 1.2, min_p=torch.rand(n, generator=g) * 0.3 - 0.05)
    sets["temperature"][3] = 0
    sets = {k: v.to(DEV) for k, v in sets.items()}
    u = torch.rand(n, generator=g).to(DEV)
    cases.check_sample(z, u, **sets)
    cases.check_sample(z.view(4, 6, cols), u.view(4, 6), mask=(torch.rand(cols, generator=g) < 0.6).to(DEV), **sets)
    for name in ("temperature", "top_p", "min_p"):
        bad = {**sets, name: sets[name].clone()}
        bad[name][5] = float("nan")
        got = ops.sample_logits(z, u, **bad)
        assert got[5] == -1
    u[7] = float("nan")
    assert ops.sample_logits(z, u, **sets)[7] == -1


def test_sample_strided_rows_and_rows_far_apart():
    g = torch.Generator().manual_seed(5)
    for cols in (2, 50, 900, 4001):
        wide = (torch.randn(6, cols + 7, generator=g) * 2).to(DEV)
        barred = (torch.rand(6, cols + 5, generator=g) < 0.8).to(DEV)
        u = torch.rand(6, generator=g).to(DEV)
        for o in (1, 3):
            for t in (wide, wide.bfloat16()):
                cases.check_sample(t[:, o:o + cols], u, mask=barred[:, o:o + cols], top_p=0.9)
        cases.check_sample(wide[:1, :cols].expand(6, cols), u, top_k=9)
    stride = 2**31 + 3
    big = torch.empty(2 * stride + 5000, dtype=torch.bfloat16, device=DEV)
    for cols in (40, 1000, 5000):
        z = torch.as_strided(big, (3, cols), (stride, 1))
        z.copy_((torch.randn(3, cols, generator=g) * 2).bfloat16())
        cases.check_sample(z, torch.rand(3, generator=g).to(DEV), top_p=0.9)


def test_sample_writes_its_rows_and_nothing_else():
    L = _lib.load()
    for rows, cols in ((5, 2), (7, 100), (3, 3000), (1, 70000), (300, 70000)):
        z, u = torch.randn(rows, cols, device=DEV), torch.rand(rows, device=DEV)
        out = torch.full((rows + 64,), 7, dtype=torch.int64, device=DEV)
        need = L.fm_sample_workspace(rows, cols)
        work = torch.full((need + 256,), 9, dtype=torch.uint8, device=DEV)
        for settings in (dict(top_p=0.8, top_k=0), dict(top_p=1.0, top_k=30), dict(top_p=1.0, top_k=0)):
            a = _lib.FmSampleArgs(device=0, rows=rows, cols=cols, logits=z.data_ptr(), stride=cols, u=u.data_ptr(), temperature=1.0,
                                  out=out.data_ptr() + 256, workspace=work.data_ptr(), workspace_bytes=need,
                                  stream=torch.cuda.current_stream(DEV).cuda_stream, **settings)
            _lib.check(L.fm_sample_logits(a), L)
            assert (out[:32] == 7).all() and (out[32 + rows:] == 7).all() and (work[need:] == 9).all()
            assert torch.equal(out[32:32 + rows], ops.sample_logits(z, u, **settings))


# ------------------------------------------------------------------ distillation
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (1000, 2, 2), (300, 5, 3), (77, 33, 5), (50, 64, 64), (20, 65, 65), (9, 300, 16), (7, 1000, 256),
                                         (5, 2001, 64), (3, 8192, 37), (4, 20011, 1024), (2, 131072, 100)])
def test_distill(rows, cols, k, kind):
    for padded, T, index in ((False, 1.0, torch.int64), (True, 2.5, torch.int32)):
        cases.check_distill(*cases.distill_inputs(rows, cols, k, cases.DTYPES[kind], DEV, padded=padded, index=index), temperature=T)


def test_distill_teacher_types_strides_and_shapes():
    for cols in (6, 700, 9001):
        z, at, t, g = cases.distill_inputs(6, cols, 5, torch.float32, DEV, padded=True)
        for dt in (torch.float16, torch.bfloat16):
            cases.check_distill(z.to(dt), at, t.to(dt), g)
            cases.check_distill(z, at, t.to(dt), g)
        cases.check_distill(z.view(2, 3, cols), at.view(2, 3, 5), t.view(2, 3, 5), g.view(2, 3))
        wide, _, _, _ = cases.distill_inputs(6, cols + 9, 5, torch.bfloat16, DEV)
        for o in (1, 4):
            cases.check_distill(wide[:, o:o + cols], at, t, g)
        two = torch.stack([at, at], 2)
        cases.check_distill(z[:1].expand(6, cols), two[:, :, 0], torch.stack([t, t], 2)[:, :, 1], g[:1].expand(6))
    loss = ops.distill_loss(z.requires_grad_(), at, t)
    a, = torch.autograd.grad(loss.mean(), z)  # the mean's gradient is one number spread over the rows
    cases.check_distill(z.detach(), at, t, torch.full((6,), 1 / 6, device=DEV))
    assert a.abs().max() > 0


@pytest.mark.parametrize("repeat", [1, 12, 130, 3000])
def test_distill_edges(repeat):
    """the same index twice, empty lists, masked students and teachers, an index that is none: in rows of every length"""
    inf = float("inf")
    z = torch.randn(7, 8 * repeat, generator=torch.Generator().manual_seed(3))
    z[3, :4] = -inf
    z[4] = torch.finfo(torch.float32).min
    at = torch.tensor([[3, 3, 1], [-1, -1, -1], [0, 7, -5], [7, 5, 4], [2, 2, 2], [6, 1, 6], [8 * repeat - 1, 0, 8 * repeat - 1]])
    t = torch.tensor([[1.0, 2.0, 0.5], [1.0, 2.0, 3.0], [-inf, 1.0, 9.0], [0.0, 1.0, 2.0], [1.0, 1.0, 1.0], [0.3, -inf, 0.1], [1.0, 2.0, 3.0]])
    g = torch.tensor([1.0, 2.0, -0.5, 0.25, 3.0, 0.0, 1.0])
    z, at, t, g = (v.to(DEV) for v in (z, at, t, g))
    loss, dz = cases.check_distill(z, at, t, g, temperature=1.5)
    assert loss[1] == 0 and not dz[1].any()
    at[0, 1] = 8 * repeat
    z[2, 7] = -inf  # a listed category that the student rules out
    t[4, 0] = float("nan")
    z.requires_grad_()
    loss = ops.distill_loss(z, at, t)
    dz, = torch.autograd.grad(loss.sum(), z)
    assert loss[0].isnan() and dz[0].isnan().all() and loss[4].isnan() and dz[4].isnan().all()
    assert loss[2] == inf and dz[2].isfinite().all() and loss[[1, 3, 5, 6]].isfinite().all() and dz[[1, 3, 5, 6]].isfinite().all()
    at[1, 0] = 2**31 + 5  # past 32 bits: still no category
    assert ops.distill_loss(z, at, t)[1].isnan()


def test_distill_rows_far_apart_and_guards():
    stride = 2**31 + 7
    big = torch.empty(2 * stride + 9000, dtype=torch.bfloat16, device=DEV)
    for cols in (30, 9000):
        z, at, t, g = cases.distill_inputs(3, cols, 7, torch.bfloat16, DEV)
        far = torch.as_strided(big, (3, cols), (stride, 1)).copy_(z)
        a, b = cases.check_distill(far, at, t, g), cases.check_distill(z, at, t, g)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    L = _lib.load()
    for rows, cols, k in ((5, 2, 2), (3, 700, 9), (2, 20000, 30), (1, 100000, 64)):
        z, at, t, g = cases.distill_inputs(rows, cols, k, torch.float32, DEV)
        loss, stats, dz = (torch.full((c + 128,), 7.0, device=DEV) for c in (rows, 2 * rows, rows * cols))
        need = L.fm_distill_workspace(rows, cols)
        work = torch.full((need + 256,), 9, dtype=torch.uint8, device=DEV)
        a = _lib.FmDistillArgs(0, 0, 5, 0, rows, cols, k, z.data_ptr(), cols, at.data_ptr(), k, t.data_ptr(), k, 1.0, loss.data_ptr() + 256,
                               stats.data_ptr() + 256, g.data_ptr(), 1, dz.data_ptr() + 256, work.data_ptr(), need,
                               torch.cuda.current_stream(DEV).cuda_stream)
        _lib.check(L.fm_distill_forward(a), L)
        _lib.check(L.fm_distill_backward(a), L)
        for v, count in ((loss, rows), (stats, 2 * rows), (dz, rows * cols)):
            assert (v[:64] == 7).all() and (v[64 + count:] == 7).all()
        assert (work[need:] == 9).all()


# ------------------------------------------------------------------ streams, graphs, together
def _all_three(s):
    y = ops.layer_norm(s["x"], s["w"], s["b"])
    token = ops.sample_logits(y, s["u"], temperature=0.8, top_k=50, top_p=0.9)
    loss = ops.distill_loss(y, s["at"], s["t"], temperature=1.5)
    dx, dw, db = torch.autograd.grad((loss * s["g"]).sum(), (s["x"], s["w"], s["b"]))
    return y.detach(), token, loss.detach(), dx, dw, db


def _state(rows, cols, seed=0):
    x, w, b, _ = cases.norm_inputs(rows, cols, torch.float32, torch.float32, DEV, seed=seed)
    _, at, t, g = cases.distill_inputs(rows, cols, min(20, cols), torch.float32, DEV, seed=seed)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(seed)).to(DEV)
    return dict(x=x.requires_grad_(), w=w.requires_grad_(), b=b.requires_grad_(), at=at, t=t, g=g, u=u)


@pytest.mark.parametrize("rows,cols", [(64, 2), (33, 100), (5, 3001), (2, 70001)])
def test_captured_together_and_replayed(rows, cols):
    """the three operators with both backward passes in one graph, and a second graph beside it: every replay on new
    inputs, with eager work and waits between, equals the eager result"""
    states = [_state(rows, cols, 0), _state(rows, cols, 1)]
    side = torch.cuda.Stream(DEV)
    graphs = []
    for s in states:
        side.wait_stream(torch.cuda.current_stream(DEV))
        with torch.cuda.stream(side):
            for _ in range(2):
                _all_three(s)
        torch.cuda.current_stream(DEV).wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _all_three(s)
        graphs.append((graph, s, out))
    for seed in range(2, 6):
        for i in (0, 1):
            new = _state(rows, cols, seed + 10 * i)
            with torch.no_grad():
                for k, v in graphs[i][1].items():
                    v.copy_(new[k])
        graphs[0][0].replay()
        graphs[1][0].replay()
        torch.cuda.synchronize(DEV)
        for i in (0, 1):
            want = _all_three(_state(rows, cols, seed + 10 * i))
            assert all(torch.equal(a, b) for a, b in zip(graphs[i][2], want)), (seed, i)


def test_two_streams_at_once():
    """the same calls on two streams, each with its own inputs, interleaved"""
    cells = [(64, 2), (300, 128), (4, 70001), (2, 131072)]
    want = [[t.clone() for t in _all_three(_state(r, c, 3))] for r, c in cells]
    streams = [torch.cuda.Stream(DEV) for _ in range(2)]
    states = [_state(r, c, 3) for r, c in cells]
    torch.cuda.synchronize(DEV)
    got = {}
    for turn in range(4):
        for i, s in enumerate(states):
            with torch.cuda.stream(streams[(i + turn) % 2]):
                got[turn, i] = _all_three(s)
    torch.cuda.synchronize(DEV)
    for (_, i), out in got.items():
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))


def test_more_rows_than_blocks_in_a_line_of_the_grid():
    """rows repeat a few kinds, whose results are those of a call with these few"""
    g = torch.Generator().manual_seed(41)
    for rows, cols in [(2**22 + 5, 64), (2**22 + 5, 65), (2**20 + 5, 2100)]:
        z = (2 * torch.randn(1, cols, generator=g)).to(DEV, torch.bfloat16)
        u, kind = torch.rand(1000, generator=g).to(DEV), torch.arange(rows, device=DEV) % 1000
        few = ops.sample_logits(z.expand(1000, cols), u, top_p=0.95)
        assert torch.equal(ops.sample_logits(z.expand(rows, cols), u[kind], top_p=0.95), few[kind])
    for rows, cols, k in [(2**22 + 5, 33, 2), (2**20 + 5, 3, 65)]:
        z, at = torch.randn(1000, cols, generator=g).to(DEV), torch.randint(cols, (1000, k), generator=g, dtype=torch.int32).to(DEV)
        t, kind = torch.randn(1, k, generator=g).to(DEV), torch.arange(rows, device=DEV) % 1000

        def run(z, at, t):
            z = z.requires_grad_()
            loss = ops.distill_loss(z, at, t, temperature=1.3)
            return (loss, *torch.autograd.grad(loss.sum(), z))

        few, all_rows = run(z, at, t.expand(1000, k)), run(z.detach()[kind], at[kind], t.expand(rows, k))
        assert all(torch.equal(b, a[kind]) for a, b in zip(few, all_rows))


def test_gpu_and_cpu_backends_agree():
    for rows, cols in ((40, 2), (9, 500), (3, 5000)):
        s = _state(rows, cols, 7)
        c = {k: (v.detach().cpu().requires_grad_() if v.requires_grad else v.cpu()) for k, v in s.items()}
        y = ops.layer_norm(s["x"], s["w"], s["b"]).detach()
        assert (y.cpu() - ops.layer_norm(c["x"], c["w"], c["b"])).abs().max() < 1e-4
        z = y.bfloat16()
        assert torch.equal(ops.sample_logits(z, s["u"], top_p=0.9).cpu(), ops.sample_logits(z.cpu(), c["u"], top_p=0.9))


def test_mixed_devices_are_refused():
    x = torch.randn(4, 8, device=DEV)
    with pytest.raises(ValueError):
        ops.layer_norm(x, torch.ones(8))
    with pytest.raises(ValueError):
        ops.sample_logits(x, torch.rand(4))
    with pytest.raises(ValueError):
        ops.distill_loss(x, torch.zeros(4, 1, dtype=torch.int64), torch.zeros(4, 1))


def test_saved_policy_teaches_a_normalised_student_on_the_gpu_env():
    """the reference's saved toggle policy as the teacher of a layer-normed student: rollouts on the GPU env by fused
    draws, the update with the distillation term; every figure finite, the teacher untouched"""
    from factory_marl_amd import FactoryVecEnv
    from factory_marl_amd.ppo import PPO, ActorCriticPolicy

    gold = os.path.join(os.path.dirname(os.path.abspath(__file__)), "golden")
    meta = json.load(open(os.path.join(gold, "policy_meta.json")))["y6lp1j7k"]
    kw = {k: v for k, v in meta["env_kwargs"].items() if k != "render_mode"}
    env = FactoryVecEnv(64, env_class=meta["env_class"], env_kwargs=kw)
    teacher = ActorCriticPolicy.for_env(env, net_arch=meta["net_arch"])
    teacher.load_state_dict({k: torch.as_tensor(v) for k, v in np.load(os.path.join(gold, "policy_y6lp1j7k.npz")).items()})
    ppo = PPO(env, policy_kwargs=dict(net_arch=(64, 64), layer_norm=True, fused_sampling=True), n_steps=4, batch_size=128, n_epochs=2, seed=0,
              teacher=teacher, distill_coef=1.0)
    before = [p.detach().clone() for p in teacher.parameters()]
    ppo.learn(64 * 4 * 2)
    assert all(np.isfinite(r[k]) for r in ppo.logs for k in ("policy_loss", "value_loss", "distill_loss"))
    assert all(torch.equal(a, b) for a, b in zip(before, teacher.parameters()))
    acts = ppo.policy.predict(env.obs, deterministic=False, temperature=0.5, top_p=0.9)
    assert set(acts.unique().tolist()) <= {0.0, 1.0}
    env.close()
