"""The policy-head operators (factory_marl_amd/ops.py) on the CPU backend: results, gradients, refusals, the C entry
points, and the policy and trainer options that call them."""
import ctypes as C

import numpy as np
import pytest
import torch

import ops_cases as cases
import ops_reference as ref
from factory_marl_amd import _lib, ops
from factory_marl_amd.ppo import PPO, ActorCriticPolicy
from test_ppo import ToyEnv

CPU = torch.device("cpu")


def test_reference_gradients_are_differences_of_the_reference():
    """the float64 statements' gradients against central differences of their values (step 1e-5: error ~1e-9)"""
    rng = np.random.default_rng(0)
    x, w, b, dy = rng.normal(size=(3, 7)), rng.normal(size=7), rng.normal(size=7), rng.normal(size=(3, 7))
    dx, dw, db = ref.layer_norm_backward(x, w, dy, 1e-5)

    def difference(f, a, i, h=1e-5):
        up, down = a.copy(), a.copy()
        up[i] += h
        down[i] -= h
        return (f(up) - f(down)) / (2 * h)

    for i in np.ndindex(*x.shape):
        assert abs(difference(lambda a: (ref.layer_norm(a, w, b, 1e-5)[0] * dy).sum(), x, i) - dx[i]) < 1e-7
    for j in range(7):
        assert abs(difference(lambda a: (ref.layer_norm(x, a, b, 1e-5)[0] * dy).sum(), w, j) - dw[j]) < 1e-7
        assert abs(difference(lambda a: (ref.layer_norm(x, w, a, 1e-5)[0] * dy).sum(), b, j) - db[j]) < 1e-7
    z, at, t, g = rng.normal(size=(2, 9)), np.array([[1, 4, -1], [8, 8, 0]]), rng.normal(size=(2, 3)), rng.normal(size=2)
    dz = ref.distill(z, at, t, 1.7, g)[1]
    for i in np.ndindex(*z.shape):
        assert abs(difference(lambda a: (ref.distill(a, at, t, 1.7) * g).sum(), z, i) - dz[i]) < 1e-7


# ------------------------------------------------------------------ layer norm
@pytest.mark.parametrize("kind,param", [("f32", "f32"), ("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("rows,cols", [(1, 1), (4, 2), (5, 63), (3, 130), (2, 1001)])
def test_norm(rows, cols, kind, param):
    cases.check_norm(*cases.norm_inputs(rows, cols, cases.DTYPES[kind], cases.DTYPES[param], CPU))


def test_norm_without_parameters_shapes_strides_and_no_rows():
    x, w, b, dy = cases.norm_inputs(6, 40, torch.float32, torch.float32, CPU)
    cases.check_norm(x, None, None, dy)
    cases.check_norm(x, w, None, dy)
    cases.check_norm(x, None, b, dy)
    cases.check_norm(x.view(2, 3, 40), w, b, dy.view(2, 3, 40))
    cases.check_norm(x[0], w, b, dy[0])
    wide = torch.randn(6, 100)
    cases.check_norm(wide[:, 7:47], w, b, dy)
    cases.check_norm(torch.randn(40, 6).t(), w, b, dy)
    y = ops.layer_norm(x[:0].requires_grad_(), w.requires_grad_(), b.requires_grad_())
    assert y.shape == (0, 40)
    gw, gb = torch.autograd.grad(y, (w, b), torch.empty(0, 40))
    assert not gw.any() and not gb.any()


def test_norm_against_differences_of_its_own_values():
    """central differences of the float32 forward pass: step 2^-6, so rounding of about 40 terms * 2^-24 / 2^-6 = 1e-4
    at most and curvature of about step^2 = 2.4e-4 times third derivatives of order one, summed over 12 columns"""
    x, w, b, dy = cases.norm_inputs(2, 12, torch.float32, torch.float32, CPU, offset=0.0)
    gx, gw, gb = torch.autograd.grad(ops.layer_norm(x.requires_grad_(), w.requires_grad_(), b.requires_grad_()), (x, w, b), dy)
    h = 2.0**-6
    with torch.no_grad():
        for t, g in ((x, gx), (w, gw), (b, gb)):
            flat = t.view(-1)
            for i in range(flat.numel()):
                v = flat[i].item()
                flat[i] = v + h
                up = (ops.layer_norm(x, w, b).double() * dy).sum()
                flat[i] = v - h
                down = (ops.layer_norm(x, w, b).double() * dy).sum()
                flat[i] = v
                assert abs((up - down) / (2 * h) - g.view(-1)[i]) < 5e-3


def test_norm_refusals():
    x, w = torch.randn(3, 8), torch.ones(8)
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(TypeError):
        ops.layer_norm(x.half(), w.bfloat16())
    with pytest.raises(TypeError):
        ops.layer_norm(x.half(), w.half(), w)
    with pytest.raises(TypeError):
        ops.layer_norm([1.0, 2.0])
    with pytest.raises(ValueError):
        ops.layer_norm(x, torch.ones(7))
    with pytest.raises(ValueError):
        ops.layer_norm(x, eps=float("nan"))
    with pytest.raises(ValueError):
        ops.layer_norm(x, eps=-1e-5)
    with pytest.raises(ValueError):
        ops.layer_norm(torch.empty(3, 0))
    with pytest.raises(ValueError):
        ops.layer_norm(x, w.to("meta"))
    y = ops.layer_norm(x.requires_grad_(), w)
    g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):  # differentiable once
        g.sum().backward()


# ------------------------------------------------------------------ drawing categories
SETTINGS = [dict(), dict(temperature=0.6), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2), dict(temperature=0.0),
            dict(temperature=1.4, top_k=12, top_p=0.9, min_p=0.05), dict(top_k=10**9, top_p=1.0), dict(top_p=0.0),
            dict(min_p=1.5), dict(temperature=1e-30), dict(temperature=float("inf"))]


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("settings", SETTINGS)
def test_sample(settings, kind):
    g = torch.Generator().manual_seed(1)
    for rows, cols in [(40, 1), (200, 2), (60, 7), (30, 64), (20, 65), (6, 1500)]:
        z = (torch.randn(rows, cols, generator=g) * 2).to(cases.DTYPES[kind])
        cases.check_sample(z, torch.rand(rows, generator=g), **settings)
        cases.check_sample(z, torch.rand(rows, generator=g, dtype=torch.float64), mask=torch.rand(rows, cols, generator=g) < 0.7, **settings)


def sample_edge_rows():
    """(logits, mask, u): rows that a mask empties, infinities and NaN in barred places, the type's lowest values,
    ties, both zeros"""
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
def test_sample_edge_rows(settings):
    z, mask, u = sample_edge_rows()
    got = cases.check_sample(z, u, mask=mask, **settings)
    assert got[1] == got[3] == got[10] == -1 and got[2] >= 2 and got[6] == 1
    for u in (0.0, 0.25, 0.5, 0.75):  # equal weights: exactly the quarters, in index order
        assert ops.sample_logits(z[8], torch.tensor(u)) == int(u * 4)
        assert ops.sample_logits(z[7], torch.tensor(u)) == int(u * 4)
        assert ops.sample_logits(z[4], torch.tensor(u)) == int(u * 4)


def test_sample_u_beyond_its_range_and_nan():
    z = torch.tensor([3.0, 1.0, 2.0])
    assert ops.sample_logits(z, torch.tensor(-1.0)) == 0
    assert ops.sample_logits(z, torch.tensor(1.0)) == 1
    assert ops.sample_logits(z, torch.tensor(7.0), top_k=2) == 2
    assert ops.sample_logits(z, torch.tensor(float("nan"))) == -1
    assert ops.sample_logits(torch.empty(0, 5), torch.empty(0)).shape == (0,)


def test_sample_settings_of_each_row():
    g = torch.Generator().manual_seed(2)
    n = 64
    z = torch.randn(n, 33, generator=g) * 2
    sets = dict(temperature=torch.rand(n, generator=g) * 2, top_k=torch.randint(-1, 40, (n,), generator=g),
                top_p=torch.rand(n, generator=g) * 1.2, min_p=torch.rand(n, generator=g) * 0.3 - 0.05)
    sets["temperature"][3] = 0
    u = torch.rand(n, generator=g)
    cases.check_sample(z, u, **sets)
    cases.check_sample(z.view(8, 8, 33), u.view(8, 8), mask=torch.rand(33, generator=g) < 0.6, **sets)
    sets["top_p"][5] = float("nan")
    assert ops.sample_logits(z, u, **sets)[5] == -1


def test_sample_refusals():
    z, u = torch.randn(4, 5), torch.rand(4)
    for bad in (dict(u=torch.rand(5)), dict(u=u[:, None]), dict(mask=torch.ones(4, 4, dtype=torch.bool)),
                dict(temperature=torch.ones(3)), dict(temperature=float("nan")), dict(top_p=torch.ones(2, 2))):
        with pytest.raises(ValueError):
            ops.sample_logits(**{"logits": z, "u": u, **bad})
    for bad in (dict(u=u.half()), dict(logits=z.double()), dict(logits=z.long()), dict(mask=torch.ones(4, 5)),
                dict(top_k=torch.ones(4)), dict(top_p=torch.ones(4, dtype=torch.int32)), dict(u=0.5)):
        with pytest.raises(TypeError):
            ops.sample_logits(**{"logits": z, "u": u, **bad})


# ------------------------------------------------------------------ distillation
@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (50, 2, 2), (9, 33, 5), (7, 65, 65), (3, 2001, 64)])
def test_distill(rows, cols, k, kind):
    for padded, T, index in ((False, 1.0, torch.int64), (True, 2.5, torch.int32)):
        cases.check_distill(*cases.distill_inputs(rows, cols, k, cases.DTYPES[kind], CPU, padded=padded, index=index), temperature=T)


def distill_edges():
    """(logits, index, teacher, grad): the same index twice, an empty list, masked students and teachers, lists in any order"""
    inf = float("inf")
    z = torch.randn(6, 8, generator=torch.Generator().manual_seed(3))
    z[3, :4] = -inf
    z[4] = torch.finfo(torch.float32).min
    at = torch.tensor([[3, 3, 1], [-1, -1, -1], [0, 7, -5], [7, 5, 4], [2, 2, 2], [6, 1, 6]])
    t = torch.tensor([[1.0, 2.0, 0.5], [1.0, 2.0, 3.0], [-inf, 1.0, 9.0], [0.0, 1.0, 2.0], [1.0, 1.0, 1.0], [0.3, -inf, 0.1]])
    return z, at, t, torch.tensor([1.0, 2.0, -0.5, 0.25, 3.0, 0.0])


def test_distill_edges():
    z, at, t, g = distill_edges()
    loss, dz = cases.check_distill(z, at, t, g, temperature=1.5)
    assert loss[1] == 0 and not dz[1].any()


def test_distill_bad_index_and_masked_student():
    z, at, t, g = distill_edges()
    at[0, 1] = 8
    z[2, 7] = -float("inf")  # a listed category that the student rules out
    loss, dz = cases.check_distill(z, at, t, g)
    assert loss[0].isnan() and dz[0].isnan().all() and loss[2] == float("inf") and dz[2].isfinite().all()
    t[4, 0] = float("nan")
    assert ops.distill_loss(z, at, t)[4].isnan()


def test_distill_refusals():
    z, at, t = torch.randn(4, 9), torch.zeros(4, 2, dtype=torch.int64), torch.randn(4, 2)
    for bad in (dict(teacher_index=at[:3]), dict(teacher_logits=t[:, :1]), dict(temperature=0.0), dict(temperature=float("nan")),
                dict(temperature=-1.0), dict(teacher_logits=t.clone().requires_grad_()),
                dict(teacher_index=at[:, :0], teacher_logits=t[:, :0]),
                dict(teacher_index=at.repeat(1, 600), teacher_logits=t.repeat(1, 600))):
        with pytest.raises(ValueError):
            ops.distill_loss(**{"logits": z, "teacher_index": at, "teacher_logits": t, **bad})
    for bad in (dict(logits=z.double()), dict(teacher_index=at.float()), dict(teacher_logits=t.double())):
        with pytest.raises(TypeError):
            ops.distill_loss(**{"logits": z, "teacher_index": at, "teacher_logits": t, **bad})


# ------------------------------------------------------------------ the C entry points
def _refused(fn, args, **changes):
    for k, v in changes.items():
        setattr(args, k, v)
    L = _lib.load()
    assert getattr(L, fn)(args) == -1 and L.fm_last_error()


def test_c_refusals():
    """every refusal of a C entry point returns FM_EINVAL with a message and touches no output"""
    L = _lib.load()
    assert L.fm_layer_norm_forward(None) == L.fm_sample_logits(None) == L.fm_distill_backward(None) == -1
    x, out = torch.randn(2, 4), torch.full((2, 4), 7.0)

    def norm(**c):
        a = _lib.FmLayerNormArgs(device=-1, rows=2, cols=4, x=x.data_ptr(), x_stride=4, eps=1e-5, y=out.data_ptr())
        _refused("fm_layer_norm_forward", a, **c)

    norm(device=-2), norm(x_dtype=3), norm(param_dtype=1), norm(rows=-1), norm(cols=0), norm(x_stride=-1), norm(x=None)
    norm(y=None), norm(eps=-1.0), norm(mean=out.data_ptr()), norm(x=x.data_ptr() + 1), norm(rows=2**61), norm(cols=2**31)
    mean = torch.zeros(2)
    b = _lib.FmLayerNormArgs(device=0, rows=2, cols=4, x=x.data_ptr(), x_stride=4, dy=x.data_ptr(), dy_stride=4, mean=mean.data_ptr(),
                             rstd=mean.data_ptr(), dweight=out.data_ptr())
    _refused("fm_layer_norm_backward", b)  # no workspace: before the device is looked at
    _refused("fm_layer_norm_backward", b, device=-1, dy=None)
    u, tok = torch.rand(2), torch.full((2,), 7)

    def sample(**c):
        a = _lib.FmSampleArgs(device=-1, rows=2, cols=4, logits=x.data_ptr(), stride=4, u=u.data_ptr(), temperature=1.0, top_p=1.0, out=tok.data_ptr())
        _refused("fm_sample_logits", a, **c)

    sample(dtype=3), sample(u_dtype=1), sample(cols=0), sample(cols=2**31), sample(u=None), sample(out=None), sample(stride=-4)
    sample(temperature=float("nan")), sample(out=tok.data_ptr() + 4), sample(mask_stride=-1)
    at, t, loss = torch.zeros(2, 1, dtype=torch.int64), torch.zeros(2, 1), torch.full((2,), 7.0)

    def distill(fn="fm_distill_forward", **c):
        a = _lib.FmDistillArgs(device=-1, index_dtype=5, rows=2, cols=4, k=1, logits=x.data_ptr(), stride=4, index=at.data_ptr(), index_stride=1,
                               teacher=t.data_ptr(), teacher_stride=1, temperature=1.0, loss=loss.data_ptr())
        _refused(fn, a, **c)

    distill(index_dtype=0), distill(teacher_dtype=4), distill(k=0), distill(k=1025), distill(temperature=0.0), distill(loss=None)
    distill(index=None), distill(fn="fm_distill_backward"), distill(index=at.data_ptr() + 4), distill(temperature=float("inf"))
    assert (out == 7).all() and (tok == 7).all() and (loss == 7).all()


def test_rows_beyond_the_most_columns_are_refused():
    """2^28 columns are taken (no rows: nothing is read), one more is not"""
    L = _lib.load()
    norm, sample = _lib.FmLayerNormArgs(device=-1, cols=2**28), _lib.FmSampleArgs(device=-1)
    distill = _lib.FmDistillArgs(device=-1, cols=2**28, k=1, index_dtype=_lib.FM_DTYPE_I32, temperature=1.0)
    assert L.fm_layer_norm_forward(norm) == L.fm_distill_forward(distill) == 0
    norm.cols = sample.cols = distill.cols = 2**28 + 1
    assert L.fm_layer_norm_forward(norm) == L.fm_layer_norm_backward(norm) == L.fm_sample_logits(sample) == -1
    assert L.fm_distill_forward(distill) == L.fm_distill_backward(distill) == -1


def test_forward_mode_derivatives_are_refused():
    ad = torch.autograd.forward_ad
    x, z = torch.randn(3, 4), torch.randn(3, 5)
    with ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.layer_norm(ad.make_dual(x, torch.ones(3, 4)))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.layer_norm(x, ad.make_dual(torch.ones(4), torch.ones(4)))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.distill_loss(ad.make_dual(z, z), torch.zeros(3, 1, dtype=torch.int64), torch.zeros(3, 1))


def test_arguments_that_are_no_tensors_are_refused():
    with pytest.raises(TypeError):
        ops.layer_norm(torch.randn(3, 4), [1.0] * 4)
    with pytest.raises(TypeError):
        ops.sample_logits(torch.randn(3, 4), torch.rand(3), mask=[True] * 4)


def test_missing_device_is_an_error_and_not_the_cpu():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    x = torch.randn(2, 4)
    a = _lib.FmLayerNormArgs(device=0, rows=2, cols=4, x=x.data_ptr(), x_stride=4, eps=1e-5, y=x.data_ptr())
    assert _lib.load().fm_layer_norm_forward(a) == -2


def test_struct_layouts_match_the_header():
    """the ctypes records' sizes are the header's (8-byte fields, ints in pairs)"""
    assert C.sizeof(_lib.FmLayerNormArgs) == 16 + 8 * 18
    assert C.sizeof(_lib.FmSampleArgs) == 16 + 8 * 19
    assert C.sizeof(_lib.FmDistillArgs) == 16 + 8 * 18


# ------------------------------------------------------------------ the policy and the trainer
def test_policy_options_leave_the_default_as_it_was():
    torch.manual_seed(0)
    a = ActorCriticPolicy(5, nvec=[2, 2, 3])
    torch.manual_seed(0)
    b = ActorCriticPolicy(5, nvec=[2, 2, 3], fused_sampling=True)
    assert list(a.state_dict()) == list(b.state_dict()) and not any("weight" in k and v.dim() == 1 for k, v in a.state_dict().items())
    obs = torch.randn(64, 5)
    assert torch.equal(a.predict(obs), b.predict(obs))
    assert [tuple(t.shape) for t in a.action_logits(torch.randn(4, 7))] == [(4, 2, 2), (4, 1, 3)]
    with pytest.raises(ValueError):
        ActorCriticPolicy(5, action_dim=3, fused_sampling=True)


def test_policy_draws_with_settings():
    torch.manual_seed(1)
    pol = ActorCriticPolicy(5, nvec=[4, 4, 3], net_arch=(16,))
    obs = torch.randn(500, 5)
    g = torch.Generator().manual_seed(3)
    best = pol.predict(obs)
    assert torch.equal(pol.predict(obs, deterministic=False, top_k=1), best)
    assert torch.equal(pol.predict(obs, deterministic=False, temperature=0.0), best)
    two = pol.predict(obs, deterministic=False, generator=g, top_k=2)
    head = pol._dist_params(obs)[0]
    for d, (o, n) in enumerate([(0, 4), (4, 4), (8, 3)]):
        rank = (head[:, o:o + n].argsort(1, descending=True) == two[:, d, None].long()).float().argmax(1)
        assert set(rank.tolist()) == {0, 1}
    fused = ActorCriticPolicy(5, nvec=[4, 4, 3], net_arch=(16,), fused_sampling=True)
    fused.load_state_dict(pol.state_dict())
    acts = torch.stack([fused(obs[:1].expand(500, 5), generator=g)[0] for _ in range(8)]).reshape(-1, 3)
    p = torch.softmax(head[0, :4], 0)
    freq = torch.bincount(acts[:, 0].long(), minlength=4) / len(acts)
    assert (freq - p).abs().max() < 5 * 0.5 / 4000**0.5  # five standard deviations of a share of 4000 draws
    for bad in (dict(deterministic=True, top_k=2), dict()):
        with pytest.raises((ValueError, TypeError)):
            pol.predict(obs, **bad) if bad else pol.predict(obs, deterministic=False, beam=3)
    with pytest.raises(ValueError):
        ActorCriticPolicy(5, action_dim=3).predict(obs, deterministic=False, temperature=0.5)


def test_layer_norm_policy_gradients_are_the_composed_ones():
    """the policy with layer_norm against the same weights through elementary torch operations in float64"""
    torch.manual_seed(2)
    pol = ActorCriticPolicy(7, nvec=[2, 2], net_arch=(24, 16), layer_norm=True)
    assert isinstance(pol.mlp_extractor.policy_net[1], ops.LayerNorm) and len(pol.mlp_extractor.policy_net) == 6
    obs, act = torch.randn(33, 7), torch.randint(0, 2, (33, 2)).float()
    v, lp, ent = pol.evaluate_actions(obs, act)
    grads = torch.autograd.grad((v + lp + 0.1 * ent).sum(), list(pol.parameters()))
    q = {k: t.detach().double().requires_grad_() for k, t in pol.named_parameters()}

    def net(name):
        h = obs.double()
        for i in (0, 3):
            h = h @ q[f"mlp_extractor.{name}.{i}.weight"].T + q[f"mlp_extractor.{name}.{i}.bias"]
            c = h - h.mean(1, keepdim=True)
            h = c / (c.square().mean(1, keepdim=True) + 1e-5).sqrt()
            h = torch.tanh(h * q[f"mlp_extractor.{name}.{i + 1}.weight"] + q[f"mlp_extractor.{name}.{i + 1}.bias"])
        return h

    head = (net("policy_net") @ q["action_net.weight"].T + q["action_net.bias"]).view(33, 2, 2)
    logp = torch.log_softmax(head, -1)
    want = (net("value_net") @ q["value_net.weight"].T + q["value_net.bias"]).sum() + \
        logp.gather(2, act.long()[..., None]).sum() - 0.1 * (logp.exp() * logp).sum()
    for (k, _), a, b in zip(pol.named_parameters(), grads, torch.autograd.grad(want, list(q.values()))):
        # sums of 33 rows through two layers: some hundred float32 roundings of the gradients' size
        assert (a.double() - b).abs().max() <= 300 * cases.E32 * (b.abs().max() + 1), k


@pytest.mark.parametrize("top", [None, 1])
def test_ppo_with_a_teacher(top, tmp_path):
    """rollout by fused draws, layer norm in the student, the teacher's top logits recorded and distilled"""
    env = ToyEnv(n=32, discrete=True)
    torch.manual_seed(4)
    teacher = ActorCriticPolicy(5, nvec=[2, 2, 2], net_arch=(8,))
    ppo = PPO(env, policy_kwargs=dict(net_arch=(16, 16), layer_norm=True, fused_sampling=True), n_steps=4, batch_size=64, n_epochs=2, seed=1,
              teacher=teacher, distill_coef=0.5, distill_temperature=2.0, distill_top_k=top)
    before = [p.detach().clone() for p in teacher.parameters()]
    ppo.learn(32 * 4 * 2)
    assert all(np.isfinite(r["distill_loss"]) and r["distill_loss"] >= 0 for r in ppo.logs)
    assert all(torch.equal(a, b) and b.grad is None for a, b in zip(before, teacher.parameters()))
    path = str(tmp_path / "student.zip")
    ppo.save(path)
    again = PPO(ToyEnv(n=8, discrete=True), policy_kwargs=dict(net_arch=(16, 16), layer_norm=True)).load_policy(path)
    obs = torch.randn(9, 5)
    assert torch.equal(again.policy.predict(obs), ppo.policy.predict(obs))
    # the recorded lists are the teacher's at the rollout's observations
    buf, _ = ppo.collect_rollouts()
    index, logits = teacher.top_logits(buf["obs"][2], top)[0]
    assert torch.equal(buf["teacher_index0"][2], index) and torch.equal(buf["teacher_logits0"][2], logits)


def test_ppo_teacher_refusals():
    env = ToyEnv(n=4, discrete=True)
    with pytest.raises(ValueError):
        PPO(env, teacher=ActorCriticPolicy(5, nvec=[2, 2]))
    with pytest.raises(ValueError):
        PPO(ToyEnv(n=4), teacher=ActorCriticPolicy(5, nvec=[2, 2, 2]))
    with pytest.raises(ValueError):
        PPO(env, teacher=ActorCriticPolicy(5, nvec=[2, 2, 2]), distill_top_k=0)
