"""The policy's and the trainer's use of the operators: what must not go by without a word."""
import pytest
import torch

from factory_marl_amd.ppo import PPO, ActorCriticPolicy
from test_ppo import ToyEnv


def broken(**kw):
    pol = ActorCriticPolicy(5, nvec=[2, 2, 3], net_arch=(8,), **kw)
    with torch.no_grad():
        pol.action_net.bias[5] = float("nan")
    return pol


def test_a_policy_that_has_become_nan_raises_where_it_draws():
    obs = torch.randn(4, 5)
    for pol, settings in ((broken(), {}), (broken(fused_sampling=True), {}), (broken(), dict(top_p=0.9))):
        with pytest.raises(RuntimeError):
            pol.predict(obs, deterministic=False, **settings)
    with pytest.raises(RuntimeError):
        broken(fused_sampling=True)(obs)
    env = ToyEnv(n=8, discrete=True)
    ppo = PPO(env, policy_kwargs=dict(net_arch=(8,), fused_sampling=True), n_steps=2, batch_size=8, n_epochs=1)
    with torch.no_grad():
        ppo.policy.action_net.weight[0, 0] = float("nan")
    with pytest.raises(RuntimeError):
        ppo.collect_rollouts()
