"""The calls of the policy that acts in 4 bits: shapes, first uses, streams, graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _agent(seed=5, central=False, num_envs=1, D=202):
    from marl_amd.policy import Agent
    from marl_amd.spaces import Box, Discrete

    torch.manual_seed(seed)
    return Agent(Box(-1, 1, (D,)), Discrete(7), 2, num_envs, build_centralised=central).cuda()


def _obs(rows, d=202, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, d, device="cuda", generator=g)
    return (x.abs() > 0.9).float() * (x * 1.3).round()


def test_a_joint_observation_of_any_shape_goes_through_the_4_bit_critic():
    net = _agent(central=True, num_envs=16)
    x = _obs(32)
    flat = x.view(-1)
    exact = net._central(flat.view(1, -1)).detach()
    assert net._central(flat).shape == (1,) and net._central(flat.view(1, 1, -1)).shape == (1, 1, 1)
    net.use_mxfp4_trunk()
    with torch.no_grad():
        want = net.get_value(x, joint_obs=flat.view(1, -1))
        assert want.shape == (1, 1) and not torch.equal(want, exact)
        for shape in ((-1,), (1, -1), (1, 1, -1)):
            value = net.get_action_and_value(x, joint_obs=flat.view(shape))[3]
            assert value.shape == flat.view(shape).shape[:-1] + (1,) and torch.equal(value.view(1, 1), want)
        both = net._central(torch.stack([flat, -flat]).view(2, 1, -1))
        assert both.shape == (2, 1, 1)
        torch.testing.assert_close(both[0], want, rtol=1e-5, atol=1e-5)  # float32 layers of another shape behind it
