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


@pytest.mark.parametrize("precision", ["float32", "mxfp4", "mxfp4 after float32"])
def test_first_steps_on_two_streams_at_once(precision):
    """no refresh before: the second stream's step reads weights that the first one's has made, however late that runs"""
    import copy

    twin = _agent().use_fused_sampling(3)
    if precision != "float32":
        twin.use_mxfp4_trunk()
    twin.refresh_rollout_heads()
    xs = [_obs(600, seed=k) for k in range(2)]
    lp = torch.empty(600, device="cuda")
    want = [torch.empty(600, device="cuda") for _ in xs]
    for x, v in zip(xs, want):
        twin.rollout_step(x, lp, v)
    net = _agent().use_fused_sampling(3)
    if precision == "mxfp4 after float32":
        net.rollout_step(xs[0], lp, torch.empty_like(lp))
    if precision != "float32":
        net.use_mxfp4_trunk()
    torch.cuda.synchronize()
    got, lps = [torch.empty(600, device="cuda") for _ in xs], [torch.empty(600, device="cuda") for _ in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for k, stream in enumerate(streams):
        with torch.cuda.stream(stream):
            if k == 0:
                torch.cuda._sleep(20_000_000)  # about ten milliseconds
            net.rollout_step(xs[k], lps[k], got[k])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_capture_does_not_leave_weights_behind_that_no_launch_has_written():
    warm = _agent(1).use_mxfp4_trunk()
    x = _obs(40)
    with torch.no_grad():
        warm.get_value(x)
    net = _agent().use_fused_sampling(3).use_mxfp4_trunk()
    twin = _agent().use_fused_sampling(3).use_mxfp4_trunk()
    lp, v = torch.empty(40, device="cuda"), torch.empty(40, device="cuda")
    net.refresh_rollout_heads()
    net._coarse.clear()  # as after use_mxfp4_trunk() on a policy that has rolled out in float32
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="refresh_rollout_heads"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), capture_error_mode="thread_local"):
            net.rollout_step(x, lp, v)
    with pytest.raises(RuntimeError, match="refresh_rollout_heads"):
        with torch.cuda.graph(torch.cuda.CUDAGraph(), capture_error_mode="thread_local"):
            net.refresh_rollout_heads()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph, capture_error_mode="thread_local"):
        value = net.get_value(x)
    assert not net._coarse
    net.rollout_step(x, lp, v)  # before the first replay
    with torch.no_grad():
        want = twin.get_value(x)
        torch.testing.assert_close(v, want.squeeze(1), rtol=1e-5, atol=1e-5)
        for step in range(3):
            for p in net.parameters():
                p.mul_(1.1)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(value, net.get_value(x))
