"""Derivatives: those that the low-bit calls do not have are refused, not dropped; the 4-bit trunk's backward passes are what
they are named."""
import numpy as np
import pytest
import torch
from torch.autograd import forward_ad

import lowbit_reference as ref

pytestmark = pytest.mark.gpu


def test_forward_mode_derivatives_are_refused():
    from marl_amd import act8, mxfp4
    from marl_amd.policy import Agent
    from marl_amd.spaces import Box, Discrete

    x, b = torch.ones(4, 40, device="cuda"), torch.zeros(8, device="cuda")
    w, act = mxfp4.quantize(torch.ones(8, 40, device="cuda")), act8.compress(x)
    net = Agent(Box(-1, 1, (40,)), Discrete(7), 2, 1, build_centralised=False).cuda().use_mxfp4_trunk()
    with torch.no_grad():
        want, out = mxfp4.linear(x, w, b), net.get_value(x)
    with forward_ad.dual_level():
        dual, dual_b = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(b, torch.ones_like(b))
        dual_g = forward_ad.make_dual(torch.ones(4, 8, device="cuda"), torch.ones(4, 8, device="cuda"))
        for call in (lambda: mxfp4.quantize(dual), lambda: mxfp4.linear(dual, w, b), lambda: mxfp4.linear(x, w, dual_b), lambda: act8.compress(dual),
                     lambda: act8.weight_grad(dual_g, act)):
            with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
                call()
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            net.get_value(dual)
        weight = net.network[0].weight
        del net.network[0].weight
        net.network[0].weight = forward_ad.make_dual(weight.detach(), torch.ones_like(weight))
        with torch.no_grad(), pytest.raises(ValueError, match="forward-mode"):
            net.get_value(x)
        del net.network[0].weight
        net.network[0].weight = weight
        with torch.no_grad():  # without one, as ever
            assert torch.equal(mxfp4.linear(x, w, b), want) and torch.equal(net.get_value(x), out)


def test_the_backward_pass_is_the_unrounded_layers():
    """g W and g^T x from the operands before they went to 4 bits, not the g Q(W) and g^T Q(x) of a straight-through estimator"""
    from marl_amd import mxfp4, policy

    g = torch.Generator(device="cuda").manual_seed(1)
    x, w = torch.randn(300, 202, device="cuda", generator=g, requires_grad=True), torch.randn(70, 202, device="cuda", generator=g, requires_grad=True)
    b = torch.zeros(70, device="cuda", requires_grad=True)
    out = policy._LinearReLU.apply(x, w, b, True, mxfp4.quantize(w))
    grad = torch.randn(300, 70, device="cuda", generator=g)
    out.backward(grad)
    with torch.no_grad():
        xq, wq = mxfp4.quantize(x).dequantize().double(), mxfp4.quantize(w).dequantize().double()
        assert torch.allclose(out.double(), torch.relu(xq @ wq.t()), rtol=0, atol=1e-4)
        cut = grad.double() * (out > 0)
        for got, want, rounded in ((x.grad, cut @ w.double(), cut @ wq), (w.grad, cut.t() @ x.double(), cut.t() @ xq)):
            assert (got.double() - want).norm() <= 4e-6 * want.norm()  # float32 sums of up to 300 terms
            assert (got.double() - rounded).norm() > 0.01 * want.norm()  # 4 bits are off by more
        assert (b.grad.double() - cut.sum(0)).norm() <= 4e-6 * cut.sum(0).norm()


def _obs(rows, d=202, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, d, device="cuda", generator=g)
    x = (x.abs() > 0.9).float() * (x * 1.3).round()
    x[::3, 5] = 30.0  # a pot's timer: its neighbours round
    return x


@pytest.mark.parametrize("rows", [5, 600, 8192])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_straight_through_backward_pass(rows, bits, dtype):
    """that of relu(Q(x) Q(W)^T + b) with the roundings' derivatives taken as one, from the formats' definition in 64 bits"""
    from marl_amd.policy import Agent
    from marl_amd.spaces import Box, Discrete

    torch.manual_seed(5)
    net = Agent(Box(-1, 1, (202,)), Discrete(7), 2, 1, build_centralised=False).cuda().to(dtype).use_mxfp4_trunk(straight_through=True)
    if bits == 8:
        net.use_activation_checkpoints()
    x = _obs(rows, seed=rows).to(dtype).requires_grad_()
    d = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    w0, w1 = (ref.mxfp4(d(net.network[k].weight))[2] for k in (0, 2))
    h, read = d(x), []
    for w in (w0, w1):  # zero biases
        read.append(ref.mxfp4(h)[2])
        h = np.maximum(read[-1] @ w.T, 0.0).astype(np.float32).astype(np.float64)
        read.append(h)
    out = h if dtype == torch.float32 else d(torch.from_numpy(h).to(dtype))
    kept = ref.act8(out, True)[2] if bits == 8 else out
    g = torch.randn(rows, 8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    gh, wh = d(g), np.concatenate([d(net.actor.weight), d(net.critic.weight)])
    g1 = (gh @ wh) * (read[3] > 0)
    g0 = (g1 @ w1) * (read[1] > 0)
    want = {"heads.weight": gh.T @ kept, "network.2.weight": g1.T @ read[2], "network.2.bias": g1.sum(0),
            "network.0.weight": g0.T @ read[0], "network.0.bias": g0.sum(0), "x": g0 @ w0}
    logits, value = net.logits_and_value(x)
    with torch.no_grad():
        assert torch.equal(net._trunk(x), (net._trunk(x.detach()) if bits == 8 else torch.enable_grad()(net._trunk)(x)))
    torch.autograd.backward([logits, value], [g[:, :7], g[:, 7:]])
    got = {k: d(p.grad) for k, p in net.named_parameters()}
    got["heads.weight"], got["x"] = np.concatenate([got.pop("actor.weight"), got.pop("critic.weight")]), d(x.grad)
    # float32: sums through at most two products of up to 256 terms.  bfloat16: the gradient is rounded behind each layer (the two
    # heads' before they are added), in the first layer's input gradient once more, and the result: at most five half steps.
    close = 4e-6 if dtype == torch.float32 else 5 * 2.0 ** -8
    for name, w in want.items():
        assert np.linalg.norm(got[name] - w) <= close * np.linalg.norm(w) + 1e-12, name
    if dtype == torch.float32 and rows > 5:  # the unrounded layers' are other numbers
        other = ((gh @ wh) * (read[3] > 0)).T @ read[1]
        assert np.linalg.norm(got["network.2.weight"] - other) > 0.01 * np.linalg.norm(other)


def test_the_straight_through_backward_pass_of_the_centralised_critic():
    from marl_amd.policy import Agent
    from marl_amd.spaces import Box, Discrete

    torch.manual_seed(5)
    net = Agent(Box(-1, 1, (40,)), Discrete(7), 2, 8).cuda().use_mxfp4_trunk(straight_through=True)
    x = _obs(16, 40)
    joint = x.view(1, -1).clone().requires_grad_()
    c = net.centralised_critics
    value = net.get_value(x, joint_obs=joint)
    with torch.no_grad():
        assert torch.equal(net.get_value(x, joint_obs=joint), value)
    value.sum().backward()
    d = lambda t: t.detach().double().cpu().numpy()  # noqa: E731
    xq, wq = ref.mxfp4(d(joint))[2], ref.mxfp4(d(c[0].weight))[2]
    h0 = np.maximum(xq @ wq.T + d(c[0].bias), 0.0)
    h1 = np.maximum(h0 @ d(c[2].weight).T + d(c[2].bias), 0.0)
    g0 = ((d(c[4].weight) * (h1 > 0)) @ d(c[2].weight)) * (h0 > 0)
    for got, want in ((c[0].weight.grad, g0.T @ xq), (joint.grad, g0 @ wq)):
        assert np.linalg.norm(d(got) - want) <= 4e-6 * np.linalg.norm(want)  # float32 sums of up to 512 terms


def test_the_command_trains_straight_through(monkeypatch, tmp_path):
    from marl_amd import train
    from marl_amd.policy import Agent

    asked = []
    use = Agent.use_mxfp4_trunk
    monkeypatch.setattr(Agent, "use_mxfp4_trunk", lambda self, *a, **kw: (asked.append((a, kw)), use(self, *a, **kw))[1])
    train.main(["--num-agents", "2", "--num-envs", "16", "--layout", "overcooked_cramped_room_v0", "--num-steps", "32", "--total-steps", "2048",
                "--ppo-epoch", "1", "--max-steps", "50", "--data-path", str(tmp_path), "--seed", "3", "--trunk-precision", "mxfp4"])
    assert asked == [((), {"straight_through": True})]


def _first(layer, tensors):
    """leaves and the squared gradients, which can be differentiated again"""
    x, w, b, v = (t.clone().requires_grad_() for t in tensors)
    out = (layer(x, w, b) * v).sum(1).square().sum()
    return (x, w, v), sum(f.square().sum() for f in torch.autograd.grad(out, (w, b), create_graph=True))


def _leaves():
    g = torch.Generator(device="cuda").manual_seed(1)
    return [torch.randn(*shape, device="cuda", generator=g) for shape in ((700, 40), (30, 40), (30,), (1, 30))]


def test_second_derivatives_of_a_float32_layer():
    from marl_amd import policy

    pairs = []
    for layer, tensors in ((lambda x, w, b: policy._LinearReLU.apply(x, w, b, True), _leaves()),
                           (lambda x, w, b: torch.relu(x @ w.t() + b), [t.double() for t in _leaves()])):
        leaves, squares = _first(layer, tensors)
        pairs.append(torch.autograd.grad(squares, leaves))
    for a, b in zip(*pairs):
        assert (a.double() - b).norm() <= 1e-5 * b.norm()  # float32, six products and sums of up to 700 terms in a row


def test_a_straight_through_pass_has_no_second_derivatives():
    from marl_amd import mxfp4, policy

    _, squares = _first(lambda x, w, b: policy._StraightLinear.apply(x, w, b, True, mxfp4.quantize(w)), _leaves())
    with pytest.raises(RuntimeError, match="once_differentiable"):
        squares.backward()
