"""Derivatives that the low-bit calls do not have are refused, not dropped."""
import pytest
import torch
from torch.autograd import forward_ad

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
