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
