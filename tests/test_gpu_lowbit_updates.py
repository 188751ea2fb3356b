"""What an update of the low-bit policy computes, keeps and leaves out."""
import numpy as np
import pytest
import torch

import lowbit_reference as ref

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


def _d(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [32, 8])
def test_an_update_computes_the_numbers_that_acted(dtype, bits, monkeypatch):
    """also where the parameters have 16 bits: the hidden layer is quantised from its float32 sums in both"""
    from marl_amd import act8

    net = _agent().to(dtype).use_mxfp4_trunk()
    with torch.no_grad():
        for layer in (net.network[0], net.network[2]):
            layer.bias.normal_(0.0, 0.1)
    x = _obs(1500).to(dtype)
    with torch.no_grad():
        acted = net._trunk(x)
    assert acted.dtype == dtype
    if bits == 32:
        h = net._trunk(x)
        assert h.requires_grad and torch.equal(h, acted)
        return
    seen = []
    compress = act8.compress
    monkeypatch.setattr(act8, "compress", lambda t, nonnegative=False: (seen.append(t.detach().clone()), compress(t, nonnegative))[1])
    net.use_activation_checkpoints()
    net.logits_and_value(x)
    assert len(seen) == 3 and torch.equal(seen[2], acted)  # the observations, then what each layer of the trunk gave


@pytest.mark.parametrize("dtype,step", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_of_a_16_bit_policy(dtype, step, bits):
    net = _agent().to(dtype).use_mxfp4_trunk()
    if bits == 8:
        net.use_activation_checkpoints()
    rows = 600
    x = _obs(rows).to(dtype)
    w0, w1 = _d(net.network[0].weight), _d(net.network[2].weight)
    h = [_d(x)]
    for w in (w0, w1):
        h.append(np.maximum(ref.mxfp4(h[-1])[2] @ ref.mxfp4(w)[2].T, 0.0).astype(np.float32).astype(np.float64))
    kept = [ref.act8(h[0], False)[2], ref.act8(h[1], True)[2], ref.act8(h[2], True)[2]] if bits == 8 else h
    g = torch.randn(rows, 8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).to(dtype)
    gh, wh = _d(g), np.concatenate([_d(net.actor.weight), _d(net.critic.weight)])
    g1 = (gh @ wh) * (h[2] > 0)
    g0 = (g1 @ w1) * (h[1] > 0)
    want = {"heads.weight": gh.T @ kept[2], "network.2.weight": g1.T @ kept[1], "network.2.bias": g1.sum(0),
            "network.0.weight": g0.T @ kept[0], "network.0.bias": g0.sum(0)}
    logits, value = net.logits_and_value(x)
    torch.autograd.backward([logits, value], [g[:, :7], g[:, 7:]])
    assert all(p.grad.dtype == dtype for p in net.parameters())
    got = {k: _d(p.grad) for k, p in net.named_parameters()}
    got["heads.weight"] = np.concatenate([got.pop("actor.weight"), got.pop("critic.weight")])
    for name, w in want.items():
        # Roundings to the type: of the layer's input, of the gradient behind each layer (the two heads' are rounded before they
        # are added: two), and of the result.  Each is off by at most half a step and they are independent, so that their sums grow
        # as the gradient's own do: at most five of them, five half steps of its norm.
        assert np.linalg.norm(got[name] - w) <= 5 * step * np.linalg.norm(w) + 1e-12, name


def test_no_gradients_are_made_up_for_the_codes(monkeypatch):
    """codes and scales are results of the layer's Function too; autograd has nothing to hand back for them"""
    from marl_amd import policy

    seen = []
    backward = policy._KeptLinear.backward
    monkeypatch.setattr(policy._KeptLinear, "backward", staticmethod(lambda ctx, gy, *kept: (seen.append(kept), backward(ctx, gy, *kept))[1]))
    net = _agent().use_activation_checkpoints()
    logits, value = net.logits_and_value(_obs(40))
    (logits.sum() + value.sum()).backward()
    assert sorted(len(k) for k in seen) == [0, 2, 2] and all(g is None for k in seen for g in k)


def test_an_output_without_a_gradient_of_its_own():
    from marl_amd import act8, policy

    class Cut(torch.autograd.Function):
        @staticmethod
        def forward(ctx, t):
            return t.clone()

        @staticmethod
        def backward(ctx, g):
            return None

    net = _agent().use_activation_checkpoints()
    x, layer = _obs(40), net.network[0]
    kept = act8.compress(x)
    out, _, _ = policy._KeptLinear.apply(x, kept.codes, kept.scales, False, layer.weight, layer.bias, True)
    Cut.apply(out).sum().backward()
    assert all(p.grad is None or not p.grad.any() for p in layer.parameters())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,out,cols", [(1, 3, 5), (130, 16, 40), (2048, 512, 202), (9001, 300, 520), (5000, 100, 1)])
def test_parameter_gradients_without_the_cut_gradient(rows, out, cols, dtype):
    """the same bits; and nothing but the two results and the workspace is written"""
    from marl_amd import _lib, act8
    from marl_amd.mxfp4 import _TYPES, _p

    g = torch.Generator(device="cuda").manual_seed(rows + out)
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    act = act8.compress(rand(rows, cols))
    mask = act8.compress(torch.relu(rand(rows, out)), nonnegative=True)
    grad = rand(rows, out).to(dtype)
    grad[mask.codes == 0] = float("nan")  # what is cut does not count
    gw, gb, masked = act8.weight_grad(grad, act, mask)
    gw2, gb2, none = act8.weight_grad(grad, act, mask, want_masked=False)
    assert none is None and torch.isfinite(gw).all() and torch.equal(gw, gw2) and torch.equal(gb, gb2)
    assert all(torch.equal(a, b) for a, b in zip(act8.weight_grad(masked, act)[:2], act8.weight_grad(masked, act, want_masked=False)[:2]))
    L = _lib.lib()
    need = L.marl_act_weight_grad_workspace_bytes(rows, out, cols)
    bufs = [torch.full((n + 128,), 7.0, device="cuda") for n in (out * cols, out)]
    work = torch.full((need + 64,), 9, dtype=torch.uint8, device="cuda")
    before = [t.clone() for t in (grad.view(torch.int32 if dtype == torch.float32 else torch.int16), mask.codes, act.codes)]
    _lib.check(L.marl_act_param_grad(_p(grad), _TYPES[dtype], rows, out, _p(act.codes), _p(act.scales), cols, 0, _p(mask.codes),
                                     _p(bufs[0][64:]), _p(bufs[1][64:]), _p(work), torch.cuda.current_stream().cuda_stream), "marl_act_param_grad")
    for buf, want in zip(bufs, (gw, gb)):
        assert torch.equal(buf[64:-64], want.flatten()) and (buf[:64] == 7).all() and (buf[-64:] == 7).all()
    assert (work[need:] == 9).all()
    after = (grad.view(torch.int32 if dtype == torch.float32 else torch.int16), mask.codes, act.codes)
    assert all(torch.equal(a, b) for a, b in zip(before, after))


def test_an_update_cuts_no_gradient_that_nothing_reads(monkeypatch):
    """the first layer's input are the observations: the gradient behind its ReLU, 512 values a sample, goes nowhere"""
    from marl_amd import act8

    wanted = []
    weight_grad = act8.weight_grad
    monkeypatch.setattr(act8, "weight_grad", lambda g, a, m=None, **kw: (wanted.append((a.shape[1], kw.get("want_masked", True))), weight_grad(g, a, m, **kw))[1])
    net = _agent().use_activation_checkpoints()
    x = _obs(40)
    logits, value = net.logits_and_value(x)
    (logits.sum() + value.sum()).backward()
    assert wanted == [(256, True), (512, True), (202, False)]
    first = net.network[0].weight.grad.clone()
    net.zero_grad()
    wanted.clear()
    x.requires_grad_()
    logits, value = net.logits_and_value(x)
    (logits.sum() + value.sum()).backward()
    assert wanted == [(256, True), (512, True), (202, True)]
    assert torch.equal(net.network[0].weight.grad, first)
    d = lambda t: t.detach().double()  # noqa: E731
    h0 = torch.relu(torch.addmm(d(net.network[0].bias), d(x), d(net.network[0].weight).t()))
    h1 = torch.relu(torch.addmm(d(net.network[2].bias), h0, d(net.network[2].weight).t()))
    g1 = (d(net.actor.weight).sum(0) + d(net.critic.weight).sum(0)) * (h1 > 0)
    want = ((g1 @ d(net.network[2].weight)) * (h0 > 0)) @ d(net.network[0].weight)
    # float32 products of up to 512 terms
    assert (x.grad.double() - want).norm() <= 4e-6 * want.norm()


def _update_peak(net, rows):
    """bytes that an update's forward and backward pass add to what was allocated before, at their peak"""
    x = _obs(rows)
    g = torch.randn(rows, 8, device="cuda") / rows
    for _ in range(2):  # the second time gradients and library workspaces are there
        net.zero_grad(set_to_none=False)
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        base = torch.cuda.memory_allocated()
        logits, value = net.logits_and_value(x)
        torch.autograd.backward([logits, value], [g[:, :7], g[:, 7:]])
        torch.cuda.synchronize()
        peak = torch.cuda.max_memory_allocated() - base
        del logits, value
    return peak


def test_the_peak_of_an_update():
    """forward and backward; bytes a sample, of float32 values unless said"""
    rows = 262144
    net = _agent()
    wide = _update_peak(net, rows)
    net.use_activation_checkpoints()
    kept = _update_peak(net, rows)
    # Float32: in the second layer's backward pass there are both hidden layers (512 + 256), the gradient of its output before and
    # behind the ReLU (256 each) and that of its input (512).
    assert wide >= rows * (512 + 256 + 256 + 256 + 512) * 4
    # 8 bits: a byte and 1/32 for every value of both layers and the observations; at the peak, in the same place, the gradient of
    # the output before and behind the ReLU and that of the input; the heads' results and their gradients (4 x 8 values); and
    # the splits' sums, at most 256 tiles of 128 x 256.
    assert kept <= rows * ((202 + 512 + 256) * 34 / 32 + (256 + 256 + 512) * 4 + 4 * 8 * 4) + 256 * 128 * 257 * 4 + (8 << 20)
    assert kept <= 0.75 * wide
    # Straight through the 4-bit trunk: 17 bytes for 32 values of the observations and of the first hidden layer more (the observations
    # in 8 bits are not kept then).  With float32 activations the second layer's input, as large as its gradient, is there while the
    # weight's gradient is formed, beside the 128 slabs that that adds up; otherwise the slabs are gone before the peak.
    trunk = _agent().use_mxfp4_trunk(straight_through=True)
    assert _update_peak(trunk, rows) <= wide + rows * (202 + 512) * 18 / 32 + 128 * 256 * 512 * 4 + (32 << 20)
    trunk.use_activation_checkpoints()
    assert _update_peak(trunk, rows) <= kept + rows * (202 + 512) * 18 / 32 + (32 << 20)
