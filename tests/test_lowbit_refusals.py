"""Bad arguments to the low-bit passes come back as errors before anything touches the GPU (no GPU needed)."""
import ctypes

import pytest
import torch

BAD = -1


def _lib():
    from marl_amd import _lib as lib

    return lib.lib()


P = 1 << 20  # an address nobody follows: every call here is refused


def _refused(rc, words):
    assert rc == BAD
    message = _lib().marl_last_error().decode()
    assert words in message, message


def test_quantise_and_read_back():
    L = _lib()
    _refused(L.marl_mx_quantize(P, 0, -1, 32, 0, P, P, None), "num_rows")
    _refused(L.marl_mx_quantize(P, 0, 4, 0, 0, P, P, None), "num_cols")
    _refused(L.marl_mx_quantize(P, 3, 4, 32, 0, P, P, None), "x_type")
    _refused(L.marl_mx_quantize(None, 0, 4, 32, 0, P, P, None), "NULL")
    _refused(L.marl_mx_quantize(P, 0, 4, 32, 31, P, P, None), "row_stride")
    _refused(L.marl_mx_quantize(P, 0, 4, 32, 0, P + 8, P, None), "aligned")
    _refused(L.marl_mx_quantize(P + 2, 0, 4, 32, 0, P, P, None), "aligned")
    _refused(L.marl_mx_quantize(P, 0, 1 << 30, 64, 0, P, P, None), "2^30")
    _refused(L.marl_mx_dequantize(P, P, 4, 32, 3, P, None), "out_type")
    _refused(L.marl_mx_dequantize(P, None, 4, 32, 0, P, None), "NULL")
    _refused(L.marl_mx_dequantize(P + 4, P, 4, 32, 0, P, None), "aligned")
    assert L.marl_mx_quantize(None, 0, 0, 32, 0, None, None, None) == 0  # no rows: nothing to do


def test_product():
    L = _lib()

    def call(x=P, xs=None, xt=0, rows=4, cols=64, stride=0, w=P, ws=P, out=8, bias=None, y=P, ys=None, yt=0, work=None):
        return L.marl_mx_linear(x, xs, xt, rows, cols, stride, w, ws, out, bias, 0, y, ys, yt, work, None)

    _refused(call(rows=-1), "num_rows")
    _refused(call(out=0), "num_out")
    _refused(call(xt=4), "x_type")
    _refused(call(yt=-1), "y_type")
    _refused(call(x=None), "NULL")
    _refused(call(ws=None), "NULL")
    _refused(call(xs=P), "d_x_scales")
    _refused(call(xt=3), "d_x_scales")
    _refused(call(yt=3), "d_y_scales")
    _refused(call(stride=63), "row_stride")
    _refused(call(xt=3, xs=P, stride=64), "row_stride")
    _refused(call(w=P + 4), "aligned")
    _refused(call(bias=P + 2), "aligned")
    _refused(call(y=P + 2), "aligned")
    _refused(call(cols=1000), "d_workspace")
    _refused(call(cols=5), "d_workspace")
    _refused(call(cols=1000, work=P + 4), "aligned")
    _refused(call(out=(1 << 22) + 1), "2^22")
    _refused(call(rows=5_000_000, cols=1000, work=P), "4,194,240")
    assert L.marl_mx_linear(None, None, 0, 0, 64, 0, None, None, 8, None, 0, None, None, 0, None, None) == 0


def test_workspace_sizes():
    L = _lib()
    assert L.marl_mx_linear_workspace_bytes(0, 131072, 512, 256) == 0 and L.marl_mx_linear_workspace_bytes(0, 1, 8, 1) == 0
    assert L.marl_mx_linear_workspace_bytes(0, 0, 1000, 8) == 0 and L.marl_mx_linear_workspace_bytes(0, 4, -1, 8) == 0
    with_codes, without = L.marl_mx_linear_workspace_bytes(0, 1, 6464, 512), L.marl_mx_linear_workspace_bytes(3, 1, 6464, 512)
    assert with_codes - without >= 202 * 17 and without >= 512 * 4
    assert L.marl_act_weight_grad_workspace_bytes(0, 8, 8) == 0
    assert L.marl_act_weight_grad_workspace_bytes(1 << 20, 256, 512) >= (256 * 512 + 256) * 4


def test_compress_and_weight_gradient():
    L = _lib()
    _refused(L.marl_act_compress(P, 0, 4, -3, 0, 1, P, P, None), "num_cols")
    _refused(L.marl_act_compress(P, 7, 4, 32, 0, 1, P, P, None), "x_type")
    _refused(L.marl_act_compress(P, 0, 4, 32, 5, 1, P, P, None), "row_stride")
    _refused(L.marl_act_compress(P, 0, 4, 32, 0, 1, None, P, None), "NULL")
    _refused(L.marl_act_dequantize(P, P, 4, 32, 1, 3, P, None), "out_type")
    _refused(L.marl_act_dequantize(P, P, 4, 32, 1, 0, P + 1, None), "aligned")

    def call(grad=P, gt=0, rows=4, out=8, codes=P, scales=P, cols=64, mask=None, masked=None, gw=P, gb=P, work=P):
        return L.marl_act_weight_grad(grad, gt, rows, out, codes, scales, cols, 0, mask, masked, gw, gb, work, None)

    _refused(call(rows=0), "positive")
    _refused(call(gt=3), "grad_type")
    _refused(call(gw=None), "NULL")
    _refused(call(mask=P), "go together")
    _refused(call(masked=2 * P), "go together")
    _refused(call(mask=P, masked=P), "must not be d_grad")
    _refused(call(gb=P + 2), "aligned")
    _refused(call(work=P + 8), "aligned")
    _refused(call(rows=1 << 41), "2^40")
    _refused(call(out=(1 << 20) + 1), "2^20")
    _refused(call(rows=1 << 20, work=None), "d_workspace")


def test_python_calls_refuse_host_tensors():
    from marl_amd import act8, mxfp4

    x = torch.zeros(4, 40)
    with pytest.raises(ValueError, match="on the GPU"):
        mxfp4.quantize(x)
    with pytest.raises(ValueError, match="on the GPU"):
        act8.compress(x)
    with pytest.raises(ValueError, match="on the GPU"):
        act8.weight_grad(x, None)
    with pytest.raises(ValueError, match="on the GPU"):
        mxfp4.MXFP4(torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), 40)
    with pytest.raises(ValueError, match="on the GPU"):
        act8.Act8(torch.zeros(4, 40, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8), True)
    with pytest.raises(ValueError, match="MXFP4"):
        mxfp4.linear(x, x)


def test_the_command_refuses_what_does_not_fit():
    from marl_amd import train

    with pytest.raises(SystemExit):
        train.main(["--trunk-precision", "int4"])
    with pytest.raises(SystemExit):
        train.main(["--activation-bits", "16"])


def test_policy_options_leave_the_host_path_alone():
    """on the CPU (no HIP) an Agent with both options computes what it computes without them"""
    from marl_amd.policy import Agent
    from marl_amd.spaces import Box, Discrete

    torch.manual_seed(0)
    net = Agent(Box(-1, 1, (20,)), Discrete(7), 2, 1)
    x = torch.randn(6, 20)
    with torch.no_grad():
        want = net.get_prob(x).logits
    net.use_mxfp4_trunk().use_activation_checkpoints()
    with torch.no_grad():
        assert torch.equal(net.get_prob(x).logits, want)
    logits, value = net.logits_and_value(x)
    (logits.sum() + value.sum()).backward()
    assert net.network[0].weight.grad is not None
