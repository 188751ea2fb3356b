"""Bad arguments to `marl_act_param_grad` come back as errors before anything touches the GPU (no GPU needed)."""

P = 1 << 20  # an address nobody follows: every call here is refused


def test_parameter_gradients():
    from marl_amd import _lib

    L = _lib.lib()

    def refused(words, grad=P, gt=0, rows=4, out=8, codes=P, scales=P, cols=64, mask=2 * P, gw=P, gb=P, work=P):
        assert L.marl_act_param_grad(grad, gt, rows, out, codes, scales, cols, 0, mask, gw, gb, work, None) == -1
        message = L.marl_last_error().decode()
        assert words in message, message

    refused("positive", rows=0)
    refused("positive", cols=-1)
    refused("grad_type", gt=3)
    refused("NULL argument to marl_act_param_grad", grad=None)
    refused("NULL argument to marl_act_param_grad", gb=None)
    refused("aligned", grad=P + 2)
    refused("aligned", gw=P + 1)
    refused("aligned", work=P + 4)
    refused("2^40", rows=1 << 41)
    refused("2^20", out=(1 << 20) + 1)
    refused("d_workspace", rows=1 << 20, work=None)
    refused("d_workspace", rows=1 << 20, work=None, mask=None)
