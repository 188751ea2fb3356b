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


def test_column_sums():
    from marl_amd import _lib

    L = _lib.lib()

    def refused(words, x=P, kind=0, rows=4, cols=8, sums=P, work=P):
        assert L.marl_column_sums(x, kind, rows, cols, sums, work, None) == -1
        message = L.marl_last_error().decode()
        assert words in message, message

    refused("positive", rows=0)
    refused("positive", cols=-1)
    refused("x_type", kind=3)
    refused("NULL", x=None)
    refused("NULL", sums=None)
    refused("aligned", x=P + 2)
    refused("aligned", sums=P + 1)
    refused("aligned", work=P + 8)
    refused("2^40", rows=1 << 40)
    refused("2^20", cols=(1 << 20) + 1)
    refused("d_workspace", rows=1 << 16, work=None)
    assert L.marl_column_sums_workspace_bytes(4, 8) == 0 and L.marl_column_sums_workspace_bytes(0, 8) == 0
    assert L.marl_column_sums_workspace_bytes(131072, 512) == 512 * 512 * 4
