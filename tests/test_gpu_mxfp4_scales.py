"""Products of MXFP4 operands whose scales lie far apart, against the formats' definition in 64 bits.  Tolerance as in
test_gpu_mxfp4.py: K terms in float32, off by at most K steps of 2^-23 of the sum of their magnitudes."""
import numpy as np
import pytest
import torch

import lowbit_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,cols,out", [(3, 202, 40), (5000, 202, 70), (5000, 512, 256), (3, 1500, 40), (70, 1500, 40), (9, 5, 20)])
def test_scales_that_cancel(rows, cols, out):
    """2^100 in x and 2^-100 in the weight leave the product's bits alone"""
    from marl_amd import mxfp4

    g = torch.Generator(device="cuda").manual_seed(rows + cols)
    x, w = torch.randn(rows, cols, device="cuda", generator=g), torch.randn(out, cols, device="cuda", generator=g)
    want = mxfp4.linear(x, mxfp4.quantize(w))
    for power in (100.0, -100.0):
        assert torch.equal(mxfp4.linear(x * 2.0 ** power, mxfp4.quantize(w * 2.0 ** -power)), want)
        assert torch.equal(mxfp4.linear(mxfp4.quantize(x * 2.0 ** power), mxfp4.quantize(w * 2.0 ** -power)), want)
    assert (mxfp4.linear(x * 2.0 ** 100, mxfp4.quantize(w * 2.0 ** 100), relu=True) == float("inf")).any()
    assert not mxfp4.linear(x * 2.0 ** -100, mxfp4.quantize(w * 2.0 ** -100)).any()


@pytest.mark.parametrize("rows,cols,out", [(7, 202, 40), (4000, 202, 70), (4000, 512, 256), (3, 1500, 40), (70, 1500, 40)])
def test_blocks_of_a_row_far_apart(rows, cols, out):
    from marl_amd import mxfp4

    rng = np.random.default_rng(rows + cols)

    def blocks(n):
        scale = np.exp2(rng.integers(-30, 31, size=(n, -(-cols // 32)))).repeat(32, axis=1)[:, :cols]
        return torch.from_numpy((rng.standard_normal((n, cols)) * scale).astype(np.float32))

    x, w = blocks(rows), blocks(out)
    got = mxfp4.linear(x.cuda(), mxfp4.quantize(w.cuda())).double().cpu().numpy()
    xv, wv = ref.mxfp4(x.double().numpy())[2], ref.mxfp4(w.double().numpy())[2]
    assert (np.abs(got - xv @ wv.T) <= cols * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)).all()
