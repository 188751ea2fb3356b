"""marl_amd.act8 against the format's definition in 64 bits (tests/lowbit_reference.py).

Codes, scales, read-back values and the cut gradient have to be equal.  A weight gradient's tolerance: each product of a
gradient and a kept value is exact before it is summed; M terms are summed in float32, off by at most M steps of 2^-23
(should the matrix unit truncate) of the sum of their magnitudes in the worst order.  Roundings of many sums do not all
fall to one side: the 2-norm over the whole gradient is held to 1e-6 of its own, which a bfloat16 (2^-9) or a
two-term split (2^-17) of the gradient would miss."""
import numpy as np
import pytest
import torch

import lowbit_reference as ref

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _x(rows, cols, dtype, seed, kind="normal"):
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((rows, cols))
    if kind == "obs":
        x = np.where(np.abs(x) > 0.9, np.rint(x * 1.3), 0.0)
    elif kind == "relu":
        x = np.maximum(x * np.exp2(rng.integers(-6, 6, size=(rows, 1))), 0.0)
    elif kind == "tail":
        x = x * np.exp(3 * rng.standard_normal((rows, cols)))
    return torch.from_numpy(x).to(dtype).cuda()


def _check(q, x64, positive):
    codes, byte, values = ref.act8(x64, positive)
    assert torch.equal(q.scales.cpu(), torch.from_numpy(byte))
    ok = np.repeat(byte != 255, ref.BLOCK, axis=1)[:, : codes.shape[1]]
    assert np.array_equal(q.codes.cpu().numpy()[ok], codes.astype(np.uint8)[ok])
    np.testing.assert_array_equal(q.dequantize().double().cpu().numpy(), values)
    # eight significant bits: bfloat16 holds every value
    np.testing.assert_array_equal(q.dequantize(torch.bfloat16).double().cpu().numpy(), values)
    return values


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 202), (512, 202), (33, 420), (300, 513), (1, 7)])
def test_codes_scales_and_values(rows, cols, dtype):
    from marl_amd import act8

    for kind, positive in (("normal", False), ("obs", False), ("tail", False), ("relu", True), ("normal", True)):
        x = _x(rows, cols, dtype, rows * 1000 + cols, kind)
        x64 = x.double().cpu().numpy()
        values = _check(act8.compress(x, nonnegative=positive), x64, positive)
        if kind == "obs":
            np.testing.assert_array_equal(values, x64)  # whole numbers are kept
        if positive:
            np.testing.assert_array_equal(values > 0, x64 > 0)  # and so is what the ReLU let through


def test_where_the_scale_steps_up():
    """127.5 steps (255.5) is where the next scale begins; one float32 step to either side, over the exponents"""
    from marl_amd import act8

    for positive, border in ((False, 127.5), (True, 255.5)):
        v = np.float32(border)
        rows = []
        for t in (np.nextafter(v, np.float32(0)), v, np.nextafter(v, np.float32(999)), np.float32(64 if not positive else 128)):
            row = np.zeros(32, dtype=np.float32)
            row[0], row[1:9] = t, [0.5, 1.5, 2.5, 63.5, 62.5, 1e-20, 0.49999997, 3]
            rows.append(row)
        for e in (-120, -10, 0, 33, 118):
            x = (np.stack(rows).astype(np.float64) * 2.0 ** e).astype(np.float32)
            for sign in (1, -1) if not positive else (1,):
                _check(act8.compress(torch.from_numpy(sign * x).cuda(), nonnegative=positive), (sign * x).astype(np.float64), positive)


def test_zeros_denormals_infinities_and_nans():
    from marl_amd import act8

    for positive in (False, True):
        x = torch.zeros(6, 96)
        x[1, 3] = 1e-40
        x[2, 40], x[2, 41] = float("inf"), 1.0
        x[3, 70] = float("nan")
        x[4, :] = -float("inf")
        x[5, 95] = 3.4e38
        q = act8.compress(x.cuda(), nonnegative=positive)
        _check(q, x.double().numpy(), positive)
        if positive:  # whatever the block reads as, its mask is the ReLU's
            on = q.codes.cpu() > 0
            assert on[2].nonzero().flatten().tolist() == [40, 41] and on[3, 70] and not on[4].any() and on[1, 3]


def test_rows_that_lie_apart_and_start_anywhere():
    from marl_amd import act8

    base = _x(40, 77, torch.bfloat16, 5)
    for view in (base[:, 3:60], base[::2, 1:34], base[5:6, 2:], base.t()[:, :39], base[:, :1]):
        _check(act8.compress(view), view.double().cpu().numpy(), False)


def _grad_case(rows, out, cols, dtype, kind, with_mask, seed, wild=False):
    from marl_amd import act8

    positive = kind == "relu"
    x = _x(rows, cols, torch.float32, seed, kind)
    act = act8.compress(x, nonnegative=positive)
    grad = (_x(rows, out, torch.float32, seed + 1, "tail") * (0.01 if dtype == torch.float16 else 1e-5)).to(dtype)
    mask = act8.compress(torch.relu(_x(rows, out, torch.float32, seed + 2)), nonnegative=True) if with_mask else None
    if wild:  # what the mask cuts does not count
        grad[mask.codes == 0] = float("nan")
        grad[0][mask.codes[0] == 0] = float("inf")
    gw, gb, masked = act8.weight_grad(grad, act, mask)
    g = grad.double().cpu().numpy()
    if with_mask:
        g = np.where(mask.codes.cpu().numpy() > 0, g, 0.0)
        assert masked.dtype == dtype
        np.testing.assert_array_equal(masked.double().cpu().numpy(), g)
    else:
        assert masked is None
    xv = act.dequantize().double().cpu().numpy()
    for got, want, size in ((gw, g.T @ xv, np.abs(g).T @ np.abs(xv)), (gb, g.sum(0), np.abs(g).sum(0))):
        got = got.double().cpu().numpy()
        assert got.shape == want.shape
        assert (np.abs(got - want) <= rows * 2.0 ** -23 * size + 2.0 ** -149).all()
        assert np.linalg.norm(got - want) <= 1e-6 * max(np.linalg.norm(want), 0.05 * np.linalg.norm(size) / max(rows, 1) ** 0.5)
    return grad, act, mask, gw, gb, masked


@pytest.mark.parametrize("rows,out,cols", [
    (1, 1, 1), (1, 512, 202), (2, 7, 5), (31, 8, 256), (32, 16, 64), (33, 17, 65), (64, 64, 64), (100, 512, 202), (2048, 512, 202),
    (2049, 256, 512), (5000, 8, 256), (777, 130, 300), (4096, 1, 512), (300, 250, 33), (70001, 20, 40)])
def test_weight_gradient(rows, out, cols):
    k = 0
    for dtype in DTYPES:
        for kind, with_mask in (("relu", True), ("obs", True), ("normal", False)):
            k += 1
            _grad_case(rows, out, cols, dtype, kind, with_mask, rows + out + cols + k, wild=with_mask and k % 2 == 0)


@pytest.mark.parametrize("rows,out,cols", [(9001, 300, 520), (33000, 130, 33), (16390, 512, 202), (131, 2000, 1500)])
def test_weight_gradient_in_the_largest_tiles(rows, out, cols):
    k = 0
    for dtype in DTYPES:
        for kind, with_mask in (("relu", True), ("normal", False)):
            k += 1
            _grad_case(rows, out, cols, dtype, kind, with_mask, rows + out + cols + k, wild=with_mask and dtype != torch.float16)


def test_rows_that_the_mask_leaves_empty():
    from marl_amd import act8

    grad = torch.full((130, 70), float("nan"), device="cuda")
    act = act8.compress(_x(130, 90, torch.float32, 1))
    mask = act8.compress(torch.zeros(130, 70, device="cuda"), nonnegative=True)
    gw, gb, masked = act8.weight_grad(grad, act, mask)
    assert not gw.any() and not gb.any() and not masked.any()


def test_infinite_and_nan_gradients_stay_in_their_features():
    from marl_amd import act8

    x = torch.rand(200, 100, device="cuda") + 0.5
    grad = _x(200, 80, torch.float32, 2)
    clean = act8.weight_grad(grad, act8.compress(x, nonnegative=True))
    grad[50, 7], grad[60, 9], grad[61, 11] = float("nan"), float("inf"), -float("inf")
    gw, gb, _ = act8.weight_grad(grad, act8.compress(x, nonnegative=True))
    assert torch.isnan(gw[7]).all() and (gw[9] == float("inf")).all() and (gw[11] == -float("inf")).all()
    assert torch.isnan(gb[7]) and gb[9] == float("inf") and gb[11] == -float("inf")
    keep = [o for o in range(80) if o not in (7, 9, 11)]
    assert torch.equal(gw[keep], clean[0][keep]) and torch.equal(gb[keep], clean[1][keep])


def test_largest_gradients_do_not_overflow_in_their_parts():
    from marl_amd import act8

    x = torch.zeros(40, 33, device="cuda")
    x[3, 5] = 0.25
    grad = torch.zeros(40, 17, device="cuda")
    grad[3, 2], grad[3, 4] = 3.4028234663852886e38, 1.17549435e-38
    gw, gb, _ = act8.weight_grad(grad, act8.compress(x))
    assert gw[2, 5].item() == 3.4028234663852886e38 * 0.25 and gb[2].item() == 3.4028234663852886e38
    assert gw[2].count_nonzero() == 1 and torch.isfinite(gw).all()


def test_kept_values_up_to_the_largest():
    """128 steps of the largest scale are no float32, but no value is 128 steps: what the gradient reads is what is read back"""
    from marl_amd import act8

    x = torch.zeros(64, 96, device="cuda")
    x[:, 0], x[:, 1], x[:, 33], x[5, 70] = 3.4028234663852886e38, 1e37, 3.0, -1.7014118346046923e38
    for rows, out in ((64, 1), (64, 20), (3, 20)):
        act = act8.compress(x[:rows])
        g = torch.zeros(rows, out, device="cuda")
        g[min(5, rows - 1)] = 2.0 ** -100
        gw, _, _ = act8.weight_grad(g, act)
        want = act.dequantize()[min(5, rows - 1)] * 2.0 ** -100  # one term: exact
        assert torch.equal(gw, want.expand(out, 96))
    # scales that compressing never writes read as the formula says
    for byte in (0, 1, 249, 254):
        codes = torch.full((8, 32), 128, dtype=torch.uint8, device="cuda")
        codes[2, 3] = 129
        act = act8.Act8(codes, torch.full((8, 1), byte, dtype=torch.uint8, device="cuda"), False)
        value = 2.0 ** (byte - 127)
        assert act.dequantize()[2, 3].item() == value and act.dequantize().count_nonzero() == 1
        gw, _, _ = act8.weight_grad(torch.full((8, 5), 2.0 ** -20 if byte > 200 else 2.0 ** 20, device="cuda"), act)
        if byte:  # a matrix unit may take bfloat16's denormals for zeros
            assert (gw[:, 3] == value * (2.0 ** -20 if byte > 200 else 2.0 ** 20)).all()
        assert gw.count_nonzero() == (5 if byte else gw[:, 3].count_nonzero())


def test_offsets_beyond_32_bits():
    from marl_amd import act8

    rows, cols, last = 4_300_000, 512, 70
    x = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    x.zero_()
    x[-last:] = _x(last, cols, torch.float16, 1)
    act, small = act8.compress(x), act8.compress(x[-last:].clone())
    assert torch.equal(act.codes[-last:], small.codes) and torch.equal(act.scales[-last:], small.scales)
    back = act.dequantize(torch.bfloat16)
    assert torch.equal(back[-last:], small.dequantize(torch.bfloat16)) and not back[:-last].any()
    del back
    mask = act8.Act8(torch.ones(rows, cols, dtype=torch.uint8, device="cuda"), act.scales, True)
    mask.codes[-1, ::2] = 0
    x.zero_()
    x[-last:] = _x(last, cols, torch.float16, 2)  # now the gradient
    gw, gb, masked = act8.weight_grad(x, act, mask)
    assert torch.equal(masked[:-1], x[:-1]) and not masked[-1, ::2].any() and torch.equal(masked[-1, 1::2], x[-1, 1::2])
    g, xv = masked[-last:].double(), small.dequantize().double()
    for got, want, size in ((gw.double(), g.t() @ xv, g.abs().t() @ xv.abs()), (gb.double(), g.sum(0), g.abs().sum(0))):
        assert ((got - want).abs() <= last * 2.0 ** -23 * size).all()


def test_every_output_is_written_and_nothing_else():
    from marl_amd import _lib, act8
    from marl_amd.mxfp4 import _p

    L = _lib.lib()
    for rows, out, cols in ((37, 65, 202), (700, 9, 33), (3000, 130, 70)):
        grad, act, mask, gw, gb, masked = _grad_case(rows, out, cols, torch.float32, "relu", True, 3)
        need = L.marl_act_weight_grad_workspace_bytes(rows, out, cols)
        bufs = [torch.full((n + 128,), 7.0, device="cuda") for n in (out * cols, out, rows * out)]
        work = torch.full((need + 64,), 9, dtype=torch.uint8, device="cuda")
        _lib.check(L.marl_act_weight_grad(_p(grad), 0, rows, out, _p(act.codes), _p(act.scales), cols, 1, _p(mask.codes), _p(bufs[2][64:]),
                                          _p(bufs[0][64:]), _p(bufs[1][64:]), _p(work), torch.cuda.current_stream().cuda_stream), "marl_act_weight_grad")
        for buf, want in zip(bufs, (gw, gb, masked)):
            assert torch.equal(buf[64:-64], want.flatten()) and (buf[:64] == 7).all() and (buf[-64:] == 7).all()
        assert (work[need:] == 9).all()


def test_same_bits_every_time_on_any_stream_and_from_a_graph():
    from marl_amd import act8

    rows, out, cols = 3000, 130, 202
    x, y = _x(rows, cols, torch.float32, 1), _x(rows, out, torch.float32, 2, "relu")
    grad = _x(rows, out, torch.float32, 3)

    def passes():
        return act8.weight_grad(grad, act8.compress(x), act8.compress(y, nonnegative=True))

    want = passes()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        got = passes()
    torch.cuda.current_stream().wait_stream(other)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, capture_error_mode="thread_local"):
        out3 = passes()
    for step in range(4):
        x.copy_(_x(rows, cols, torch.float32, 10 + step))
        grad.copy_(_x(rows, out, torch.float32, 30 + step))
        want = passes()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out3, want))


def test_two_calls_at_once_do_not_share_anything():
    from marl_amd import act8

    cases = []
    for k, (rows, out, cols) in enumerate(((30000, 256, 512), (30000, 8, 256), (2048, 70, 202))):
        x, y = _x(rows, cols, torch.float32, k), _x(rows, out, torch.float32, 10 + k, "relu")
        cases.append((_x(rows, out, torch.float32, 20 + k), act8.compress(x), act8.compress(y, nonnegative=True)))
    want = [act8.weight_grad(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for case, stream in zip(cases, streams):
            with torch.cuda.stream(stream):
                got.append(act8.weight_grad(*case))
    torch.cuda.synchronize()
    for k, r in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(r, want[k % len(cases)]))


def test_no_rows():
    from marl_amd import act8

    act = act8.compress(torch.zeros(0, 40, device="cuda"))
    gw, gb, masked = act8.weight_grad(torch.zeros(0, 8, device="cuda"), act, act8.compress(torch.zeros(0, 8, device="cuda"), True))
    assert gw.shape == (8, 40) and not gw.any() and not gb.any() and masked.shape == (0, 8)
    assert act.dequantize().shape == (0, 40)


def test_refusals():
    from marl_amd import act8

    x = torch.zeros(4, 40, device="cuda")
    for bad in (x.double(), x.cpu(), x[0], x[:, :0], "x"):
        with pytest.raises(ValueError):
            act8.compress(bad)
    act = act8.compress(x)
    grad = torch.zeros(4, 8, device="cuda")
    mask = act8.compress(torch.zeros(4, 8, device="cuda"), nonnegative=True)
    for args in ((grad[:3], act), (grad.double(), act), (grad, x), (grad, act, act), (grad[:, :7], act, mask),
                 (grad, act, act8.Act8(mask.codes, mask.scales, False))):
        with pytest.raises(ValueError):
            act8.weight_grad(*args)
    with pytest.raises(ValueError):
        act8.Act8(act.codes, act.scales[:, :1], True)
    with pytest.raises(ValueError):
        act8.Act8(act.codes.int(), act.scales, True)
    with pytest.raises(ValueError):
        act.dequantize(torch.float64)
    with pytest.raises(ValueError):  # a C int counts the columns
        act8.compress(torch.empty(1, (1 << 32) + 32, dtype=torch.float16, device="cuda"))
