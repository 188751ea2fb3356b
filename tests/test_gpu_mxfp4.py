"""marl_amd.mxfp4 against the formats' definition in 64 bits (tests/lowbit_reference.py).

Codes, scales and read-back values have to be equal.  A product's tolerance: every 4-bit product is exact, a sum of K of
them in float32 is off by at most K steps of 2^-23 (should the matrix unit truncate) of the sum of their magnitudes, the
bias adds one rounding, and a 16-bit result one of eps / 2 of its type."""
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
    elif kind == "wide":
        x = x * np.exp2(rng.integers(-10, 8, size=(rows, 1)))
    return torch.from_numpy(x).to(dtype).cuda()


def _check_codes(q, x64):
    codes, byte, values = ref.mxfp4(x64)
    assert torch.equal(q.scales.cpu(), torch.from_numpy(byte))
    ok = byte != 255
    got = q.codes.cpu().numpy().reshape(byte.shape + (16,))
    want = ref.pack(codes).reshape(byte.shape + (16,))
    # the sign of a value that rounds to zero is kept by neither side's definition: compare what the codes stand for
    def canon(c):
        lo, hi = c & 15, c >> 4
        lo, hi = np.where(lo == 8, 0, lo), np.where(hi == 8, 0, hi)
        return lo | (hi << 4)
    assert np.array_equal(canon(got)[ok], canon(want)[ok])
    return values


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 202), (512, 202), (33, 420), (1, 6464), (300, 513)])
def test_codes_scales_and_values(rows, cols, dtype):
    from marl_amd import mxfp4

    for kind in ("normal", "obs", "wide"):
        x = _x(rows, cols, dtype, rows * 1000 + cols, kind)
        q = mxfp4.quantize(x)
        values = _check_codes(q, x.double().cpu().numpy())
        np.testing.assert_array_equal(q.dequantize().double().cpu().numpy(), values)
        np.testing.assert_array_equal(q.dequantize(dtype).double().cpu().numpy(), torch.from_numpy(values).to(dtype).double().numpy())


def test_every_border_and_its_neighbours():
    """the midpoints between neighbouring values, one float32 step to either side, at several scales; 8 - 1 step saturates"""
    from marl_amd import mxfp4

    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0, 7.9999995, 6.5]
    v = np.array([f for m in mids for f in (np.nextafter(np.float32(m), np.float32(0)), np.float32(m), np.nextafter(np.float32(m), np.float32(9)))],
                 dtype=np.float32)
    v = v[v < 8]
    for e in (-126, -120, -3, 0, 5, 100, 125):
        for sign in (1, -1):
            x = np.zeros((v.size, 32), dtype=np.float32)
            x[:, 0], x[:, 17] = np.float32(4.0), sign * v
            x = (x.astype(np.float64) * 2.0 ** e).astype(np.float32)
            q = mxfp4.quantize(torch.from_numpy(x).cuda())
            values = _check_codes(q, x)
            np.testing.assert_array_equal(q.dequantize().double().cpu().numpy(), values)


def test_zeros_denormals_infinities_and_nans():
    from marl_amd import mxfp4

    x = torch.zeros(6, 96)
    x[1, 3] = 1e-40  # denormal: below the smallest scale, rounds to 0
    x[2, 40] = float("inf")
    x[3, 70] = float("nan")
    x[4, :] = -float("inf")
    x[5, 95] = 3.4e38
    q = mxfp4.quantize(x.cuda())
    values = _check_codes(q, x.double().numpy())
    got = q.dequantize().double().cpu().numpy()
    np.testing.assert_array_equal(got, values)
    assert np.isnan(got[2, 32:64]).all() and not np.isnan(got[2, :32]).any() and np.isnan(got[4]).all()


def test_rows_that_lie_apart_and_start_anywhere():
    from marl_amd import mxfp4

    base = _x(40, 77, torch.bfloat16, 5)
    for view in (base[:, 3:60], base[::2, 1:34], base[5:6, 2:], base.t()[:, :39], base[:, :1]):
        q = mxfp4.quantize(view)
        _check_codes(q, view.double().cpu().numpy())


def _linear_case(x, w, bias, relu, out_dtype):
    from marl_amd import mxfp4

    wq = mxfp4.quantize(w)
    y = mxfp4.linear(x, wq, bias, relu=relu, out_dtype=out_dtype)
    xv = ref.mxfp4(x.double().cpu().numpy())[2]
    wv = ref.mxfp4(w.double().cpu().numpy())[2]
    want = xv @ wv.T
    room = x.shape[1] * 2.0 ** -23 * (np.abs(xv) @ np.abs(wv).T)
    if bias is not None:
        want = want + bias.double().cpu().numpy()
    room = room + 2.0 ** -24 * (np.abs(want) + room)
    if relu:
        want = np.maximum(want, 0.0)
    if out_dtype != torch.float32:
        room = room + torch.finfo(out_dtype).eps / 2 * (np.abs(want) + room) + float(torch.finfo(out_dtype).smallest_normal)
    got = y.double().cpu().numpy()
    assert got.shape == want.shape and y.dtype == out_dtype
    off = np.abs(got - want) - room
    assert (off <= 0).all(), (float(off.max()), np.unravel_index(off.argmax(), off.shape))
    return wq, y


@pytest.mark.parametrize("rows,cols,out", [
    (1, 1, 1), (1, 202, 512), (2, 5, 7), (32, 202, 512), (33, 202, 65), (17, 32, 64), (100, 129, 63), (513, 420, 250),
    (64, 512, 256), (5, 384, 1000), (4099, 202, 8), (31, 33, 513), (0, 202, 8),
    (1, 513, 512), (1, 6464, 512), (16, 1000, 70), (17, 1000, 70), (200, 2000, 130), (3, 100003, 9), (65, 545, 33)])
def test_product_of_float_rows(rows, cols, out):
    k = 0
    for dtype in DTYPES:
        for relu, with_bias in ((True, True), (False, False)):
            k += 1
            x = _x(rows, cols, dtype, rows + 3 * cols + k, ("obs", "normal", "wide")[k % 3])
            w = _x(out, cols, torch.float32, out + 7 * cols) * 0.06
            bias = 0.1 * _x(1, out, torch.float32, k)[0] if with_bias else None
            _linear_case(x, w, bias, relu, DTYPES[(k + 1) % 3])
            _linear_case(x, w, bias, relu, torch.float32)


@pytest.mark.parametrize("cols", [8, 202, 256, 257, 512])
@pytest.mark.parametrize("out", [8, 200, 512])
def test_many_rows_equal_their_pieces(cols, out):
    """the forms that many rows take add in the order of those that few take, which are held to 64 bits above"""
    from marl_amd import mxfp4

    rows, piece = 20011, 4000
    w, b = mxfp4.quantize(_x(out, cols, torch.float32, 1)), torch.randn(out, device="cuda")
    for dtype in DTYPES:
        x = _x(rows, cols, dtype, 2)
        x[777], x[778, 0], x[-1, -1] = 0.0, float("nan"), float("inf")
        q = mxfp4.quantize(x)
        parts = [mxfp4.MXFP4(c.contiguous(), s.contiguous(), cols) for c, s in zip(q.codes.split(piece), q.scales.split(piece))]
        for out_dtype in (torch.float32, torch.bfloat16, torch.float16):
            want = torch.cat([mxfp4.linear(v, w, b, relu=True, out_dtype=out_dtype) for v in x.split(piece)])
            for rows_in in (x, q):
                torch.testing.assert_close(mxfp4.linear(rows_in, w, b, relu=True, out_dtype=out_dtype), want, rtol=0, atol=0, equal_nan=True)
            small = torch.cat([mxfp4.linear(v, w, b, relu=True, out_dtype=out_dtype) for v in parts])
            torch.testing.assert_close(small, want, rtol=0, atol=0, equal_nan=True)
        want = mxfp4.quantize(mxfp4.linear(x, w, b))
        for rows_in in (x, q):
            got = mxfp4.linear(rows_in, w, b, out_dtype="mxfp4")
            assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
        for v, c, s in zip(parts, want.codes.split(piece), want.scales.split(piece)):
            got = mxfp4.linear(v, w, b, out_dtype="mxfp4")
            assert torch.equal(got.codes, c) and torch.equal(got.scales, s)


@pytest.mark.parametrize("rows,cols,out", [(1, 202, 512), (40, 202, 512), (130, 512, 33), (9, 700, 96), (70, 1500, 40)])
def test_layers_in_a_row_quantised_between(rows, cols, out):
    """out_dtype="mxfp4" holds what quantising the float32 result would give, and is the next layer's x; an x that is
    quantised beforehand gives the bits of one that is quantised within"""
    from marl_amd import mxfp4

    x, w = _x(rows, cols, torch.float32, 1), _x(out, cols, torch.float32, 2) * 0.06
    bias = 0.1 * _x(1, out, torch.float32, 3)[0]
    wq = mxfp4.quantize(w)
    for relu in (False, True):
        y = mxfp4.linear(x, wq, bias, relu=relu)
        yq, want = mxfp4.linear(x, wq, bias, relu=relu, out_dtype="mxfp4"), mxfp4.quantize(y)
        assert torch.equal(yq.codes, want.codes) and torch.equal(yq.scales, want.scales)
        assert torch.equal(mxfp4.linear(mxfp4.quantize(x), wq, bias, relu=relu), y)
        w2 = mxfp4.quantize(_x(11, out, torch.float32, 4))
        assert torch.equal(mxfp4.linear(yq, w2), mxfp4.linear(y, w2))


@pytest.mark.parametrize("cols", [64, 202, 1000])
def test_a_nan_reaches_its_row_and_its_feature_only(cols):
    from marl_amd import mxfp4

    x, w = _x(50, cols, torch.float32, 1), _x(70, cols, torch.float32, 2)
    clean = mxfp4.linear(x, mxfp4.quantize(w), relu=True)
    x[7, cols - 1] = float("nan")
    x[20, 3] = float("inf")
    w[33, 40] = float("nan")
    y = mxfp4.linear(x, mxfp4.quantize(w), relu=True)
    bad = torch.zeros_like(y, dtype=torch.bool)
    bad[7], bad[20], bad[:, 33] = True, True, True
    assert torch.equal(torch.isnan(y), bad)
    assert torch.equal(y[~bad], clean[~bad])


def test_every_output_is_written_and_nothing_else():
    from marl_amd import _lib, mxfp4

    for rows, cols, out in ((37, 202, 65), (3, 700, 9), (16, 520, 64)):
        x, wq = _x(rows, cols, torch.float32, 1), mxfp4.quantize(_x(out, cols, torch.float32, 2))
        room = torch.full((rows * out + 512,), 7.0, device="cuda")
        L = _lib.lib()
        p = mxfp4._p
        need = L.marl_mx_linear_workspace_bytes(0, rows, cols, out)
        work = torch.full((need + 256,), 9, dtype=torch.uint8, device="cuda")
        _lib.check(L.marl_mx_linear(p(x), None, 0, rows, cols, 0, p(wq.codes), p(wq.scales), out, None, 0, p(room[256:]), None, 0,
                                    p(work), torch.cuda.current_stream().cuda_stream), "marl_mx_linear")
        assert torch.equal(room[256:256 + rows * out].view(rows, out), mxfp4.linear(x, wq))
        assert (room[:256] == 7).all() and (room[256 + rows * out:] == 7).all() and (work[need:] == 9).all()


def test_same_bits_every_time_on_any_stream_and_from_a_graph():
    from marl_amd import mxfp4

    cases = [(32, 202, 512), (1, 6464, 512), (300, 1000, 70)]
    for rows, cols, out in cases:
        x, w = _x(rows, cols, torch.float32, 1), _x(out, cols, torch.float32, 2)
        bias = _x(1, out, torch.float32, 3)[0]
        wq = mxfp4.quantize(w)
        y = mxfp4.linear(x, wq, bias, relu=True)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            y2 = mxfp4.linear(x, wq, bias, relu=True)
        torch.cuda.current_stream().wait_stream(other)
        assert torch.equal(y, y2)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, capture_error_mode="thread_local"):
            mxfp4.quantize(w, out=wq)
            y3 = mxfp4.linear(x, wq, bias, relu=True)
        for step in range(4):
            x.copy_(_x(rows, cols, torch.float32, 10 + step))
            w.copy_(_x(out, cols, torch.float32, 20 + step))
            want = mxfp4.linear(x, mxfp4.quantize(w), bias, relu=True)
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(y3, want)


def test_two_calls_at_once_do_not_share_anything():
    from marl_amd import mxfp4

    x = [_x(2, 50000, torch.float32, k) for k in range(2)]
    w = [mxfp4.quantize(_x(64, 50000, torch.float32, 10 + k)) for k in range(2)]
    want = [mxfp4.linear(x[k], w[k]) for k in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(mxfp4.linear(x[k], w[k]))
    torch.cuda.synchronize()
    for k in range(2):
        assert all(torch.equal(y, want[k]) for y in got[k])


@pytest.mark.parametrize("cols", [5, 202, 700])
def test_no_rows(cols):
    from marl_amd import mxfp4

    w = mxfp4.quantize(torch.ones(9, cols, device="cuda"))
    x = torch.zeros(0, cols, device="cuda")
    q = mxfp4.quantize(x)
    assert q.shape == (0, cols) and q.dequantize().shape == (0, cols)
    for rows in (x, q):
        assert mxfp4.linear(rows, w).shape == (0, 9) and mxfp4.linear(rows, w, out_dtype="mxfp4").shape == (0, 9)


def test_offsets_beyond_32_bits():
    from marl_amd import mxfp4

    rows, cols, last = 4_300_000, 512, 40  # many rows: values, codes, results behind 2^32 bytes, values behind 2^31 elements
    x = torch.empty(rows, cols, dtype=torch.float16, device="cuda")
    x.zero_()
    x[-last:] = torch.from_numpy(np.random.default_rng(1).standard_normal((last, cols))).half()
    w = mxfp4.quantize(torch.from_numpy(np.random.default_rng(2).standard_normal((512, cols))).float().cuda())
    q, small = mxfp4.quantize(x), mxfp4.quantize(x[-last:].clone())
    assert torch.equal(q.codes[-last:], small.codes) and torch.equal(q.scales[-last:], small.scales) and not q.codes[:-last].any()
    back = q.dequantize(torch.float16)
    assert torch.equal(back[-last:], small.dequantize(torch.float16)) and not back[:-last].any()
    del back
    y, want = mxfp4.linear(x, w, out_dtype=torch.float16), mxfp4.linear(small, w, out_dtype=torch.float16)
    assert torch.equal(y[-last:], want) and not y[:-last].any()
    del y
    y = mxfp4.linear(q, w, out_dtype="mxfp4")
    want = mxfp4.linear(small, w, out_dtype="mxfp4")
    assert torch.equal(y.codes[-last:], want.codes) and torch.equal(y.scales[-last:], want.scales)


@pytest.mark.parametrize("rows", [1, 20])
def test_a_weight_beyond_32_bits(rows):
    """rows of 2^26 values, the last of them in the row's last stretch: 4.7 GB of codes"""
    from marl_amd import mxfp4

    out, cols = 140, (1 << 26) - 7
    w = torch.zeros(out, cols, dtype=torch.float16, device="cuda")
    x = torch.zeros(rows, cols, dtype=torch.float16, device="cuda")
    w[:, 3], w[:, -5:], x[:, 3] = 1.0, torch.arange(1, 6, device="cuda").half() / 2, 2.0
    w[-1, -1] = 6.0
    x[:, -5:] = torch.tensor([1.0, 2.0, 0.5, 4.0, 3.0], device="cuda").half()
    # The rows of 0.5 .. 2.5 have a scale of 1/2, of which they are 1, 2, 3, 4 and 5, halfway between 4 and 6: the even code is
    # 4's, so 2.5 reads as 2.  The last row (a scale of 1) and x are MXFP4 numbers as they stand.
    read = w[:, -5:].float()
    read[:-1, 4] = 2.0
    want = read @ x[:, -5:].float().t() + 2.0
    assert torch.equal(mxfp4.linear(x, mxfp4.quantize(w)), want.t())


def test_refusals():
    from marl_amd import mxfp4

    x = torch.zeros(4, 40, device="cuda")
    w = mxfp4.quantize(torch.zeros(8, 40, device="cuda"))
    for bad in (x.double(), x.cpu(), x[0], x[:, :0], "x"):
        with pytest.raises(ValueError):
            mxfp4.quantize(bad)
    with pytest.raises(ValueError):
        mxfp4.linear(x[:, :39], w)
    with pytest.raises(ValueError):
        mxfp4.linear(x, w, bias=torch.zeros(7, device="cuda"))
    with pytest.raises(ValueError):
        mxfp4.linear(x, w, bias=torch.zeros(8, device="cuda", dtype=torch.float64))
    with pytest.raises(ValueError):
        mxfp4.linear(x, w, out_dtype=torch.float64)
    with pytest.raises(ValueError):
        mxfp4.linear(x, x)
    with pytest.raises(ValueError, match="no gradient"):
        mxfp4.linear(x.clone().requires_grad_(), w)
    with pytest.raises(ValueError):
        mxfp4.MXFP4(w.codes, w.scales, 100)
    with pytest.raises(ValueError):
        mxfp4.MXFP4(w.codes[:, :16], w.scales, 40)
    with pytest.raises(ValueError):
        mxfp4.quantize(x, out=w)
    with pytest.raises(ValueError):  # a C int counts the columns
        mxfp4.quantize(torch.empty(1, (1 << 32) + 32, dtype=torch.float16, device="cuda"))
    learned = torch.zeros(w.shape[0], device="cuda", requires_grad=True)
    with pytest.raises(ValueError):
        mxfp4.linear(x, w, learned)
    with torch.no_grad():
        mxfp4.linear(x, w, learned)
