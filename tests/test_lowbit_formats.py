"""What the low-bit formats leave of the numbers that the policy gives them, from the formats' definition (no GPU needed)."""
import glob
import os

import numpy as np
import pytest

import lowbit_reference as ref

REPLAYS = sorted(glob.glob(os.path.join(os.path.dirname(__file__), "golden", "replay_*.npz")))


def _observations(path):
    x = np.load(path)["obs"].astype(np.float64)
    return x.reshape(-1, x.shape[-1])


@pytest.mark.parametrize("path", REPLAYS, ids=[os.path.basename(p)[7:-4] for p in REPLAYS])
def test_recorded_observations(path):
    x = _observations(path)
    assert np.array_equal(x, np.rint(x)) and np.abs(x).max() <= 30
    assert np.array_equal(ref.act8(x, False)[2], x)  # whole numbers up to 127: 8 bits keep them
    four = ref.mxfp4(x)[2]
    before, after = ref.blocks(x), ref.blocks(four)
    top = np.abs(before).max(axis=2, keepdims=True)
    assert (np.abs(after - before) <= top / 4).all()
    small = np.broadcast_to(top <= 4, before.shape)
    assert np.array_equal(before[small], after[small])
    # ... and every recorded kitchen has blocks with larger numbers, which 4 bits do not keep
    assert top.max() > 4 and not np.array_equal(four, x)


@pytest.mark.parametrize("timer,reads,one,three", [(4, 4, 1, 3), (5, 4, 1, 3), (7, 6, 1, 3), (8, 8, 1, 3), (15, 12, 1, 3), (16, 16, 0, 4), (30, 24, 0, 4)])
def test_small_numbers_beside_a_timer(timer, reads, one, three):
    x = np.zeros((1, 32))
    x[0, :4] = timer, 1, 3, -1
    assert ref.mxfp4(x)[2][0, :4].tolist() == [reads, one, three, -one]
    x[0, 0] = 0
    assert np.array_equal(ref.mxfp4(x)[2], x)


@pytest.mark.parametrize("positive", [False, True])
def test_how_far_8_bits_are_off(positive):
    rng = np.random.default_rng(1)
    most = 255 if positive else 127
    x = np.abs(rng.standard_normal((4000, 64))) * np.exp(3 * rng.standard_normal((4000, 64)))
    if not positive:
        x *= rng.choice([-1.0, 1.0], x.shape)
    x[0] = np.linspace(0, most + 0.5, 64)  # the largest value that takes the next scale
    x[1] = np.linspace(0, np.nextafter(most + 0.5, 0), 64)
    x[2], x[3] = x[0] * 2.0 ** -133, x[0] * 2.0 ** 110  # the smallest scale, and near the largest
    x[4] = 3.4028234663852886e38 * np.linspace(0, 1, 64)
    _, byte, values = ref.act8(x, positive)
    step = np.exp2(byte.astype(np.float64) - 127)[:, :, None]
    before, after = ref.blocks(x), ref.blocks(values)
    top = np.abs(before).max(axis=2, keepdims=True)
    ordinary = top >= 2.0 ** (-119 if positive else -120)
    assert (top >= step * ((most + 0.5) / 2))[ordinary].all() and (step[~ordinary] == 2.0 ** -126).all()
    assert (step > top * 2 / (most + 1))[ordinary].any()  # 1/64 and 1/128 do not hold
    error = np.abs(after - before) / step
    raised = (before > 0) & (before < 0.5 * step) if positive else np.zeros(before.shape, bool)
    cut = (step == 2.0 ** (120 if positive else 121)) & (np.abs(before) > most * step)
    assert (error[~raised & ~cut] <= 0.5).all() and (error[raised | cut] <= 1.0).all()
    assert cut.any() and raised.any() == positive
    assert not positive or np.array_equal(values > 0, x > 0)
