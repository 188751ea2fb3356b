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
