"""The weight gradient in every tile that it can take, at output and input counts that fill none of them.

Inputs and tolerances are those of test_gpu_act8.py.  Its float16 gradients have a tail that now and then passes 65504 and is
infinite: a feature with such a gradient has to read as the sum in 64 bits does, infinite or no number."""
import numpy as np
import pytest
import torch

from test_gpu_act8 import DTYPES, _x


def _cut(rows, out, cols):
    """(output features, input features, splits of the rows) of a tile, as the entry point's rule on sizes picks them"""
    steps = -(-rows // 32)

    def tiles(bo, bi):
        return -(-out // bo) * -(-cols // bi)

    bo, bi = (16, 256) if out <= 16 or cols < 4 else (128, 256) if cols > 64 and tiles(128, 256) * (steps // 4) >= 256 else (64, 64)
    splits = max(1, (256 if bo == 128 else 512) // tiles(bo, bi))
    least = (4 if steps > 512 else 2) if bo == 16 else 4
    splits = min(splits, -(-steps // least))
    each = -(-steps // splits)
    return bo, bi, -(-steps // each)


LARGE = [(33000, 131, 77), (20001, 301, 259), (70001, 130, 65), (16390, 515, 201), (33001, 17, 303)]
SMALL = [(300, 33, 5), (2049, 130, 33), (131, 2001, 1503), (1, 17, 4)]
HEADS = [(777, 15, 303), (65003, 7, 257), (300, 16, 4)]
NARROW = [(5000, 100, 1), (300, 33, 2), (777, 250, 3), (4001, 3, 66), (65, 1, 300), (31, 2, 2)]


@pytest.mark.parametrize("sizes,tile", [(LARGE, (128, 256)), (SMALL, (64, 64)), (HEADS, (16, 256)), (NARROW, (16, 256))])
def test_which_tile_a_size_takes(sizes, tile):
    """the rule above is the library's: so is the workspace, which is what its splits need"""
    from marl_amd import _lib

    L = _lib.lib()
    for rows, out, cols in sizes:
        bo, bi, splits = _cut(rows, out, cols)
        assert (bo, bi) == tile
        need = 0 if splits == 1 else splits * (out * cols + out) * 4
        assert L.marl_act_weight_grad_workspace_bytes(rows, out, cols) == need, (rows, out, cols)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,out,cols", NARROW + HEADS + SMALL + LARGE)
def test_sizes_that_fill_no_tile(rows, out, cols, dtype):
    from marl_amd import act8

    for k, (kind, with_mask) in enumerate((("relu", True), ("obs", True), ("normal", False))):
        seed = rows + out + cols + k
        act = act8.compress(_x(rows, cols, torch.float32, seed, kind), nonnegative=kind == "relu")
        grad = (_x(rows, out, torch.float32, seed + 1, "tail") * (0.01 if dtype == torch.float16 else 1e-5)).to(dtype)
        mask = act8.compress(torch.relu(_x(rows, out, torch.float32, seed + 2)), nonnegative=True) if with_mask else None
        if with_mask and k == 0:  # what the mask cuts does not count
            grad[mask.codes == 0] = float("nan")
        gw, gb, masked = act8.weight_grad(grad, act, mask)
        gw2, gb2, none = act8.weight_grad(grad, act, mask, want_masked=False)
        assert none is None and torch.equal(gw.view(torch.int32), gw2.view(torch.int32)) and torch.equal(gb.view(torch.int32), gb2.view(torch.int32))
        g = grad.double().cpu().numpy()
        if with_mask:
            g = np.where(mask.codes.cpu().numpy() > 0, g, 0.0)
            np.testing.assert_array_equal(masked.double().cpu().numpy(), g)
        xv = act.dequantize().double().cpu().numpy()
        with np.errstate(invalid="ignore"):
            pairs = ((gw, g.T @ xv, np.abs(g).T @ np.abs(xv)), (gb, g.sum(0), np.abs(g).sum(0)))
        for got, want, size in pairs:
            got, real = got.double().cpu().numpy(), np.isfinite(want)
            np.testing.assert_array_equal(got[~real], want[~real])
            got, want, size = got[real], want[real], size[real]
            assert (np.abs(got - want) <= rows * 2.0 ** -23 * size + 2.0 ** -149).all()
            assert np.linalg.norm(got - want) <= 1e-6 * max(np.linalg.norm(want), 0.05 * np.linalg.norm(size) / max(rows, 1) ** 0.5)
