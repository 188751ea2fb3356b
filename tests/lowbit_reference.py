"""The low-bit number formats in 64 bits on the CPU, from their definitions (numpy, no code of the package)."""
import numpy as np

BLOCK = 32
E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=np.float64)


def blocks(x):
    """float64 [rows, blocks, 32], padded with zeros"""
    x = np.asarray(x, dtype=np.float64)
    pad = -x.shape[1] % BLOCK
    return np.concatenate([x, np.zeros((x.shape[0], pad))], axis=1).reshape(x.shape[0], (x.shape[1] + pad) // BLOCK, BLOCK)


def _floor_log2(v):
    with np.errstate(divide="ignore", invalid="ignore"):
        return np.where(v > 0, np.frexp(np.where(np.isfinite(v), v, 1.0))[1] - 1, -(10 ** 6))


def mxfp4(x):
    """(codes uint8 [rows, blocks, 32], scale bytes uint8 [rows, blocks], values float64 [rows, cols])"""
    b = blocks(x)
    top = np.abs(b).max(axis=2)
    bad = ~np.isfinite(top)
    e = np.maximum(_floor_log2(top) - 2, -126)
    v = np.where(bad[..., None], 0.0, b) / np.exp2(e)[..., None]
    size = np.abs(v)
    border = (E2M1[1:] + E2M1[:-1]) / 2
    low = np.searchsorted(border, size, side="left")  # borders below the size
    tie = np.searchsorted(border, size, side="right") > low
    code = np.where(tie & (low % 2 == 1), low + 1, low)
    values = np.where(v < 0, -1.0, 1.0) * E2M1[code] * np.exp2(e)[..., None]
    values = np.where(bad[..., None], np.nan, values)
    codes = (code | ((v < 0) << 3)).astype(np.uint8)
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    return codes, byte, values.reshape(b.shape[0], b.shape[1] * BLOCK)[:, : np.shape(x)[1]]


def pack(codes):
    """[rows, blocks, 32] codes to bytes, the lower half first"""
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).reshape(codes.shape[0], -1)


def act8(x, positive):
    """(codes uint8 [rows, cols], scale bytes uint8 [rows, blocks], values float64 [rows, cols])"""
    b = blocks(x)
    if positive:
        b = np.where(b < 0, 0.0, b)
    most = 255 if positive else 127
    top = np.abs(b).max(axis=2)
    bad = ~np.isfinite(top)
    e = _floor_log2(top) - (7 if positive else 6)
    with np.errstate(invalid="ignore"):
        e = np.where(np.rint(np.where(bad, 0.0, top) / np.exp2(e.astype(np.float64))) > most, e + 1, e)
    e = np.clip(e, -126, 120 if positive else 121)  # the largest scale of which `most` are finite in float32
    scale = np.exp2(e.astype(np.float64))[..., None]
    with np.errstate(invalid="ignore", over="ignore"):
        code = np.clip(np.rint(np.where(np.isfinite(b), b, 0.0) / scale), -most, most)
    if positive:
        code = np.where(b > 0, np.maximum(code, 1), code)
    values = np.where(bad[..., None], np.nan, code * scale)
    byte = np.where(bad, 255, e + 127).astype(np.uint8)
    cols = np.shape(x)[1]
    stored = (code + (0 if positive else 128)).reshape(b.shape[0], b.shape[1] * BLOCK)[:, :cols]
    return stored, byte, values.reshape(b.shape[0], b.shape[1] * BLOCK)[:, :cols]
