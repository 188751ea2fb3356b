"""4-bit microscaled floating point for the layers of the policy (libmarl_amd.so `marl_mx_*`).

Blocks of 32 values along a row share a power-of-two scale; a value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 or their
negatives times it.  `linear` computes a layer with both operands in that form and sums in float32: the reference's
layers (model.py:13-27) at an eighth of the weight bytes, and on the matrix cores' 4-bit rate.  Nothing here has a
gradient of its own: `linear` refuses tensors that want one, all calls refuse forward-mode derivatives, and what trains
through them brings its own backward pass (policy.py).

A value is off by at most a quarter of the largest in its block of 32.  Whole numbers come through unchanged in a block
whose largest is at most 4; beside larger ones small ones are coarser, and beside the timer of a cooking pot in an
observation (up to 30) they can vanish: 30 reads as 24, 3 as 4 and 1 as 0.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from . import _lib

BLOCK = 32
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MXFP4 = 3


def _p(t):
    return None if t is None else t.data_ptr()


def _no_tangent(t, name):
    """a forward-mode derivative would be lost without a word"""
    if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
        raise ValueError(f"{name} has a forward-mode derivative, and this call has none to give")


def _rows(x, name):
    """a 2-d float tensor on the GPU whose rows are contiguous (they may lie apart): (tensor, rows, cols, row stride)"""
    if not isinstance(x, torch.Tensor) or x.dtype not in _TYPES or x.dim() != 2 or not x.is_cuda:
        raise ValueError(f"{name} must be a float32, bfloat16 or float16 [rows, cols] tensor on the GPU")
    _no_tangent(x, name)
    rows, cols = x.shape
    if cols >= 1 << 31:  # a C int
        raise ValueError(f"{name} has 2^31 or more columns")
    if x.is_contiguous():
        if cols == 0:
            raise ValueError(f"{name} has no columns")
        return x, rows, cols, cols
    if x.stride(1) != 1 or x.stride(0) < cols:
        return x.contiguous(), rows, cols, cols
    return x, rows, cols, x.stride(0)


def _bytes_on_gpu(t, name):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() != 2 or not t.is_cuda or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous 2-d uint8 tensor on the GPU")
    return t.shape


class MXFP4:
    """A [rows, cols] tensor in 4 bits: `codes` uint8 [rows, 16 * blocks] (two codes a byte, the lower half first) and
    `scales` uint8 [rows, blocks] (2^(byte - 127); 255: the block reads as NaN), blocks = ceil(cols / 32).  Codes behind the
    last column are 0, or 8 (minus 0): a product counts them."""

    __slots__ = ("codes", "scales", "shape", "device")

    def __init__(self, codes, scales, cols):
        rows, width = _bytes_on_gpu(codes, "codes")
        blocks = -(-cols // BLOCK)
        if not 0 < cols < 1 << 31 or width != 16 * blocks or _bytes_on_gpu(scales, "scales") != (rows, blocks) or scales.device != codes.device:
            raise ValueError(f"codes and scales of {cols} columns must be [rows, {16 * blocks}] and [rows, {blocks}] on one device")
        self.codes, self.scales, self.shape, self.device = codes, scales, torch.Size((rows, cols)), codes.device

    @property
    def cols(self):
        return self.shape[1]

    def dequantize(self, dtype=torch.float32):
        """the values, as a [rows, cols] tensor (rounded once more for the 16-bit types)"""
        if dtype not in _TYPES:
            raise ValueError("dtype must be torch.float32, torch.bfloat16 or torch.float16")
        rows, cols = self.shape
        out = torch.empty(rows, cols, dtype=dtype, device=self.device)
        _lib.call(_lib.lib().marl_mx_dequantize, "marl_mx_dequantize", self.device, self.codes.data_ptr(), self.scales.data_ptr(),
                  rows, cols, _TYPES[dtype], out.data_ptr())
        return out


def _empty(shape, device):
    rows, cols = shape
    blocks = -(-cols // BLOCK)
    new = MXFP4.__new__(MXFP4)
    new.codes = torch.empty(rows, 16 * blocks, dtype=torch.uint8, device=device)
    new.scales = torch.empty(rows, blocks, dtype=torch.uint8, device=device)
    new.shape, new.device = shape, device
    return new


def quantize(x, out=None):
    """x: float32, bfloat16 or float16 [rows, cols] on the GPU (rows may lie apart).  `out`: an MXFP4 of the same shape
    to write into (a weight that captured launches read) instead of a new one."""
    x, rows, cols, stride = _rows(x, "x")
    if out is None:
        out = _empty(x.shape, x.device)
    elif not isinstance(out, MXFP4) or out.shape != x.shape or out.device != x.device:
        raise ValueError(f"out must be an MXFP4 of shape {tuple(x.shape)} on the device of x")
    _lib.call(_lib.lib().marl_mx_quantize, "marl_mx_quantize", x.device, x.data_ptr(), _TYPES[x.dtype], rows, cols, stride,
              out.codes.data_ptr(), out.scales.data_ptr())
    return out


def linear(x, weight, bias=None, relu=False, out_dtype=torch.float32):
    """relu?(x W^T + bias).  `x`: [rows, cols], an MXFP4 or a float tensor that is quantised within the call; `weight`: the
    MXFP4 of the layer's [out, cols] weight; `bias`: float32 [out] or None.  Returns [rows, out] in `out_dtype`, or, with
    out_dtype="mxfp4", an MXFP4 (the next layer's x)."""
    if not isinstance(weight, MXFP4):
        raise ValueError("weight must be an MXFP4 (mxfp4.quantize)")
    n, cols = weight.shape
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in (x, bias)):
        raise ValueError("mxfp4.linear has no gradient: call it under torch.no_grad()")
    if isinstance(x, MXFP4):
        rows, xcols = x.shape
        x_data, x_scales, x_type, stride = x.codes, x.scales, _MXFP4, 0
    else:
        x, rows, xcols, stride = _rows(x, "x")
        x_data, x_scales, x_type = x, None, _TYPES[x.dtype]
    device = x.device
    if xcols != cols or device != weight.device:
        raise ValueError(f"x has {xcols} columns on {device}, the weight {cols} on {weight.device}")
    if n == 0 or n > 1 << 22:
        raise ValueError("weight has no rows, or more than 2^22")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous() or bias.device != device):
        raise ValueError(f"bias must be a contiguous float32 tensor of {n} entries on the device of x")
    if bias is not None:
        _no_tangent(bias, "bias")
    if out_dtype == "mxfp4":
        y = _empty(torch.Size((rows, n)), device)
        y_data, y_scales, y_type = y.codes, y.scales, _MXFP4
    elif out_dtype in _TYPES:
        y = y_data = torch.empty(rows, n, dtype=out_dtype, device=device)
        y_scales, y_type = None, _TYPES[out_dtype]
    else:
        raise ValueError('out_dtype must be torch.float32, torch.bfloat16, torch.float16 or "mxfp4"')
    L = _lib.lib()
    need = L.marl_mx_linear_workspace_bytes(x_type, rows, cols, n)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _lib.call(L.marl_mx_linear, "marl_mx_linear", device, x_data.data_ptr(), _p(x_scales), x_type, rows, cols, stride,
              weight.codes.data_ptr(), weight.scales.data_ptr(), n, _p(bias), 1 if relu else 0, y_data.data_ptr(), _p(y_scales), y_type,
              _p(work))
    return y
