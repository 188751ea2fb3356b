"""4-bit microscaled floating point for the layers of an acting policy (libmarl_amd.so `marl_mx_*`).

Blocks of 32 values along a row share a power-of-two scale; a value is one of 0, .5, 1, 1.5, 2, 3, 4, 6 or their
negatives times it.  `linear` computes a layer with both operands in that form and sums in float32: the reference's
layers (model.py:13-27) at an eighth of the weight bytes, and on the matrix cores' 4-bit rate.  Inference only: nothing
here has a gradient.  (The whole numbers of the two-agent observations, -3 to 4, come through unchanged.)
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib

BLOCK = 32
_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_MXFP4 = 3


def _p(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _rows(x, name):
    """a 2-d float tensor on the GPU whose rows are contiguous (they may lie apart): (tensor, row stride)"""
    if not isinstance(x, torch.Tensor) or x.dim() != 2 or not x.is_cuda or x.dtype not in _TYPES:
        raise ValueError(f"{name} must be a float32, bfloat16 or float16 [rows, cols] tensor on the GPU")
    if x.shape[1] == 0:
        raise ValueError(f"{name} has no columns")
    if x.shape[0] > 1 and (x.stride(1) != 1 or x.stride(0) < x.shape[1]) or x.shape[0] == 1 and x.shape[1] > 1 and x.stride(1) != 1:
        x = x.contiguous()
    return x, (x.stride(0) if x.shape[0] > 1 else x.shape[1])


class MXFP4:
    """A [rows, cols] tensor in 4 bits: `codes` uint8 [rows, 16 * blocks] (two codes a byte, the lower half first) and
    `scales` uint8 [rows, blocks] (2^(byte - 127); 255: the block reads as NaN), blocks = ceil(cols / 32)."""

    def __init__(self, codes, scales, cols):
        cols = int(cols)
        blocks = -(-cols // BLOCK)
        for t, width, name in ((codes, 16 * blocks, "codes"), (scales, blocks, "scales")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() != 2 or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"{name} must be a contiguous 2-d uint8 tensor on the GPU")
            if cols <= 0 or t.shape[1] != width or t.shape[0] != codes.shape[0] or t.device != codes.device:
                raise ValueError(f"{name} of {cols} columns must be [rows, {width}], the same rows and device as the codes")
        self.codes, self.scales, self.cols = codes, scales, cols

    @property
    def shape(self):
        return torch.Size((self.codes.shape[0], self.cols))

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32):
        """the values, as a [rows, cols] tensor (rounded once more for the 16-bit types)"""
        if dtype not in _TYPES:
            raise ValueError("dtype must be torch.float32, torch.bfloat16 or torch.float16")
        out = torch.empty(tuple(self.shape), dtype=dtype, device=self.device)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().marl_mx_dequantize(_p(self.codes), _p(self.scales), self.shape[0], self.cols, _TYPES[dtype],
                                                     _p(out), _stream(self.device)), "marl_mx_dequantize")
        return out


def _empty(rows, cols, device):
    blocks = -(-cols // BLOCK)
    return MXFP4(torch.empty((rows, 16 * blocks), dtype=torch.uint8, device=device),
                 torch.empty((rows, blocks), dtype=torch.uint8, device=device), cols)


def quantize(x, out=None):
    """x: float32, bfloat16 or float16 [rows, cols] on the GPU (rows may lie apart).  `out`: an MXFP4 of the same shape
    to write into (a weight that captured launches read) instead of a new one."""
    x, stride = _rows(x.detach() if isinstance(x, torch.Tensor) else x, "x")
    if out is None:
        out = _empty(x.shape[0], x.shape[1], x.device)
    elif not isinstance(out, MXFP4) or out.shape != x.shape or out.device != x.device:
        raise ValueError(f"out must be an MXFP4 of shape {tuple(x.shape)} on the device of x")
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().marl_mx_quantize(_p(x), _TYPES[x.dtype], x.shape[0], x.shape[1], stride, _p(out.codes), _p(out.scales),
                                               _stream(x.device)), "marl_mx_quantize")
    return out


def linear(x, weight, bias=None, relu=False, out_dtype=torch.float32):
    """relu?(x W^T + bias).  `x`: [rows, cols], an MXFP4 or a float tensor that is quantised within the call; `weight`: the
    MXFP4 of the layer's [out, cols] weight; `bias`: float32 [out] or None.  Returns [rows, out] in `out_dtype`, or, with
    out_dtype="mxfp4", an MXFP4 (the next layer's x)."""
    if not isinstance(weight, MXFP4):
        raise ValueError("weight must be an MXFP4 (mxfp4.quantize)")
    quantised = isinstance(x, MXFP4)
    if not quantised:
        if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
            raise ValueError("mxfp4.linear has no gradient: call it under torch.no_grad()")
        x, stride = _rows(x, "x")
    if x.shape[1] != weight.cols or x.device != weight.device:
        raise ValueError(f"x has {x.shape[1]} columns on {x.device}, the weight {weight.cols} on {weight.device}")
    rows, n = x.shape[0], weight.shape[0]
    if n == 0:
        raise ValueError("weight has no rows")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (n,) or not bias.is_contiguous() or bias.device != x.device):
        raise ValueError(f"bias must be a contiguous float32 tensor of {n} entries on the device of x")
    device = x.device
    if out_dtype == "mxfp4":
        y = _empty(rows, n, device)
        y_data, y_scales, y_type = y.codes, y.scales, _MXFP4
    elif out_dtype in _TYPES:
        y = y_data = torch.empty((rows, n), dtype=out_dtype, device=device)
        y_scales, y_type = None, _TYPES[out_dtype]
    else:
        raise ValueError('out_dtype must be torch.float32, torch.bfloat16, torch.float16 or "mxfp4"')
    L = _lib.lib()
    x_data, x_scales, x_type, stride = (x.codes, x.scales, _MXFP4, 0) if quantised else (x, None, _TYPES[x.dtype], stride)
    need = L.marl_mx_linear_workspace_bytes(x_type, rows, weight.cols, n)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    with torch.cuda.device(device):
        _lib.check(L.marl_mx_linear(_p(x_data), _p(x_scales), x_type, rows, weight.cols, stride, _p(weight.codes), _p(weight.scales),
                                    n, _p(bias), int(bool(relu)), _p(y_data), _p(y_scales), y_type, _p(work), _stream(device)),
                   "marl_mx_linear")
    return y
