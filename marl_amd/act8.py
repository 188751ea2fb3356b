"""Activations kept in 8 bits between the forward and the backward pass of an update (libmarl_amd.so `marl_act_*`).

Autograd keeps every layer's float32 input until its backward pass: at 8.4 million samples a minibatch (131,072 envs)
the trunk's inputs and outputs (202 + 512 + 256 values a sample) are 33 GB.  Here they are kept as one byte a value and
one scale byte per 32, a quarter of that (an update's peak, with its gradients in flight, falls by three tenths), and the
backward pass reads them as they are: a code times a power of two is exactly a bfloat16, so the weight gradient takes it
straight into the bf16 matrix cores while the gradient itself goes in with all its bits.  What the ReLU of a layer let through is read off its kept output's codes, exactly.
"""
from __future__ import annotations

import torch

from . import _lib
from .mxfp4 import BLOCK, _TYPES, _bytes_on_gpu, _p, _rows


class Act8:
    """A [rows, cols] activation in 8 bits: `codes` uint8 [rows, cols], `scales` uint8 [rows, blocks] (2^(byte - 127); 255:
    the block reads as NaN), blocks = ceil(cols / 32).  `nonnegative`: codes are 0 .. 255 and 0 only for zero; otherwise
    128 is zero."""

    __slots__ = ("codes", "scales", "nonnegative", "shape", "device")

    def __init__(self, codes, scales, nonnegative):
        rows, cols = _bytes_on_gpu(codes, "codes")
        if not 0 < cols < 1 << 31 or _bytes_on_gpu(scales, "scales") != (rows, -(-cols // BLOCK)) or scales.device != codes.device:
            raise ValueError("scales must be [rows, ceil(cols / 32)] beside the codes' [rows, cols], on the same device")
        self.codes, self.scales, self.nonnegative = codes, scales, bool(nonnegative)
        self.shape, self.device = codes.shape, codes.device

    def dequantize(self, dtype=torch.float32):
        """the values, as a [rows, cols] tensor (exact also in bfloat16)"""
        if dtype not in _TYPES:
            raise ValueError("dtype must be torch.float32, torch.bfloat16 or torch.float16")
        rows, cols = self.shape
        out = torch.empty(rows, cols, dtype=dtype, device=self.device)
        _lib.call(_lib.lib().marl_act_dequantize, "marl_act_dequantize", self.device, self.codes.data_ptr(), self.scales.data_ptr(),
                  rows, cols, 1 if self.nonnegative else 0, _TYPES[dtype], out.data_ptr())
        return out


def compress(x, nonnegative=False):
    """x: float32, bfloat16 or float16 [rows, cols] on the GPU (rows may lie apart).  `nonnegative`: x has no negative
    values (it comes from a ReLU); any there are count as 0.  A block's largest value is at least 63.75 of its steps
    (nonnegative: 127.75), unless it lies below 2^-120 (2^-119), where a step is 2^-126, and a value is off by at most half a step.  Two are off by up to a
    step: a positive value that would round to 0 becomes one step (nonnegative), and what lies above 127 (255) steps of the
    largest scale is cut to them."""
    x, rows, cols, stride = _rows(x, "x")
    out = Act8.__new__(Act8)
    out.codes = torch.empty(rows, cols, dtype=torch.uint8, device=x.device)
    out.scales = torch.empty(rows, -(-cols // BLOCK), dtype=torch.uint8, device=x.device)
    out.nonnegative, out.shape, out.device = bool(nonnegative), x.shape, x.device
    _lib.call(_lib.lib().marl_act_compress, "marl_act_compress", x.device, x.data_ptr(), _TYPES[x.dtype], rows, cols, stride,
              1 if nonnegative else 0, out.codes.data_ptr(), out.scales.data_ptr())
    return out


def weight_grad(grad, act, mask=None, want_masked=True):
    """Gradients of a linear layer y = x W^T + b, or relu of that, from the gradient of y ([rows, out], float32, bfloat16 or
    float16) and the kept x (`act`).  `mask`: y as it was kept (nonnegative) where a ReLU stood behind the layer.
    Returns (grad_weight float32 [out, cols], grad_bias float32 [out], the gradient behind the ReLU in grad's type, or None
    without a mask or with `want_masked` False: a layer whose input needs no gradient has no use for it)."""
    grad, rows, out, stride = _rows(grad, "grad")
    if stride != out:
        grad = grad.contiguous()
    device = grad.device
    if not isinstance(act, Act8) or act.shape[0] != rows or act.device != device:
        raise ValueError("act must be an Act8 with the rows and the device of grad")
    if mask is not None and (not isinstance(mask, Act8) or not mask.nonnegative or mask.shape != grad.shape or mask.device != device):
        raise ValueError("mask must be a nonnegative Act8 of grad's shape, on its device")
    cols = act.shape[1]
    masked = torch.empty_like(grad) if mask is not None and want_masked else None
    if rows == 0:
        return torch.zeros((out, cols), device=device), torch.zeros(out, device=device), masked
    gw = torch.empty(out, cols, dtype=torch.float32, device=device)
    gb = torch.empty(out, dtype=torch.float32, device=device)
    L = _lib.lib()
    need = L.marl_act_weight_grad_workspace_bytes(rows, out, cols)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    mask_codes = None if mask is None else mask.codes.data_ptr()
    if mask is not None and not want_masked:
        _lib.call(L.marl_act_param_grad, "marl_act_param_grad", device, grad.data_ptr(), _TYPES[grad.dtype], rows, out,
                  act.codes.data_ptr(), act.scales.data_ptr(), cols, 1 if act.nonnegative else 0, mask_codes, gw.data_ptr(), gb.data_ptr(), _p(work))
        return gw, gb, None
    _lib.call(L.marl_act_weight_grad, "marl_act_weight_grad", device, grad.data_ptr(), _TYPES[grad.dtype], rows, out,
              act.codes.data_ptr(), act.scales.data_ptr(), cols, 1 if act.nonnegative else 0,
              mask_codes, _p(masked), gw.data_ptr(), gb.data_ptr(), _p(work))
    return gw, gb, masked


def column_sums(x):
    """x.sum(0) of a float32, bfloat16 or float16 [rows, cols] tensor on the GPU, in float32.  It clears no memory, so a captured
    graph of it is right in every replay (torch's sum over many rows records a memory-set node, which is not)."""
    x, rows, cols, stride = _rows(x, "x")
    if stride != cols:
        x = x.contiguous()
    if rows == 0:
        return torch.zeros(cols, device=x.device)
    out = torch.empty(cols, dtype=torch.float32, device=x.device)
    L = _lib.lib()
    need = L.marl_column_sums_workspace_bytes(rows, cols)
    work = torch.empty(need, dtype=torch.uint8, device=x.device) if need else None
    _lib.call(L.marl_column_sums, "marl_column_sums", x.device, x.data_ptr(), _TYPES[x.dtype], rows, cols, out.data_ptr(), _p(work))
    return out
