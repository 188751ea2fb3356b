"""Activations kept in 8 bits between the forward and the backward pass of an update (libmarl_amd.so `marl_act_*`).

Autograd keeps every layer's float32 input until its backward pass: at 8.4 million samples a minibatch (131,072 envs)
the trunk's inputs and outputs (202 + 512 + 256 values a sample) are 33 GB.  Here they are kept as one byte a value and
one scale byte per 32, a quarter of that, and the backward pass reads them as they are: a code times a power of two is
exactly a bfloat16, so the weight gradient takes it straight into the bf16 matrix cores while the gradient itself goes in
with all its bits.  What the ReLU of a layer let through is read off its kept output's codes, exactly.
"""
from __future__ import annotations

import torch

from . import _lib
from .mxfp4 import BLOCK, _TYPES, _p, _rows, _stream


class Act8:
    """A [rows, cols] activation in 8 bits: `codes` uint8 [rows, cols], `scales` uint8 [rows, blocks] (2^(byte - 127); 255:
    the block reads as NaN), blocks = ceil(cols / 32).  `nonnegative`: codes are 0 .. 255 and 0 only for zero; otherwise
    128 is zero."""

    def __init__(self, codes, scales, nonnegative):
        for t, name in ((codes, "codes"), (scales, "scales")):
            if not isinstance(t, torch.Tensor) or t.dtype != torch.uint8 or t.dim() != 2 or not t.is_contiguous() or not t.is_cuda:
                raise ValueError(f"{name} must be a contiguous 2-d uint8 tensor on the GPU")
        if codes.shape[1] == 0 or scales.shape != (codes.shape[0], -(-codes.shape[1] // BLOCK)) or scales.device != codes.device:
            raise ValueError("scales must be [rows, ceil(cols / 32)] beside the codes' [rows, cols], on the same device")
        self.codes, self.scales, self.nonnegative = codes, scales, bool(nonnegative)

    @property
    def shape(self):
        return self.codes.shape

    @property
    def device(self):
        return self.codes.device

    def dequantize(self, dtype=torch.float32):
        """the values, as a [rows, cols] tensor (exact also in bfloat16)"""
        if dtype not in _TYPES:
            raise ValueError("dtype must be torch.float32, torch.bfloat16 or torch.float16")
        out = torch.empty(tuple(self.shape), dtype=dtype, device=self.device)
        with torch.cuda.device(self.device):
            _lib.check(_lib.lib().marl_act_dequantize(_p(self.codes), _p(self.scales), self.shape[0], self.shape[1],
                                                      int(self.nonnegative), _TYPES[dtype], _p(out), _stream(self.device)),
                       "marl_act_dequantize")
        return out


def compress(x, nonnegative=False):
    """x: float32, bfloat16 or float16 [rows, cols] on the GPU (rows may lie apart).  `nonnegative`: x has no negative
    values (it comes from a ReLU); any there are count as 0.  One step of a block is at most 1/64 (nonnegative: 1/128) of
    its largest value, so a value is off by at most half that; a positive one that would round to 0 becomes one step."""
    x, stride = _rows(x.detach() if isinstance(x, torch.Tensor) else x, "x")
    rows, cols = x.shape
    out = Act8(torch.empty((rows, cols), dtype=torch.uint8, device=x.device),
               torch.empty((rows, -(-cols // BLOCK)), dtype=torch.uint8, device=x.device), nonnegative)
    with torch.cuda.device(x.device):
        _lib.check(_lib.lib().marl_act_compress(_p(x), _TYPES[x.dtype], rows, cols, stride, int(out.nonnegative), _p(out.codes),
                                                _p(out.scales), _stream(x.device)), "marl_act_compress")
    return out


def weight_grad(grad, act, mask=None):
    """Gradients of a linear layer y = x W^T + b, or relu of that, from the gradient of y ([rows, out], float32, bfloat16 or
    float16) and the kept x (`act`).  `mask`: y as it was kept (nonnegative) where a ReLU stood behind the layer.
    Returns (grad_weight float32 [out, cols], grad_bias float32 [out], the gradient behind the ReLU in grad's type, or None
    without a mask)."""
    grad, _ = _rows(grad.detach() if isinstance(grad, torch.Tensor) else grad, "grad")
    grad = grad.contiguous()
    if not isinstance(act, Act8) or act.shape[0] != grad.shape[0] or act.device != grad.device:
        raise ValueError("act must be an Act8 with the rows and the device of grad")
    if mask is not None and (not isinstance(mask, Act8) or not mask.nonnegative or mask.shape != grad.shape or mask.device != grad.device):
        raise ValueError("mask must be a nonnegative Act8 of grad's shape, on its device")
    rows, out = grad.shape
    cols, device = act.shape[1], grad.device
    masked = torch.empty_like(grad) if mask is not None else None
    if rows == 0:
        return torch.zeros((out, cols), device=device), torch.zeros(out, device=device), masked
    gw = torch.empty((out, cols), dtype=torch.float32, device=device)
    gb = torch.empty(out, dtype=torch.float32, device=device)
    L = _lib.lib()
    need = L.marl_act_weight_grad_workspace_bytes(rows, out, cols)
    work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    with torch.cuda.device(device):
        _lib.check(L.marl_act_weight_grad(_p(grad), _TYPES[grad.dtype], rows, out, _p(act.codes), _p(act.scales), cols,
                                          int(act.nonnegative), _p(mask.codes) if mask is not None else None, _p(masked), _p(gw),
                                          _p(gb), _p(work), _stream(device)), "marl_act_weight_grad")
    return gw, gb, masked
