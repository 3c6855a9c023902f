"""MXFP4 tensors and linears: E2M1 codes with one power-of-two scale per 32 columns.

  mx_quantize(x)        a matrix to MXFP4
  MxTensor              codes and scales; from_packed() takes a checkpoint's order
  MxLinear              y = residual + gate * act(x . W^T + bias), x quantised in the call

Beside the MLX affine `Linear`, whose weights are dequantised for bf16 products,
`MxLinear` quantises the activations too and multiplies codes on the tensor
cores' block-scaled 4-bit path.  Its `forward_fused` takes the epilogue's
arguments of `Linear.forward_fused` (gate, residual, activation, out, bias,
residual_mul), so callers that pass these run with either.  Forward only.
"""
from __future__ import annotations

import math
from typing import Optional, Union

import torch

from . import _block
from ._block import bad_argument, bad_shape
from .quant import ACTIVATIONS, OWN_BIAS
from . import _lib
from ._lib import QmmError

BLOCK = 32

_host = _block.host
_checked = _block.checked


def _sizes(rows: int, k: int):
    """Shape of the codes and bytes of the scales of [rows, k]."""
    return (rows, -(-k // BLOCK) * 16), -(-rows // 128) * -(-k // 256) * 1024


class MxTensor:
    """An MXFP4 matrix [rows, k] (qmm_mx4 of include/qmm_block.h).

    codes: uint8 [rows, 16 * ceil(k / 32)], column 2 j in the low four bits of
    byte j; scales: uint8, in the order of the tensor cores (row_scales() gives
    them as [rows, ceil(k / 32)]).  Both contiguous, of exactly these sizes,
    16-byte aligned and on one device; lead, whose product is rows, shapes
    results."""

    __slots__ = ("codes", "scales", "rows", "k", "lead")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, rows: int, k: int, lead=None):
        rows, k = int(rows), int(k)
        lead = (rows,) if lead is None else tuple(int(n) for n in lead)  # leading dimensions of the quantised tensor
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise bad_argument(f"MXFP4 codes and scales are uint8, not {codes.dtype} and {scales.dtype}")
        if rows < 0 or k <= 0 or math.prod(lead) != rows or any(n < 0 for n in lead):
            raise bad_shape(f"an MXFP4 matrix of [{rows}, {k}] with leading dimensions {lead}")
        want, tiles = _sizes(rows, k)
        if tuple(codes.shape) != want or tuple(scales.shape) != (tiles,):
            raise bad_shape(f"MXFP4 [{rows}, {k}] needs codes {want} and {tiles} bytes of scales, not {tuple(codes.shape)} and {tuple(scales.shape)}")
        if codes.device != scales.device or not codes.is_contiguous() or not scales.is_contiguous():
            raise bad_argument(f"MXFP4 codes on {codes.device} and scales on {scales.device}: both must be contiguous, on one device")
        if codes.data_ptr() % 16 or scales.data_ptr() % 16:
            raise QmmError(_lib.QMM_ERR_MISALIGNED, "MXFP4 codes and scales must be 16-byte aligned")
        self.codes, self.scales, self.rows, self.k, self.lead = codes, scales, rows, k, lead

    @classmethod
    def _made(cls, codes: torch.Tensor, scales: torch.Tensor, rows: int, k: int, lead) -> "MxTensor":
        """Buffers that this package allocated for [rows, k]: nothing to check."""
        t = cls.__new__(cls)
        t.codes, t.scales, t.rows, t.k, t.lead = codes, scales, rows, k, tuple(lead)
        return t

    @classmethod
    def empty(cls, rows: int, k: int, device, lead=None) -> "MxTensor":
        shape, tiles = _sizes(rows, k)
        return cls._made(torch.empty(shape, dtype=torch.uint8, device=device), torch.empty((tiles,), dtype=torch.uint8, device=device), rows, k,
                         (rows,) if lead is None else lead)

    @classmethod
    def from_packed(cls, codes: torch.Tensor, scales: torch.Tensor, k: Optional[int] = None) -> "MxTensor":
        """codes uint8 [rows, 16 * blocks], scales uint8 [rows, blocks] (E8M0),
        as checkpoints store them; k (default 32 * blocks) of the last block
        may be short, its codes past k must be 0."""
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise bad_argument(f"MXFP4 codes and scales are uint8, not {codes.dtype} and {scales.dtype}")
        if codes.dim() != 2 or scales.dim() != 2 or codes.shape[0] != scales.shape[0] or codes.shape[1] != 16 * scales.shape[1]:
            raise bad_shape(f"MXFP4 codes {tuple(codes.shape)} do not match scales {tuple(scales.shape)}")
        rows, blocks = scales.shape
        k = BLOCK * blocks if k is None else int(k)
        if rows == 0 or -(-k // BLOCK) != blocks:
            raise bad_shape(f"{blocks} blocks of 32 do not hold [{rows}, {k}]")
        device = _block.require_cuda(codes, "codes")
        if scales.device != device:
            raise bad_argument(f"codes are on {device}, scales on {scales.device}")
        t = cls.empty(rows, k, device)
        t.codes.copy_(codes)
        scales = scales.contiguous()
        _block.run("qmm_mx4_tile_scales", device, scales.data_ptr(), rows, k, t.scales.data_ptr())
        return t

    @property
    def shape(self):
        return (*self.lead, self.k)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    def row_scales(self) -> torch.Tensor:
        """The E8M0 scales as uint8 [rows, ceil(k / 32)]."""
        out = torch.empty((self.rows, -(-self.k // BLOCK)), dtype=torch.uint8, device=self.device)
        if self.rows:
            _block.run("qmm_mx4_row_scales", self.device, self.scales.data_ptr(), self.rows, self.k, out.data_ptr())
        return out

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The values, [..., k]; exact in bf16 and f32 (below 2^128)."""
        if dtype is torch.bfloat16 and len(self.lead) == 1:
            out = _host().mx_dequantize(self.codes, self.scales, self.rows, self.k)
            if out is not None:
                return _checked(out)
        e = _block.ELEMS.get(dtype)
        if e is None:
            raise bad_argument(f"dequantize does not support {dtype}")
        out = torch.empty((*self.lead, self.k), dtype=dtype, device=self.codes.device)
        if self.rows:
            _block.run("qmm_mx4_dequantize", self.codes.device,
                       _block.MX4.pack(self.codes.data_ptr(), self.scales.data_ptr(), self.rows, self.k), out.data_ptr(), e)
        return out


def mx_quantize(x: torch.Tensor) -> MxTensor:
    """x [..., k] (bf16, f16 or f32) to MXFP4, blocks of 32 along the last dimension.

    Each block's scale is the power of two that brings its largest magnitude
    to [4, 8); values round to the nearest code, ties to the even one, and
    saturate at 6 scales.  A block with an infinity or NaN becomes NaN."""
    made = _host().mx_quantize(x)
    if made is not None:
        codes, scales = _checked(made)
        lead = x.shape[:-1]
        return MxTensor._made(codes, scales, codes.shape[0], x.shape[-1], lead)
    device = _block.require_cuda(x, "input")
    e = _block.elem_of(x, "input")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise bad_shape(f"a tensor of shape {tuple(x.shape)} has no blocks")
    lead, k = x.shape[:-1], x.shape[-1]
    x2 = _block.rows_of(x, k)
    rows = x2.shape[0]
    t = MxTensor.empty(rows, k, device, lead)
    if rows:
        _block.run("qmm_mx4_quantize", device, x2.data_ptr(), e, rows, k, x2.stride(0), t.codes.data_ptr(), t.scales.data_ptr())
    return t


class MxLinear:
    """A linear with MXFP4 weights [output, input] and an optional bias."""

    def __init__(self, weight: MxTensor, bias: Optional[torch.Tensor] = None):
        if bias is not None:
            if bias.numel() != weight.rows:
                raise bad_shape(f"bias {tuple(bias.shape)} does not match {weight.rows} outputs")
            bias = bias.reshape(weight.rows).to(device=weight.device, dtype=torch.bfloat16).contiguous()
        self.weight, self.bias = weight, bias
        self.input, self.output = weight.k, weight.rows

    @classmethod
    def from_dense(cls, weight: torch.Tensor, bias: Optional[torch.Tensor] = None) -> "MxLinear":
        """Quantises a dense weight [output, input]."""
        if weight.dim() != 2:
            raise bad_shape(f"weight {tuple(weight.shape)} is not a matrix")
        return cls(mx_quantize(weight), bias)

    @property
    def device(self) -> torch.device:
        return self.weight.device

    def forward(self, x: Union[torch.Tensor, MxTensor]) -> torch.Tensor:
        return self.forward_fused(x)

    __call__ = forward

    def forward_fused(self, x: Union[torch.Tensor, MxTensor], *, gate: Optional[torch.Tensor] = None,
                      residual: Optional[torch.Tensor] = None, activation: Optional[str] = None,
                      out: Optional[torch.Tensor] = None, bias=OWN_BIAS, residual_mul: bool = False) -> torch.Tensor:
        """bf16 [..., output] = residual + gate * act(x . W^T + bias).

        x: bf16, f16 or f32 [..., input], quantised to MXFP4 by the rule of
        mx_quantize, or an MxTensor.  gate [output]; residual as the output
        (out may be the residual); bias replaces the layer's own (None: none);
        residual_mul: residual * (gate * act(...)).  One rounding, to bf16."""
        act = ACTIVATIONS.get(activation)
        if act is None:
            raise bad_argument(f"unknown activation {activation!r}")
        if residual_mul:
            act |= _lib.QMM_EPILOGUE_RESIDUAL_MUL
        w = self.weight
        if out is None:
            b = self.bias if bias is OWN_BIAS else bias
            if x.__class__ is not MxTensor:
                y = _host().mx_linear(x, None, w.codes, w.scales, self.output, self.input, b, gate, residual, act)
            elif x.k == self.input and len(x.lead) == 1:
                y = _host().mx_linear(x.codes, x.scales, w.codes, w.scales, self.output, self.input, b, gate, residual, act)
            else:
                y = None
            if y is not None:
                return _checked(y)
        device, n, k = w.codes.device, self.output, self.input
        x_ptr = stride = x_codes = x_scales = elem = 0
        if isinstance(x, MxTensor):
            lead, m = x.lead, x.rows
            if x.k != k:
                raise bad_shape(f"MXFP4 linear expects {k} inputs, got {x.k}")
            if x.codes.device != device:
                raise bad_argument(f"the input is on {x.codes.device}, the weight on {device}")
            x_codes, x_scales = x.codes.data_ptr(), x.scales.data_ptr()
        else:
            elem = _block.elem_of(x, "input")
            if x.dim() == 0 or x.shape[-1] != k:
                raise bad_shape(f"MXFP4 linear expects {k} inputs, got {tuple(x.shape)}")
            if x.device != device:
                _block.require_cuda(x, "input")
                raise bad_argument(f"the input is on {x.device}, the weight on {device}")
            lead = x.shape[:-1]
            x = _block.rows_of(x, k)
            m, stride, x_ptr = x.shape[0], x.stride(0), x.data_ptr()
        if out is None:
            y = torch.empty((*lead, n), dtype=torch.bfloat16, device=device)
        else:
            y = out
            if y.dtype != torch.bfloat16 or y.device != device or y.numel() != m * n or y.shape[-1] != n or not y.is_contiguous():
                raise bad_argument(f"out must be contiguous bfloat16 {(*lead, n)} on {device}")
        if m == 0:
            return y
        bias = self.bias if bias is OWN_BIAS else self._vector(bias, "bias")
        gate = self._vector(gate, "gate")
        if residual is not None:
            if residual.numel() != m * n or residual.shape[-1] != n or residual.device != device:
                raise bad_shape(f"residual {tuple(residual.shape)} on {residual.device} does not match {(*lead, n)} on {device}")
            residual = residual.to(torch.bfloat16).contiguous()
            if residual.data_ptr() % 16:
                residual = residual.clone()
        result = y
        if y.data_ptr() % 16:  # an odd slice as `out`: through an aligned buffer
            y = torch.empty((m, n), dtype=torch.bfloat16, device=device)
        work, nbytes = None, 0
        if x_ptr:
            nbytes = _block.load().qmm_mx4_linear_workspace_bytes(m, n, k)
            if nbytes:
                work = torch.empty((nbytes,), dtype=torch.uint8, device=device)
        _block.run("qmm_mx4_linear", device, _block.LINEAR.pack(
            w.codes.data_ptr(), w.scales.data_ptr(), n, k, m, x_ptr, stride, x_codes, x_scales,
            0 if bias is None else bias.data_ptr(), 0 if gate is None else gate.data_ptr(),
            0 if residual is None else residual.data_ptr(), y.data_ptr(), 0 if work is None else work.data_ptr(), nbytes, elem, act))
        if result is not y:
            result.view(m, n).copy_(y)
        return result

    def _vector(self, v: Optional[torch.Tensor], what: str) -> Optional[torch.Tensor]:
        if v is None:
            return None
        if v.numel() != self.output or v.device != self.weight.device:
            raise bad_shape(f"{what} {tuple(v.shape)} on {v.device} does not match {self.output} outputs on {self.weight.device}")
        return v.reshape(self.output).to(torch.bfloat16).contiguous()
