"""The norms before and after a sublayer with its gate and residual, in one pass.

Generalises the block's LayerNorm + modulation (qmm_layernorm_modulate) and gated
residual (src/dit.rs:50, 88-93) to blocks that also norm the branch before its
gate: other norms, element types and widths, a scaled residual, modulation per
sequence, and an MXFP4 result for the linear that follows.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch

from . import _block
from ._block import bad_argument, bad_shape
from .mxfp4 import MxTensor


def gated_residual_norm(x: torch.Tensor, branch: Optional[torch.Tensor] = None, *, post: Optional[str] = None,
                        post_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None,
                        residual_scale: float = 1.0, pre: Optional[str] = "layer",
                        pre_weight: Optional[torch.Tensor] = None, scale: Optional[torch.Tensor] = None,
                        shift: Optional[torch.Tensor] = None, eps: float = 1e-6, x_out: Optional[torch.Tensor] = None,
                        n_out: Optional[torch.Tensor] = None, quantize: bool = False
                        ) -> Tuple[torch.Tensor, Union[torch.Tensor, MxTensor]]:
    """(x', n) with h = norm_post(branch) * post_weight, x' = residual_scale * x
    + gate * h and n = norm_pre(x') * pre_weight * (1 + scale) + shift.

    x, branch [..., hidden] in bf16, f16 or f32 (each its own); x' and n have
    x's type.  post, pre: None or "none", "rms", "layer".  post_weight and
    pre_weight [hidden]; gate, scale, shift [hidden], or [groups, hidden] (or
    [groups, 1, hidden]) for rows in `groups` equal runs, e.g. the sequences of
    a batch.  f32 inside, one rounding per output, n from the unrounded x'.
    x_out may be x or branch, n_out may be either too; quantize=True gives n as
    an MxTensor.  Without a branch and with residual_scale 1, x' is x itself
    (nothing is written) unless x_out is given."""
    same = branch is None and residual_scale == 1.0 and x_out is None  # x' would be a copy of x
    if x_out is None and n_out is None:
        made = _block.host().gated_norm(x, branch, _block.NORMS.get(post, -1), post_weight, gate, residual_scale,
                                        _block.NORMS.get(pre, -1), pre_weight, scale, shift, eps, quantize, same)
        if made is not None:
            made = _block.checked(made)
            if not quantize:
                return made
            return made[0], MxTensor._made(made[1], made[2], made[1].shape[0], x.shape[-1], x.shape[:-1])
    device = _block.require_cuda(x, "x")
    x_elem = _block.elem_of(x, "x")
    post_kind, pre_kind = _block.NORMS.get(post), _block.NORMS.get(pre)
    if post_kind is None or pre_kind is None:
        raise bad_argument(f"norms are 'rms', 'layer' or None, not {post!r} and {pre!r}")
    if x.dim() == 0 or x.shape[-1] == 0:
        raise bad_shape(f"x {tuple(x.shape)} has no columns")
    shape, hidden = x.shape, x.shape[-1]
    x2 = _block.rows_of(x, hidden)
    rows = x2.shape[0]
    b_ptr = b_stride = b_elem = 0
    if branch is not None:
        if branch.shape != shape or branch.device != device:
            raise bad_shape(f"branch {tuple(branch.shape)} on {branch.device} does not match x {tuple(shape)} on {device}")
        b_elem = _block.elem_of(branch, "branch")
        b2 = _block.rows_of(branch, hidden)
        b_ptr, b_stride = b2.data_ptr(), b2.stride(0)
    if quantize and n_out is not None:
        raise bad_argument("n_out holds n in x's type; quantize=True returns it as an MxTensor")
    x_new, xo = (x, None) if same else _output(x_out, x, shape, hidden, "x_out")
    n_ptr = n_stride = c_ptr = s_ptr = 0
    if quantize:
        n_new = MxTensor.empty(rows, hidden, device, shape[:-1])
        c_ptr, s_ptr = n_new.codes.data_ptr(), n_new.scales.data_ptr()
    else:
        n_new, no = _output(n_out, x, shape, hidden, "n_out")
        n_ptr, n_stride = no.data_ptr(), no.stride(0)
    if rows == 0:
        return x_new, n_new
    vectors = (post_weight, pre_weight, gate, scale, shift)
    dtype = None
    for v in vectors:
        if v is not None:
            if v.device != device:
                raise bad_argument(f"x is on {device}, a weight or modulation on {v.device}")
            dtype = v.dtype if dtype is None or dtype == v.dtype else torch.float32
    dtype = torch.bfloat16 if dtype is None else dtype
    if dtype not in _block.ELEMS:
        raise bad_argument(f"weights and modulation are {dtype}; bfloat16, float16 or float32 is needed")
    groups = 1
    for v in (gate, scale, shift):
        if v is not None:
            if v.shape[-1] != hidden or v.numel() % hidden:
                raise bad_shape(f"modulation {tuple(v.shape)} does not match {hidden} columns")
            groups = max(groups, v.numel() // hidden)
    if rows % groups:
        raise bad_shape(f"{rows} rows are not {groups} equal groups")
    (pw, _), (qw, _) = (_vector(v, dtype, hidden, 1, "weight") for v in (post_weight, pre_weight))
    (g, gs), (sc, ss), (sh, hs) = (_vector(v, dtype, hidden, groups, "modulation") for v in (gate, scale, shift))
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    _block.run("qmm_gated_residual_norm", device, _block.NORM.pack(
        x2.data_ptr(), b_ptr, ptr(xo), n_ptr, c_ptr, s_ptr, ptr(pw), ptr(qw), ptr(g), ptr(sh), ptr(sc), rows, hidden,
        x2.stride(0), b_stride, 0 if xo is None else xo.stride(0), n_stride, gs, hs, ss, groups, x_elem, b_elem, _block.ELEMS[dtype], post_kind,
        pre_kind, residual_scale, eps))
    return x_new, n_new


def _output(out: Optional[torch.Tensor], x: torch.Tensor, shape, hidden: int, what: str):
    """(the tensor to return, the same as rows)"""
    if out is None:
        out = torch.empty(shape, dtype=x.dtype, device=x.device)
        return out, (out if out.dim() == 2 else out.view(-1, hidden))
    if out.shape != shape or out.dtype != x.dtype or out.device != x.device:
        raise bad_shape(f"{what} {tuple(out.shape)} {out.dtype} does not match x {tuple(shape)} {x.dtype}")
    try:
        rows = out.view(-1, hidden)
    except RuntimeError:
        raise bad_shape(f"{what}'s rows are not evenly spaced") from None
    if hidden > 1 and rows.stride(1) != 1:
        raise bad_shape(f"{what}'s columns are not consecutive")
    return out, rows


def _vector(v: Optional[torch.Tensor], dtype: torch.dtype, hidden: int, groups: int, what: str):
    """v as [groups, hidden] rows in `dtype` and their stride (0: one row for every group)."""
    if v is None:
        return None, 0
    if v.shape[-1] != hidden or v.numel() not in (hidden, groups * hidden):
        raise bad_shape(f"{what} {tuple(v.shape)} is not [{hidden}] or [{groups}, {hidden}]")
    v = v.reshape(-1, hidden)
    if v.dtype != dtype:
        v = v.to(dtype)
    if hidden > 1 and v.stride(1) != 1:
        v = v.contiguous()
    return v, (v.stride(0) if v.shape[0] > 1 else 0)
