"""Rotary positions with several axes (time, height, width), with the RMSNorm of
q and k per head that precedes them in the block (the reference rotates normed
heads, src/dit.rs:51-62 with src/ops.rs:12-58).
"""
from __future__ import annotations

import math
from typing import Optional, Sequence, Tuple, Union

import torch

from . import _block
from ._block import bad_argument, bad_shape

_POSITIONS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}


class RotaryAxes:
    """Which axis and frequency turns each pair of a head's columns.

    dims: pairs of each axis, in the order of the positions' last dimension;
    2 * sum(dims) columns of a head are rotated, the rest pass through.
    pairs: "adjacent" turns columns (2 p, 2 p + 1), "halves" (p, P + p).
    ladder: "own" gives every axis its own frequencies theta^(-i / n),
    "shared" lays one ladder theta^(-i / P) over all pairs.  theta: one base,
    or one for each axis ("own")."""

    def __init__(self, dims: Sequence[int], theta: Union[float, Sequence[float]] = 10000.0, pairs: str = "adjacent",
                 ladder: str = "own", device="cuda"):
        dims = [int(n) for n in dims]
        if not dims or min(dims) < 0:
            raise bad_shape(f"axes of {dims} pairs")
        if ladder not in ("own", "shared"):
            raise bad_argument(f"ladder must be own or shared, not {ladder!r}")
        several = isinstance(theta, (list, tuple))
        if several and (ladder == "shared" or len(theta) != len(dims)):
            raise bad_argument("several bases need one for each axis and ladder 'own'")
        bases = [float(t) for t in theta] if several else [float(theta)] * len(dims)
        total = sum(dims)
        if ladder == "own":
            freq = [bases[a] ** (-i / n) for a, n in enumerate(dims) for i in range(n)]
        else:
            freq = [bases[0] ** (-i / total) for i in range(total)]
        self._init([a for a, n in enumerate(dims) for _ in range(n)], freq, len(dims), pairs, device)

    @classmethod
    def from_pairs(cls, axis: Sequence[int], freq: Sequence[float], axes: int, pairs: str = "adjacent", device="cuda") -> "RotaryAxes":
        """Any assignment: pair p turns by positions[axis[p]] * freq[p] radians."""
        self = cls.__new__(cls)
        self._init([int(a) for a in axis], [float(f) for f in freq], int(axes), pairs, device)
        return self

    def _init(self, axis, freq, axes, pairs, device):
        if pairs not in ("adjacent", "halves"):
            raise bad_argument(f"pairs must be adjacent or halves, not {pairs!r}")
        if len(axis) != len(freq) or not 1 <= axes <= 256 or any(not 0 <= a < axes for a in axis):
            raise bad_shape(f"{len(axis)} pairs, {len(freq)} frequencies over {axes} axes")
        if any(not math.isfinite(f) for f in freq):
            raise bad_argument("a frequency is not finite")
        self.pairs, self.count, self.axes = pairs, len(axis), axes
        self._adjacent = int(pairs == "adjacent")
        turns = torch.tensor(freq, dtype=torch.float64) / (2.0 * math.pi)
        lead = turns.float()
        self._turns = torch.stack([lead, (turns - lead.double()).float()], -1).contiguous().to(device)
        self._axis = torch.tensor(axis, dtype=torch.uint8).to(device)
        self.device = self._turns.device


def qk_norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, axes: RotaryAxes, *,
                   q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None, eps: float = 1e-6,
                   q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None
                   ) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """q and k after RMSNorm per head (with a weight) and rotation.

    q [tokens, heads, dim] or [batch, tokens, heads, dim], any strides with
    consecutive columns (slices of a fused projection); k likewise, its heads
    may differ, or None.  positions [tokens, axes], or [batch, tokens, axes]:
    int32, int64 or f32; whole turns drop out exactly, so far positions keep
    their accuracy (include/qmm_block.h).
    Outputs are new contiguous tensors, or q_out / k_out, which may be q / k."""
    if q_out is None and k_out is None:
        made = _block.host().qk_norm_rotary(q, k, positions, axes._turns, axes._axis, axes.axes, axes._adjacent, q_weight, k_weight, eps)
        if made is not None:
            made = _block.checked(made)
            return made if k is not None else (made, None)
    device = _block.require_cuda(q, "q")
    elem = _block.elem_of(q, "q")
    batched = q.dim() == 4
    if q.dim() not in (3, 4):
        raise bad_shape(f"q {tuple(q.shape)} is not [tokens, heads, dim] or [batch, tokens, heads, dim]")
    batch, (tokens, q_heads, dim) = (q.shape[0] if batched else 1), q.shape[-3:]
    k_heads = 0
    if k is not None:
        if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != dim or k.dtype != q.dtype or k.device != device:
            raise bad_shape(f"k {tuple(k.shape)} {k.dtype} on {k.device} does not match q {tuple(q.shape)} {q.dtype} on {device}")
        k_heads = k.shape[-2]
    if 2 * axes.count > dim:
        raise bad_shape(f"{axes.count} pairs do not fit heads of {dim} columns")
    kind = _POSITIONS.get(positions.dtype)
    if kind is None:
        raise bad_argument(f"positions are {positions.dtype}; int32, int64 or float32 is needed")
    pshape = positions.shape
    if positions.device != device or axes._turns.device != device:
        raise bad_argument(f"q is on {device}, positions on {positions.device}, the axes on {axes.device}")
    if not ((len(pshape) == 2 or (len(pshape) == 3 and batched and pshape[0] in (1, batch)))
            and pshape[-2] == tokens and pshape[-1] == axes.axes):
        raise bad_shape(f"positions {tuple(pshape)} are not [tokens, axes] = [{tokens}, {axes.axes}] (of each batch)")
    if not positions.is_contiguous():
        positions = positions.contiguous()
    pos_stride = tokens * axes.axes if len(pshape) == 3 and pshape[0] > 1 else 0
    q, q_out, qs, qo = _operand(q, q_out, "q_out")
    ks = ko = (0, 0, 0)
    if k is not None:
        k, k_out, ks, ko = _operand(k, k_out, "k_out")
    q_weight, k_weight = _weight(q_weight, q, dim, "q_weight"), _weight(k_weight, q, dim, "k_weight")
    _block.run("qmm_qk_norm_rotary", device, _block.ROTARY.pack(
        q.data_ptr(), 0 if k is None else k.data_ptr(), q_out.data_ptr(), 0 if k is None else k_out.data_ptr(),
        0 if q_weight is None else q_weight.data_ptr(), 0 if k_weight is None else k_weight.data_ptr(), positions.data_ptr(),
        axes._turns.data_ptr(), axes._axis.data_ptr(), batch, tokens, *qs, *ks, *qo, *ko, pos_stride, q_heads, k_heads, dim,
        axes.count, axes.axes, axes._adjacent, kind, elem, eps))
    return q_out, (k_out if k is not None else None)


def _strides(t: torch.Tensor):
    s = t.stride()
    return s[:3] if len(s) == 4 else (0, s[0], s[1])


def _operand(t: torch.Tensor, out: Optional[torch.Tensor], what: str):
    if out is None:
        if t.stride(-1) != 1 and t.shape[-1] != 1:
            t = t.contiguous()
        out = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    else:
        if out.shape != t.shape or out.dtype != t.dtype or out.device != t.device or (out.stride(-1) != 1 and out.shape[-1] != 1):
            raise bad_shape(f"{what} {tuple(out.shape)} {out.dtype} does not match {tuple(t.shape)} {t.dtype} with consecutive columns")
        if t.stride(-1) != 1 and t.shape[-1] != 1:
            t = t.contiguous()
    return t, out, _strides(t), _strides(out)


def _weight(w: Optional[torch.Tensor], q: torch.Tensor, dim: int, what: str) -> Optional[torch.Tensor]:
    if w is None:
        return None
    if w.numel() != dim or w.device != q.device:
        raise bad_shape(f"{what} {tuple(w.shape)} on {w.device} does not match heads of {dim} columns on {q.device}")
    return w.reshape(dim).to(q.dtype).contiguous()
