"""Rotary embedding from positions on several axes (time, height, width), on MI355X (``pasa_rope_axes``).

The prologue's rotary forms (``pasa_amd.prologue``) read a table of coefficients, a row for every token.  This one
takes the tokens' positions: a frame may begin at any time, text and video may be mixed, requests of any length
lie behind each other, and nothing is laid out beforehand.

    axes = RotaryAxes.video(128, device=q.device)
    q, k = rope_axes(q, k, positions, axes)        # positions [3, S]: time, height, width

Gradients of q and k go through the inverse rotation.  There is no CPU path.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import Optional, Sequence, Tuple

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16, torch.float32: _lib.DTYPE_F32}
_POS = {torch.int32: 0, torch.int64: 1, torch.float32: 2}
PAIRINGS = {"interleaved": 0, "halves": 1}


@dataclass(frozen=True)
class RotaryAxes:
    """Frequencies of a head's channel pairs and the axis whose position turns each.

    inv_freq: fp64 [pairs], radians per position; axis: int32 [pairs].  ``pairing``: pair i is channels (2i, 2i+1)
    ('interleaved') or (i, i + pairs) ('halves').  Channels from 2 * pairs on are not rotated."""
    inv_freq: torch.Tensor
    axis: torch.Tensor
    pairing: str = "interleaved"

    @classmethod
    def sections(cls, dims: Sequence[int], theta: float = 10000.0, pairing: str = "interleaved", shared: bool = False,
                 device=None) -> "RotaryAxes":
        """``dims``: rotated channels of each axis (even).  Each axis has frequencies theta ** (-2 i / dim) of its own;
        with ``shared``, one sequence theta ** (-2 i / sum(dims)) runs through all of them."""
        if not dims or any(d < 0 or d % 2 for d in dims) or sum(dims) == 0:
            raise ValueError(f"dims must be even and not all 0, got {tuple(dims)}")
        axis = torch.tensor([a for a, d in enumerate(dims) for _ in range(d // 2)], dtype=torch.int32)
        if shared:
            power = torch.arange(sum(dims) // 2, dtype=torch.float64) * (2 / sum(dims))
        else:
            power = torch.cat([torch.arange(d // 2, dtype=torch.float64) * (2 / max(d, 1)) for d in dims])
        return cls((float(theta) ** -power).to(device), axis.to(device), pairing)

    @classmethod
    def video(cls, head_dim: int, theta: float = 10000.0, device=None) -> "RotaryAxes":
        """Wan's split: height and width take 2 * (head_dim // 6) channels each, time the rest (44, 42, 42 of 128;
        the rotary_emb that the reference's processor is given, svg/models/wan/attention.py:31-57)."""
        hw = 2 * (head_dim // 6)
        return cls.sections((head_dim - 2 * hw, hw, hw), theta, device=device)


def grid_positions(frames: int, height: int, width: int, first_frame: int = 0, device=None) -> torch.Tensor:
    """int32 [3, frames * height * width]: time, height and width of a video's tokens, frame-major."""
    t = torch.arange(frames * height * width, device=device, dtype=torch.int32)
    return torch.stack([first_frame + t // (height * width), t // width % height, t % width])


def _tokens(t: torch.Tensor) -> Tuple[int, int]:
    """Batch and sequence of a [B, S, heads, D] or [tokens, heads, D] tensor."""
    return (1, t.shape[0]) if t.dim() == 3 else t.shape[:2]


def _check_tensor(t: torch.Tensor, name: str) -> None:
    if t.dim() not in (3, 4):
        raise ValueError(f"{name} must be [tokens, heads, D] or [B, S, heads, D], got {tuple(t.shape)}")
    if t.dtype not in _DTYPES:
        raise ValueError(f"{name}: dtype {t.dtype} is not bfloat16, float16 or float32")
    if t.numel() and t.stride(-1) != 1:
        raise ValueError(f"{name}: the channels must be contiguous, got stride {t.stride(-1)}")


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """First and last byte address (exclusive) that ``t`` reaches."""
    n = 1 + sum((s - 1) * st for s, st in zip(t.shape, t.stride())) if t.numel() else 0
    return t.data_ptr(), t.data_ptr() + n * t.element_size()


def _rotate(q, k, positions, axes, inverse, out):
    """The launch: outputs ``out`` (one for each of q, k)."""
    if not q.is_cuda:
        raise ValueError("the rotary kernel needs ROCm device tensors (there is no CPU path)")
    B, S = _tokens(q)
    pos_stride = positions.stride()
    if len(pos_stride) == 2:  # one row of positions serves every batch
        pos_stride = (pos_stride[0], 0, pos_stride[1])

    def tensor(x, y):
        xs, ys = x.stride(), y.stride()
        if len(xs) == 3:
            xs, ys = (0,) + xs, (0,) + ys
        return ctypes.byref(_lib.RopeTensor(x.data_ptr(), y.data_ptr(), xs[:3], ys[:3], x.shape[-2]))

    _lib.on_stream(q.device, "pasa_rope_axes", tensor(q, out[0]), None if k is None else tensor(k, out[1]), positions.data_ptr(),
                   _POS[positions.dtype], *pos_stride, positions.shape[0], axes.inv_freq.data_ptr(), axes.axis.data_ptr(),
                   axes.inv_freq.numel(), B, S, q.shape[-1], PAIRINGS[axes.pairing], int(inverse), _DTYPES[q.dtype])
    return out


def _new(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    if t is None:
        return None
    # A tensor whose elements share memory (an expanded one) gets an output of its own layout.
    return torch.empty(t.shape, dtype=t.dtype, device=t.device) if _lib.shares_memory(t) else torch.empty_like(t)


class _RopeAxes(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, axes, inverse):
        ctx.save_for_backward(positions, axes.inv_freq, axes.axis)
        ctx.pairing, ctx.inverse = axes.pairing, inverse
        ctx.set_materialize_grads(False)
        q_out, k_out = _rotate(q, k, positions, axes, inverse, (_new(q), _new(k)))
        return q_out if k is None else (q_out, k_out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dq, dk=None):
        positions, inv_freq, axis = ctx.saved_tensors
        axes = RotaryAxes(inv_freq, axis, ctx.pairing)
        grads = [None if d is None else d if d.numel() == 0 or d.stride(-1) == 1 else d.contiguous() for d in (dq, dk)]
        have = [d for d in grads if d is not None]
        out = iter(_rotate(have[0], have[1] if len(have) > 1 else None, positions, axes, not ctx.inverse,
                           tuple(_new(d) for d in have) + (None,) * (2 - len(have)))) if have else iter(())
        return tuple(None if d is None else next(out) for d in grads) + (None, None, None)


def rope_axes(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, axes: RotaryAxes, *,
              inverse: bool = False, inplace: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Rotate q and k (k may be None; it may have fewer heads) by the tokens' positions.

    q, k: [B, S, heads, D] or [tokens, heads, D] in bf16, fp16 or fp32, any strides but for the channels', which are
    contiguous ([B, heads, S, D] tensors are passed as ``t.transpose(1, 2)``).  positions: [axes, S] (for every
    batch) or [axes, B, S], int32, int64 or fp32.  The angle positions[axis[i]] * inv_freq[i] is reduced in fp64;
    the rotation is fp32, rounded once.  ``inverse`` turns back.  ``inplace`` writes q and k themselves (no
    gradient).  Returns (q, k).

    Under graph capture with gradients, leaves must have no living graph from before: torch ties a leaf's gradient to
    the stream of its first graph, and waiting for that stream breaks the capture.  Where such a graph came from here,
    the call is refused; ``q.detach().requires_grad_()`` is a leaf of its own."""
    _check_tensor(q, "q")
    if k is not None:
        _check_tensor(k, "k")
        if k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1] or k.dtype != q.dtype:
            raise ValueError(f"k must have q's tokens, head dim and dtype, got {k.dtype} {tuple(k.shape)} for q {q.dtype} {tuple(q.shape)}")
    B, S = _tokens(q)
    if positions.dtype not in _POS:
        raise ValueError(f"positions: dtype {positions.dtype} is not int32, int64 or float32")
    if tuple(positions.shape[1:]) not in ((S,), (B, S)) or positions.dim() < 2:
        raise ValueError(f"positions must be [axes, {S}] or [axes, {B}, {S}], got {tuple(positions.shape)}")
    if axes.pairing not in PAIRINGS:
        raise ValueError(f"unknown pairing {axes.pairing!r}")
    f, a = axes.inv_freq, axes.axis
    if f.dtype != torch.float64 or a.dtype != torch.int32 or f.dim() != 1 or f.shape != a.shape or \
            not (f.is_contiguous() and a.is_contiguous()):
        raise ValueError("RotaryAxes needs contiguous float64 inv_freq and int32 axis of one length")
    for name, t in (("k", k), ("positions", positions), ("inv_freq", f), ("axis", a)):
        if t is not None and t.device != q.device:
            raise ValueError(f"{name} is on {t.device}, q on {q.device}")
    if positions.requires_grad:
        raise ValueError("rope_axes has no gradient of the positions")
    if inplace:
        if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
            raise ValueError("rope_axes(inplace=True) has no gradient")
        if _lib.shares_memory(q) or (k is not None and _lib.shares_memory(k)):
            raise ValueError("rope_axes(inplace=True) needs tensors whose elements do not share memory")
        if k is not None and q.numel() and k.numel():
            (a0, a1), (b0, b1) = _span(q), _span(k)
            # q and k as slices of one projection interleave; otherwise they may not meet.
            if a0 < b1 and b0 < a1 and (q.untyped_storage().data_ptr() != k.untyped_storage().data_ptr() or
                                        not _slices_of_one(q, k)):
                raise ValueError("rope_axes(inplace=True): q and k share memory")
        _rotate(q, k, positions, axes, inverse, (q, k))
        return q, k
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        out = _RopeAxes.apply(q, k, positions, axes, inverse)
        _check_leaves(out if k is None else out[0], q.device)
        return (out, None) if k is None else out
    return tuple(_rotate(q, k, positions, axes, inverse, (_new(q), _new(k))))


def _check_leaves(out: torch.Tensor, device) -> None:
    """Mark the nodes that take the leaves' gradients with the stream that this module first met them on (a node lives as
    long as some graph of its leaf does), and refuse a capture beside a graph that was made on another one."""
    stream = _lib._raw_stream(device.index)
    for node, _ in out.grad_fn.next_functions:
        if hasattr(node, "variable") and node.metadata.setdefault("rope_axes stream", stream) != stream and \
                torch.cuda.is_current_stream_capturing():
            raise ValueError("rope_axes under graph capture: a graph of this leaf made on another stream is alive; give "
                             "the call t.detach().requires_grad_()")


def _slices_of_one(q: torch.Tensor, k: torch.Tensor) -> bool:
    """Whether q and k are [.., heads, D] slices, side by side, of the rows of one tensor."""
    if q.stride()[:-2] != k.stride()[:-2]:
        return False
    row = min([st for n, st in zip(q.shape[:-2], q.stride()[:-2]) if n > 1], default=1 << 62)
    reach = lambda t: (t.shape[-2] - 1) * t.stride(-2) + t.shape[-1]
    gap = (k.data_ptr() - q.data_ptr()) // q.element_size()
    return (gap >= reach(q) and gap + reach(k) <= row) or (-gap >= reach(k) and -gap + reach(q) <= row)
