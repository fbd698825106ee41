"""Rotary positions of q and k: a table of angles per token grid, and the rotation as one kernel over both tensors.

``build_rotary_metadata`` is to the rotation what ``build_vsa_metadata`` is to the tiling: made once per latent shape and
handed to every call.  ``video_rotary`` works on ``[batch, heads, seq_len, dim]`` tensors (with ``positions=meta["tile_map"]``
where they are in tile order), ``video_rotary_raster`` on ``[batch, seq_len, heads, dim]``; ``tile_heads`` and
``video_sparse_attn_raster`` take the same metadata and rotate on the way into tile order.
"""

from __future__ import annotations

import math
from typing import Dict, Optional, Sequence, Tuple, Union

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib, ops
from ._lib import call

Scaling = Optional[Dict[str, object]]


def _axis_frequencies(dims: int, theta: float, scaling: Scaling, device) -> Tuple[Tensor, float]:
    """Angle per position of an axis's ``dims/2`` pairs (float64), and the factor of its cosines and sines."""
    pairs = torch.arange(0, dims, 2, device=device, dtype=torch.float64)
    if scaling is None:
        return theta ** (-pairs / max(1, dims)), 1.0
    kind, factor = scaling.get("kind"), float(scaling.get("factor", 1.0))
    if not factor > 0 or not math.isfinite(factor):
        raise ValueError("rotary scaling factor must be positive")
    if kind == "linear":                      # positions squeezed into the trained range
        return theta ** (-pairs / max(1, dims)) / factor, 1.0
    if kind == "ntk":                         # a larger base: the slowest pair slows down by `factor`, the fastest stays
        return (theta * factor ** (dims / (dims - 2.0)) if dims > 2 else theta) ** (-pairs / max(1, dims)), 1.0
    if kind == "yarn":                        # pairs that turn often within the trained length stay, slow ones are squeezed
        length = scaling.get("original_length")
        if length is None or not float(length) > 0:
            raise ValueError("rotary scaling 'yarn' needs a positive original_length")
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not fast > slow:
            raise ValueError("rotary scaling 'yarn' needs beta_fast > beta_slow")
        freq = theta ** (-pairs / max(1, dims))
        keep = ((freq * float(length) / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        return freq * keep + freq / factor * (1.0 - keep), 1.0 + 0.1 * math.log(factor) if factor > 1 else 1.0
    raise ValueError(f"rotary scaling kind must be 'linear', 'ntk' or 'yarn', got {kind!r}")


def build_rotary_metadata(dit_seq_shape: Sequence[int], rotary_dim: int, *, axes_dims: Optional[Sequence[int]] = None,
                          theta: float = 10000.0, scaling: Union[Scaling, Sequence[Scaling]] = None,
                          interleaved: bool = True, device="cpu") -> Dict[str, object]:
    """Rotary table of a token grid: ``cos`` and ``sin`` ``[tokens, rotary_dim/2]`` fp32, rows in raster order.

    ``dit_seq_shape`` is ``(T, H, W)``, or ``(tokens,)`` for text.  The pairs of a head are dealt to the axes in order,
    ``axes_dims`` dims each (default: equal shares, what is left over to the first).  ``scaling`` stretches the positions for
    grids beyond the trained one: ``{"kind": "linear" | "ntk" | "yarn", "factor": f, ...}`` for every axis, or one such
    dict or None per axis (yarn: ``original_length``, ``beta_fast``, ``beta_slow``).  Angles are computed in float64: those of
    far positions would lose their fraction in 32 bits.  ``interleaved`` says how a head's pairs lie: ``(2i, 2i+1)``, or
    halves ``(i, i + rotary_dim/2)``."""
    shape = tuple(int(n) for n in dit_seq_shape)
    if not shape or any(n < 0 for n in shape):
        raise ValueError("dit_seq_shape must hold the extents of the token grid")
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_dim must be a positive even number, got {rotary_dim}")
    axes, pairs = len(shape), rotary_dim // 2
    if axes_dims is None:
        share = pairs // axes
        axes_dims = [2 * (pairs - (axes - 1) * share)] + [2 * share] * (axes - 1)
    axes_dims = [int(d) for d in axes_dims]
    if len(axes_dims) != axes or sum(axes_dims) != rotary_dim or any(d < 0 or d % 2 for d in axes_dims):
        raise ValueError(f"axes_dims must be {axes} even numbers that add up to rotary_dim={rotary_dim}")
    if not theta > 0:
        raise ValueError("theta must be positive")
    per_axis = [scaling] * axes if scaling is None or isinstance(scaling, dict) else list(scaling)
    if len(per_axis) != axes:
        raise ValueError(f"scaling must be one dict, or one entry for each of the {axes} axes")
    cos, sin = [], []
    for axis, (n, d, how) in enumerate(zip(shape, axes_dims, per_axis)):
        freq, factor = _axis_frequencies(d, float(theta), how, device)
        angle = torch.arange(n, device=device, dtype=torch.float64)[:, None] * freq[None, :]
        view = [1] * axes + [d // 2]
        view[axis] = n
        for parts, values in ((cos, angle.cos()), (sin, angle.sin())):
            parts.append((values * factor).float().view(view).expand(*shape, d // 2))
    return {"cos": torch.cat(cos, dim=-1).reshape(-1, pairs).contiguous(),
            "sin": torch.cat(sin, dim=-1).reshape(-1, pairs).contiguous(), "interleaved": bool(interleaved)}


def _table(rotary: Dict[str, object], head_dim: int, device) -> Tuple[Tensor, Tensor, bool]:
    """The metadata's tables on the tensors' device, checked."""
    cos, sin = rotary["cos"], rotary["sin"]
    if cos.ndim != 2 or cos.shape != sin.shape:
        raise ValueError("the rotary table's cos and sin must share the shape [positions, rotary_dim/2]")
    if 2 * cos.shape[1] > head_dim:
        raise ValueError(f"the rotary table turns {2 * cos.shape[1]} dims of a head, the tensors have {head_dim}")
    if cos.requires_grad or sin.requires_grad or ops._has_tangent(cos) or ops._has_tangent(sin):
        raise ValueError("the rotary table is a constant: it receives no gradient")
    if cos.device != device or cos.dtype != torch.float32 or sin.device != device or sin.dtype != torch.float32:
        cos, sin = cos.to(device=device, dtype=torch.float32), sin.to(device=device, dtype=torch.float32)
    cos, sin = cos.contiguous(), sin.contiguous()
    return cos, sin, bool(rotary.get("interleaved", True))


def _rows(x: Tensor) -> Tensor:
    """The tensor itself where its head dim is contiguous (any other strides), else a dense copy."""
    return x if x.stride(3) == 1 or x.shape[3] <= 1 else x.contiguous()


_DTYPES = {torch.bfloat16: _lib.VSA_BF16, torch.float16: _lib.VSA_F16, torch.float32: _lib.VSA_F32}
_PACK = _lib.Rotary.PACK.pack
_ARGUMENTS = _lib.Rotary.from_buffer_copy


def rotate(xs, ys, cos, sin, interleaved: bool, inverse: bool, *, x_raster: bool, y_raster: bool, positions=None,
           src_map=None) -> None:
    """``ys[i]`` = ``xs[i]`` with its heads turned (one or two tensors, one launch); the layouts may differ where
    ``src_map`` moves the rows."""
    x0, y0, x1, y1 = xs[0], ys[0], xs[-1], ys[-1]
    (xa, xb, xc, _), (xd, xe, xf, _), (ya, yb, yc, _), (yd, ye, yf, _) = x0.stride(), x1.stride(), y0.stride(), y1.stride()
    if x_raster:
        xb, xc, xe, xf = xc, xb, xf, xe
    if y_raster:
        yb, yc, ye, yf = yc, yb, yf, ye
        B, rows, heads, D = y0.shape
    else:
        B, heads, rows, D = y0.shape
    a = _ARGUMENTS(_PACK(
        x0.data_ptr(), x1.data_ptr(), y0.data_ptr(), y1.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        0 if positions is None else positions.data_ptr(), 0 if src_map is None else src_map.data_ptr(),
        B, rows, x0.shape[1 if x_raster else 2], cos.shape[0], rows if positions is not None and positions.ndim == 2 else 0,
        xa, xb, xc, xd, xe, xf, ya, yb, yc, yd, ye, yf,
        heads, y1.shape[2 if y_raster else 1] if len(ys) > 1 else 0, D, 2 * cos.shape[1], interleaved, inverse, _DTYPES[y0.dtype]))
    call("vsa_rotary", a, ops._stream(y0.device))


def _turned(q, k, cos, sin, positions, interleaved, raster):
    xs = [_rows(x) for x in ((q,) if k is None else (q, k))]
    ys = [ops._like(x) for x in xs]
    rotate(xs, ys, cos, sin, interleaved, False, x_raster=raster, y_raster=raster, positions=positions)
    return ys[0], ys[1] if k is not None else None


class _Rotary(torch.autograd.Function):
    """Both tensors in one launch; the backward is the same kernel with the angles reversed, on whichever gradients came."""

    @staticmethod
    def forward(ctx, q, k, cos, sin, positions, interleaved, raster):
        ctx.save_for_backward(cos, sin, positions)
        ctx.interleaved, ctx.raster = interleaved, raster
        ctx.set_materialize_grads(False)
        return _turned(q, k, cos, sin, positions, interleaved, raster)

    @staticmethod
    @once_differentiable
    def backward(ctx, dq, dk):
        (cos, sin, positions), raster = ctx.saved_tensors, ctx.raster
        with torch.cuda.device(cos.device):
            there = [_rows(g) for g in (dq, dk) if g is not None]
            back = [ops._like(g) for g in there]
            if there:
                rotate(there, back, cos, sin, ctx.interleaved, True, x_raster=raster, y_raster=raster, positions=positions)
        return back[0] if dq is not None else None, back[-1] if dk is not None else None, None, None, None, None, None


def _turn(q: Tensor, k: Optional[Tensor], rotary: Dict[str, object], positions: Optional[Tensor], raster: bool):
    layout = "[batch, seq_len, heads, head_dim]" if raster else "[batch, heads, seq_len, dim]"
    if q.ndim != 4 or (k is not None and k.ndim != 4):
        raise ValueError(f"q and k must have shape {layout}")
    ops._check_device_dtype(q, q if k is None else k, q)
    seq = 1 if raster else 2
    B, L, D = q.shape[0], q.shape[seq], q.shape[3]
    if k is not None and (k.shape[0] != B or k.shape[seq] != L or k.shape[3] != D):
        raise ValueError("q and k must share batch, sequence length and head dimension")
    if D > 256:
        raise ValueError(f"rotary positions support head dimensions up to 256, got {D}")
    cos, sin, interleaved = _table(rotary, D, q.device)
    if positions is None:
        if cos.shape[0] < L:
            raise ValueError(f"the rotary table holds {cos.shape[0]} positions, the tensors hold {L} tokens")
    else:
        if not ops._integers(positions):
            raise ValueError("positions must be integers of a signed type or uint8")
        if tuple(positions.shape) not in ((L,), (B, L)):
            raise ValueError(f"positions must have shape [{L}] or [{B}, {L}], got {list(positions.shape)}")
        if positions.dtype == torch.int64:           # a position beyond 32 bits stays outside the table
            positions = positions.clamp(-1, 2 ** 31 - 1)
    with torch.cuda.device(q.device):
        if positions is not None:
            positions = positions.to(device=q.device, dtype=torch.int32).contiguous()
        out_q, out_k = (_Rotary.apply if ops._differentiated(q, k) else _turned)(q, k, cos, sin, positions, interleaved, raster)
    return out_q if k is None else (out_q, out_k)


def video_rotary(q: Tensor, k: Optional[Tensor], rotary: Dict[str, object], *, positions: Optional[Tensor] = None):
    """q and k ``[batch, heads, seq_len, dim]`` (their head counts may differ, k may be None) with rotary positions.

    The first ``rotary_dim`` dims of each head turn by the angles of the token's row of the table (``rotary`` from
    ``build_rotary_metadata``, or any dict of ``cos``, ``sin`` ``[positions, rotary_dim/2]`` and ``interleaved``); the rest are
    copied.  Row of token l: l, or ``positions[l]`` / ``positions[b, l]`` -- ``meta["tile_map"]`` for tensors in tile order,
    the step of each sample for single tokens.  A position outside the table (a padding token's -1) leaves the token as it
    is.  fp32 arithmetic, one rounding; differentiable in q and k.  Returns ``(q, k)``, or q alone without a k."""
    return _turn(q, k, rotary, positions, False)


def video_rotary_raster(q: Tensor, k: Optional[Tensor], rotary: Dict[str, object], *, positions: Optional[Tensor] = None):
    """:func:`video_rotary` for ``[batch, seq_len, heads, head_dim]`` activations."""
    return _turn(q, k, rotary, positions, True)
