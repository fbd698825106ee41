"""Cross attention of the video tokens to an encoder's states: every query attends to all live keys of its sample.

Beside the sparse self-attention of a video transformer's layer stands a dense attention to the states of a prompt (or an image)
encoder: queries by the ten thousand, keys by the hundred, of another length per sample.  ``video_cross_attn`` takes
``[batch, heads, seq_len, dim]`` tensors, ``video_cross_attn_raster`` the ``[batch, seq_len, heads, head_dim]`` that the
projections leave; both read and write any strides with a contiguous head dim in place.
"""

from __future__ import annotations

import math
from typing import Optional

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib, ops
from ._lib import call


def _usable(x: Tensor) -> Tensor:
    """The tensor itself where its rows can be read in place, else a dense copy: head dim contiguous, and in 16-bit types with
    head dims of whole 16-byte pieces everything on 16-byte boundaries (other rows run on CUDA cores, element by element)."""
    shape, stride = x.shape, x.stride()
    if shape[3] > 1 and stride[3] != 1:
        return x.contiguous()
    if shape[3] % 8 == 0 and x.dtype != torch.float32:
        if x.data_ptr() % 16 or (stride[0] | stride[1] | stride[2]) % 8 or not (stride[0] and stride[1] and stride[2]):
            if x.data_ptr() % 16 or any(n > 1 and (s % 8 or s == 0) for s, n in zip(stride[:3], shape[:3])):
                return ops._dense(x)
    return x


_PACK = _lib.Cross.PACK.pack
_ARGUMENTS = _lib.Cross.from_buffer_copy
_NO_STRIDES = (0, 0, 0)
_LARGEST = torch.finfo(torch.float32).max


def _steps(x: Optional[Tensor], raster: bool):
    """Batch, head and token stride."""
    if x is None:
        return _NO_STRIDES
    a, b, c, _ = x.stride()
    return (a, c, b) if raster else (a, b, c)


def _launch(name: str, backward: int, raster: bool, scale: float, dt: int, q, k, v, out, lse, kv_lengths, key_bits, dout=None,
            dq=None, dk=None, dv=None, delta=None) -> None:
    if raster:
        (B, Lq, H, D), (_, Lkv, Hkv, _) = q.shape, k.shape
    else:
        (B, H, Lq, D), (_, Hkv, Lkv, _) = q.shape, k.shape
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    n = _lib.lib.vsa_cross_workspace_bytes(backward, B, H, Hkv, Lq, Lkv, D, dt, key_bits is not None)
    ws = torch.empty(n, device=q.device, dtype=torch.uint8) if n > 0 else None
    bounds = torch.empty(B * Hkv * _lib.Cross.BOUNDS, device=q.device, dtype=torch.float32) if backward and dt == _lib.VSA_F16 else None
    grads = (*_steps(dout, raster), *_steps(dq, raster), *_steps(dk, raster), *_steps(dv, raster)) if backward else _NO_STRIDES * 4
    a = _ARGUMENTS(_PACK(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), ptr(dout), out.data_ptr(), ptr(dq), ptr(dk), ptr(dv), lse.data_ptr(), ptr(delta),
        ptr(kv_lengths), ptr(key_bits), ptr(ws), ptr(bounds), B, H, Hkv, Lq, Lkv, *_steps(q, raster), *_steps(k, raster), *_steps(v, raster),
        *_steps(out, raster), *grads, scale, D, dt))
    call(name, a, ops._stream(q.device))


def _forward(q, k, v, kv_lengths, key_bits, scale: float, raster: bool):
    B, H, L, D = q.shape
    if raster:
        H, L = L, H
    out = ops._like(q)
    lse = torch.empty((B * H, -(-L // 128) * 128), device=q.device, dtype=torch.float32)
    _launch("vsa_cross_fwd", 0, raster, scale, ops._check_device_dtype(q, k, v), q, k, v, out, lse, kv_lengths, key_bits)
    return out, lse


def _key_bits(kv_mask: Tensor, kv_lengths: Optional[Tensor]) -> Tensor:
    """The mask packed to a bit per key, whole tiles of 128 keys, the lengths folded in."""
    B, T = kv_mask.shape
    bits = torch.empty((B, -(-T // 128) * 4), device=kv_mask.device, dtype=torch.int32)
    call("vsa_cross_key_bits", kv_mask.data_ptr(), kv_mask.stride(0), ops._ptr(kv_lengths), bits.data_ptr(), B, T,
         ops._stream(kv_mask.device))
    return bits


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_lengths, key_bits, scale, raster):
        out, lse = _forward(q, k, v, kv_lengths, key_bits, scale, raster)
        ctx.save_for_backward(q, k, v, out, lse, kv_lengths, key_bits)
        ctx.scale, ctx.raster = scale, raster
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, out, lse, kv_lengths, key_bits = ctx.saved_tensors
        with torch.cuda.device(q.device):
            dq, delta = ops._like(q), torch.empty_like(lse)
            # the pass over the keys is left out where neither needs its gradient
            dk, dv = (ops._like(k), ops._like(v)) if ctx.needs_input_grad[1] or ctx.needs_input_grad[2] else (None, None)
            _launch("vsa_cross_bwd", 1, ctx.raster, ctx.scale, ops._check_device_dtype(q, k, v), q, k, v, out, lse, kv_lengths, key_bits,
                    _usable(dout), dq, dk, dv, delta)
        return dq, dk, dv, None, None, None, None


def _scale(sm_scale: Optional[float], dim: int) -> float:
    scale = float(sm_scale) if sm_scale is not None else 1.0 / math.sqrt(dim)
    if not abs(scale) * math.log2(math.e) <= _LARGEST:           # the kernels' factor of exponents of two, in fp32
        raise ValueError(f"sm_scale must be finite in fp32 (magnitude up to {_LARGEST * math.log(2):.3g}), got {scale}")
    return scale


def _attend(q, k, v, kv_lengths, kv_mask, sm_scale, raster: bool) -> Tensor:
    layout = "[batch, seq_len, heads, head_dim]" if raster else "[batch, heads, seq_len, dim]"
    if q.ndim != 4 or k.ndim != 4 or v.ndim != 4:
        raise ValueError(f"q, k, and v must have shape {layout}")
    seq, head = (1, 2) if raster else (2, 1)
    B, H, D = q.shape[0], q.shape[head], q.shape[3]
    T, Hkv = k.shape[seq], k.shape[head]
    if k.shape[0] != B or v.shape[0] != B:
        raise ValueError("q, k, and v must share the batch dimension")
    if v.shape[head] != Hkv or v.shape[seq] != T:
        raise ValueError("k and v must have the same heads and sequence length")
    if Hkv == 0 and H or Hkv and H % Hkv:
        raise ValueError(f"the {H} query heads must be a multiple of the {Hkv} key heads")
    if k.shape[3] != D or v.shape[3] != D:
        raise ValueError("q, k, and v must have the same head dimension")
    if not 1 <= D <= 256:
        raise ValueError(f"cross attention supports head dimensions from 1 to 256, got {D}")
    ops._check_device_dtype(q, k, v)
    if kv_lengths is not None and (not ops._integers(kv_lengths) or tuple(kv_lengths.shape) != (B,)):
        raise ValueError(f"kv_lengths must hold {B} integers of a signed type or uint8, one per sample")
    if kv_mask is not None and (kv_mask.dtype != torch.bool or tuple(kv_mask.shape) != (B, T)):
        raise ValueError(f"kv_mask must be a bool tensor of shape [{B}, {T}], True where a key takes part")
    scale = _scale(sm_scale, D)
    with torch.cuda.device(q.device):
        if kv_lengths is not None:
            if kv_lengths.dtype == torch.int64:
                kv_lengths = kv_lengths.clamp(0, T)
            kv_lengths = ops._sizes(kv_lengths, q.device)
        key_bits = None
        if kv_mask is not None:
            kv_mask = kv_mask.to(q.device)
            key_bits = _key_bits(kv_mask if T <= 1 or kv_mask.stride(1) == 1 else kv_mask.contiguous(), kv_lengths)
        q, k, v = _usable(q), _usable(k), _usable(v)
        if ops._differentiated(q, k, v):
            return _CrossAttention.apply(q, k, v, kv_lengths, key_bits, scale, raster)
        return _forward(q, k, v, kv_lengths, key_bits, scale, raster)[0]


def video_cross_attn(q: Tensor, k: Tensor, v: Tensor, kv_lengths: Optional[Tensor] = None, *, kv_mask: Optional[Tensor] = None,
                     sm_scale: Optional[float] = None) -> Tensor:
    """Attention of ``q [batch, heads, seq_len, dim]`` to ``k, v [batch, kv_heads, kv_len, dim]`` of another length.

    ``heads`` is a multiple of ``kv_heads``; neighbouring query heads share a key head.  Key j of sample b takes part where
    ``j < kv_lengths[b]`` (None: all; lengths beyond kv_len are kv_len) and ``kv_mask[b, j]`` (bool, None: all).  What stands in
    the other keys and values does not matter, NaN included; a sample without a key that takes part gives zeros and zero
    gradients.  Scale ``1/sqrt(dim)`` unless ``sm_scale`` says otherwise (finite in fp32).  bf16, fp16 or fp32; head dims up to 256.  In
    16-bit types with head dims that are multiples of 8 up to 128 and a positive scale the tensor cores do the work (a backward up to
    2^19 keys in bf16, 2^16 in fp16); the rest runs on CUDA cores in fp32, many times slower per FLOP.  Differentiable in q, k and v;
    forward-mode derivatives are refused."""
    return _attend(q, k, v, kv_lengths, kv_mask, sm_scale, False)


def video_cross_attn_raster(q: Tensor, k: Tensor, v: Tensor, kv_lengths: Optional[Tensor] = None, *,
                            kv_mask: Optional[Tensor] = None, sm_scale: Optional[float] = None) -> Tensor:
    """:func:`video_cross_attn` for ``[batch, seq_len, heads, head_dim]`` activations, as the projections leave them; no tensor is
    re-laid, and the output comes in the same layout."""
    return _attend(q, k, v, kv_lengths, kv_mask, sm_scale, True)
