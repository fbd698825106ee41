"""Which kernels a call of cross attention runs on, as the library says."""

import math

import pytest
import torch

from simple_vsa_b200 import _lib, video_cross_attn


def call_of(B, H, Hkv, Lq, Lkv, D, dtype=_lib.VSA_BF16, scale=0.1):
    """The arguments of a call on dense tensors; their addresses are never looked at."""
    a = _lib.Cross()
    a.B, a.H, a.Hkv, a.Lq, a.Lkv, a.D, a.dtype, a.scale = B, H, Hkv, Lq, Lkv, D, dtype, scale
    for i, n in enumerate(("q", "k", "v", "dout", "out", "dq", "dk", "dv")):
        setattr(a, n, 4096 * (i + 1))
        heads, rows = (Hkv, Lkv) if n in ("k", "v", "dk", "dv") else (H, Lq)
        getattr(a, n + "_stride")[:] = (heads * rows * D, rows * D, D)
    return a


def on_tensor_cores(a, backward):
    return _lib.lib.vsa_cross_on_tensor_cores(a, int(backward))


@pytest.mark.parametrize("args,forward,backward", [
    ((1, 40, 40, 92160, 512, 128), 1, 1), ((2, 12, 4, 8190, 1001, 64, _lib.VSA_F16), 1, 1), ((1, 2, 2, 9, 7, 8), 1, 1),
    ((8, 40, 40, 1, 512, 128), 0, 1),            # a row each: a pass over the keys, without tensor cores; its gradient is theirs
    ((1, 4, 2, 1, 300, 64), 0, 1), ((1, 4, 4, 2, 2048, 72), 0, 1), ((1, 4, 2, 1, 2049, 64), 1, 1),
    # from five rows on the tiles are faster, up to three times at eight; from three on where the pass over the keys fills the GPU
    ((8, 40, 8, 1, 512, 128), 1, 1), ((1, 4, 4, 3, 512, 64), 0, 1), ((1, 4, 2, 2, 513, 64), 1, 1), ((4, 80, 40, 2, 300, 64), 1, 1),
    ((4, 40, 40, 2, 300, 64), 0, 1), ((1, 4, 4, 5, 100, 64), 1, 1),
    ((1, 2, 2, 100, 100, 128, _lib.VSA_F32), 0, 0), ((1, 2, 2, 100, 100, 136), 0, 0), ((1, 2, 2, 100, 100, 20), 0, 0),
    ((1, 2, 2, 100, 100, 64, _lib.VSA_BF16, -1.0), 0, 0), ((1, 2, 2, 1, 100, 64, _lib.VSA_BF16, 0.0), 0, 0),
    ((1, 0, 0, 100, 100, 64), 0, 0), ((0, 2, 2, 100, 100, 64), 0, 0), ((1, 2, 2, 0, 100, 64), 0, 0), ((1, 2, 2, 100, 0, 64), 0, 0),
    ((1, 3, 2, 100, 100, 64), 0, 0)])
def test_which_calls_run_on_the_tensor_cores(args, forward, backward):
    a = call_of(*args)
    assert (on_tensor_cores(a, False), on_tensor_cores(a, True)) == (forward, backward)
    a.q = a.q + 2                                # rows off the 16-byte grid
    assert on_tensor_cores(a, False) == on_tensor_cores(a, True) == 0


def test_no_call_no_tensor_cores():
    assert _lib.lib.vsa_cross_on_tensor_cores(None, 0) == 0


def test_a_scale_that_fp32_does_not_hold_is_refused():
    from simple_vsa_b200 import cross
    assert cross._scale(None, 64) == 0.125 and cross._scale(-2e38, 64) == -2e38 and cross._scale(1e-60, 64) == 1e-60
    for scale in (1e39, -1e300, 3e38, math.inf, math.nan):
        with pytest.raises(ValueError, match="finite"):
            cross._scale(scale, 64)
    a = call_of(1, 2, 2, 100, 100, 64)
    for scale in (3e38, -3e38, math.inf, math.nan):
        a.scale = scale
        for f in (_lib.lib.vsa_cross_fwd, _lib.lib.vsa_cross_bwd):
            assert f(a, None) == _lib.ERR_BAD_ARGUMENT and "scale" in _lib.last_error()      # refused before any launch


@pytest.mark.parametrize("dtype,most", [(_lib.VSA_F16, 1 << 16), (_lib.VSA_BF16, 1 << 19)])
def test_long_sums_are_cut(dtype, most):
    """The tensor cores' accumulators drop low bits: no sum of more terms than a half step of the type allows is left to one of them."""
    for Lq in (300, 92160):
        a = call_of(1, 8, 8, Lq, most, 64, dtype)
        assert on_tensor_cores(a, False) and on_tensor_cores(a, True)
        a = call_of(1, 8, 8, Lq, most + 1, 64, dtype)
        assert on_tensor_cores(a, False) and not on_tensor_cores(a, True)
    space = lambda backward, H, Hkv, Lq, Lkv, mask=0: _lib.lib.vsa_cross_workspace_bytes(backward, 1, H, Hkv, Lq, Lkv, 64, dtype, mask)
    # forward with enough query rows for the GPU: parts of the keys only where they are too many
    part = 296 * 256 * 65 * 4
    assert space(0, 296, 1, 256, most) == 0
    for keys, parts in ((most + 1, 2), (4 * most, 4), (256 * most, 256)):
        assert space(0, 296, 1, 256, keys) >= parts * part and space(0, 296, 1, 256, keys) % part == 0
    # dK and dV with enough key heads: parts of the query rows of all heads that share one
    part = 2 * 148 * 16 * 64 * 4
    assert space(1, 148, 148, most, 16) == 0
    for H, rows, parts in ((148, most + 1, 2), (148, 4 * most, 4), (592, most, 4), (148, 128 * most, 128)):
        assert space(1, H, 148, rows, 16) >= parts * part and space(1, H, 148, rows, 16) % part == 0
    # keys of a backward off the tensor cores are not gathered
    assert space(1, 8, 8, 92160, most, 1) > space(1, 8, 8, 92160, most) and space(1, 8, 8, 92160, 2 * most, 1) == space(1, 8, 8, 92160, 2 * most)


# Sums of terms of one sign, where dropped bits add up; the softmax's weights are exact here (1, or a power of two).  Off: half a step of the
# type for the result's rounding, and 2^-27 for each of the terms of one accumulator (2^16 in fp16, 2^19 in bf16): another half step.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,keys", [(torch.float16, 1 << 16), (torch.float16, 1 << 20), (torch.bfloat16, 1 << 19), (torch.bfloat16, 1 << 22)])
def test_forward_sums_of_many_keys(dtype, keys):
    q, k = torch.zeros(1, 296, 256, 8, device="cuda", dtype=dtype), torch.zeros(1, 1, keys, 8, device="cuda", dtype=dtype)
    v = torch.linspace(0.5, 1.5, 1024, device="cuda").to(dtype).repeat(keys // 1024)[None, None, :, None].expand(1, 1, keys, 8).contiguous()
    with torch.no_grad():
        out = video_cross_attn(q, k, v)
    assert _lib.device_status() == 0
    want = v.double().mean()
    assert ((out.double() - want).abs() <= want * torch.finfo(dtype).eps).all(), (out.double() / want - 1).abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("keys", [1 << 16, 1 << 20])
def test_gradient_of_the_queries_of_many_keys(keys):
    L, D, eps = 130, 8, torch.finfo(torch.float16).eps
    v = torch.randn(1, 1, keys, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    dout = torch.ones(1, 1, L, D, device="cuda").half()
    k = v.double().sum(-1, keepdim=True).expand(1, 1, keys, D).half()       # along dP: the terms of dQ are squares
    q = torch.zeros(1, 1, L, D, device="cuda", dtype=torch.float16, requires_grad=True)
    (dq,) = torch.autograd.grad(video_cross_attn(q, k, v, sm_scale=1.0), q, dout)
    assert _lib.device_status() == 0
    dp = v.double().sum(-1)[0, 0]
    want = ((dp - dp.mean())[:, None] * k.double()[0, 0]).mean(0)
    # delta comes from the rounded output and moves dq by its error times the mean of k
    off = want.abs() * eps + D * eps / 2 * v.double().mean((0, 1, 2)).abs().max() * k.double().mean().abs()
    assert ((dq.double() - want).abs() <= off).all(), (dq.double() / want - 1).abs().max()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1 << 16, 1 << 20])
def test_gradient_of_the_values_of_many_queries(rows):
    H, T = 148, 16
    q = torch.zeros(1, H, rows, 8, device="cuda", dtype=torch.float16)
    k = torch.zeros(1, H, T, 8, device="cuda", dtype=torch.float16)
    v = torch.zeros_like(k).requires_grad_()
    column = (torch.linspace(0.5, 1.5, 1024, device="cuda") * 2.0 ** -7).half()
    dout = column.repeat(rows // 1024)[None, None, :, None].expand(1, H, rows, 8).contiguous()
    (dv,) = torch.autograd.grad(video_cross_attn(q, k, v), v, dout)
    assert _lib.device_status() == 0
    want = column.double().mean() * rows / T
    assert ((dv.double() - want).abs() <= want * torch.finfo(torch.float16).eps).all(), (dv.double() / want - 1).abs().max()
