"""Which kernels a call of cross attention runs on, as the library says."""

import math

import pytest

from simple_vsa_b200 import _lib


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
    ((8, 40, 8, 1, 512, 128), 0, 1), ((1, 4, 2, 4, 300, 64), 0, 1), ((1, 4, 2, 5, 300, 64), 1, 1),
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
