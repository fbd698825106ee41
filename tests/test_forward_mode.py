"""Forward-mode derivatives: no operator here has them, and each says so instead of returning an output without its tangent."""

import pytest
import torch
from torch.autograd import forward_ad

import simple_vsa_b200 as V

DEV = "cuda:0"


def test_which_calls_are_differentiated():
    from simple_vsa_b200 import ops
    x = torch.ones(2, 3)
    leaf = torch.ones(2, 3, requires_grad=True)
    assert not ops._differentiated(x, None, x) and ops._differentiated(x, leaf, None)
    with torch.no_grad():
        assert not ops._differentiated(leaf)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, x)
        assert ops._differentiated(x, dual) and not ops._differentiated(x)
        assert ops._differentiated(dual.view(3, 2).contiguous())
        with torch.no_grad():
            assert ops._differentiated(None, dual)
        table = {"cos": torch.ones(3, 1), "sin": forward_ad.make_dual(torch.ones(3, 1), torch.ones(3, 1))}
        from simple_vsa_b200 import rotary
        with pytest.raises(ValueError, match="constant"):
            rotary._table(table, 8, torch.device("cpu"))
    assert not ops._differentiated(x)


@pytest.mark.gpu
@pytest.mark.parametrize("grad", [True, False])
def test_a_tangent_is_refused_not_dropped(grad):
    x = torch.randn(1, 2, 6, 16, device=DEV)
    rot = V.build_rotary_metadata((6,), 8, device=DEV)
    meta = V.build_vsa_metadata((1, 2, 3), (1, 2, 2), device=DEV)
    swap = lambda t: t.transpose(1, 2)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: V.video_cross_attn(dual, x, x), lambda: V.video_cross_attn(x, dual, x), lambda: V.video_cross_attn(x, x, dual),
                     lambda: V.video_cross_attn_raster(swap(x), swap(x), swap(dual)), lambda: V.video_rotary(dual, x, rot),
                     lambda: V.video_rotary(x, dual, rot), lambda: V.video_rotary_raster(swap(dual), None, rot),
                     lambda: V.tile_heads(swap(dual), meta, rot)):
            with pytest.raises(NotImplementedError):
                call()
        V.video_cross_attn(x, x, x)
        V.video_rotary(x, x, rot)
