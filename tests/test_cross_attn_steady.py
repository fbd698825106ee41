"""Cross attention in the state that long calls spend their time in: persistent CTAs with several pieces of work, pieces of several key
tiles that are not cut, rings of shared memory that wrap, accumulators that the next piece takes over.  Against float64, head by head.

The shapes are checked to be of that kind: the tensor path, no workspace (nothing is cut), more than two pieces a CTA of the forward."""

import math

import pytest
import torch

from simple_vsa_b200 import _lib, video_cross_attn, video_cross_attn_raster
from tests.test_cross_attn import DEV, _bound, _live
from tests.test_cross_attn_kernels import call_of, on_tensor_cores

SMS = 148


def _exact(q, k, v, live, scale, dout):
    """The formulas in float64 on the device, sample by sample, and what dq and dk may be off by [B, heads] because delta is formed from
    the rounded output (derived beside the oracle of the small shapes)."""
    B, H, L, D = q.shape
    Hk, T = k.shape[1:3]
    G, e = H // Hk, 2 * torch.finfo(q.dtype).eps / 2
    out = [torch.zeros(x.shape, device=DEV, dtype=torch.float64) for x in (q, q, k, k)]
    off_q, off_k = torch.zeros(B, H, device=DEV, dtype=torch.float64), torch.zeros(B, Hk, device=DEV, dtype=torch.float64)
    for b in range(B):
        at = live[b].nonzero().flatten().to(DEV)
        if at.numel() == 0:
            continue
        qq, dd = q[b].double(), dout[b].double()
        kk, vv = (x[b][:, at].double().repeat_interleave(G, 0) for x in (k, v))
        p = torch.softmax(qq @ kk.transpose(1, 2) * scale, dim=-1)
        o = p @ vv
        ds = p * (dd @ vv.transpose(1, 2) - (dd * o).sum(-1, keepdim=True)) * scale
        out[0][b], out[1][b] = o, ds @ kk
        dk, dv = ds.transpose(1, 2) @ qq, p.transpose(1, 2) @ dd
        out[2][b][:, at], out[3][b][:, at] = (x.view(Hk, G, -1, D).sum(1) for x in (dk, dv))
        ei = e * (o * dd).norm(dim=-1) * scale
        off_q[b] = (ei * (p @ kk).norm(dim=-1)).norm(dim=-1)
        rows = (p.square().transpose(1, 2) @ (ei * qq.norm(dim=-1)).square().unsqueeze(-1)).sum((1, 2))
        off_k[b] = 2 * rows.view(Hk, G).sum(1).sqrt()
    return out, (0 * off_q, off_q, off_k, 0 * off_k)


def _compare(got, want, off, dtype, slack=1.0):
    for name, x, y, o in zip(("out", "dq", "dk", "dv"), got, want, off):
        x = x.detach().double()
        assert torch.isfinite(x).all(), name
        err, norm = (x - y).norm(dim=(2, 3)), y.norm(dim=(2, 3))
        bad = err > slack * _bound(dtype) * norm + o
        assert not bad.any(), (name, bad.nonzero()[:5].tolist(), (err / norm).max().item())


def _inputs(B, H, Hk, L, T, D, dtype, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    make = lambda h, n: torch.randn(B, h, n, D, device=DEV, generator=g).to(dtype)
    return make(H, L), make(Hk, T), make(Hk, T), make(H, L)


def _run(q, k, v, dout, lengths=None, mask=None, raster=False):
    f = video_cross_attn_raster if raster else video_cross_attn
    turn = (lambda x: x.transpose(1, 2).contiguous()) if raster else (lambda x: x)
    leaves = [turn(x.detach()).requires_grad_() for x in (q, k, v)]
    out = f(*leaves, lengths, kv_mask=mask)
    res = [out.detach(), *torch.autograd.grad(out, leaves, turn(dout))]
    assert _lib.device_status() == 0
    return [x.transpose(1, 2) for x in res] if raster else res


def _space(backward, B, H, Hk, L, T, D, code):
    return _lib.lib.vsa_cross_workspace_bytes(backward, B, H, Hk, L, T, D, code, 0)


SHAPES = [  # B, H, Hk, L, T; parts that dK/dV is cut into
    (4, 40, 20, 641, 400, 1),          # 480 pieces of two query tiles, the last of a single row more than one; 22 steps of dK/dV
    (4, 40, 8, 600, 400, 1),           # last pieces of one query tile; 50 steps
    (4, 40, 10, 900, 400, 2),          # 640 pieces; dK/dV in two parts of 30 steps
]


@pytest.mark.parametrize("code", [_lib.VSA_BF16, _lib.VSA_F16])
@pytest.mark.parametrize("D", [64, 72, 128])
@pytest.mark.parametrize("B,H,Hk,L,T,parts", SHAPES)
def test_the_shapes_are_of_that_kind(B, H, Hk, L, T, parts, D, code):
    a = call_of(B, H, Hk, L, T, D, code)
    assert on_tensor_cores(a, False) and on_tensor_cores(a, True)
    assert _space(0, B, H, Hk, L, T, D, code) == 0 and B * H * -(-L // 256) > 3 * SMS and T > 3 * 128
    assert _space(1, B, H, Hk, L, T, D, code) == (0 if parts == 1 else parts * 2 * B * Hk * T * D * 4)
    assert B * H * -(-L // 128) > 3 * SMS                                   # pieces of dQ
    assert -(-L // 64) * (H // Hk) // parts > 3 * 5                         # steps of dK/dV: its rings of five wrap three times


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float16, 64), (torch.float16, 128), (torch.bfloat16, 72)])
@pytest.mark.parametrize("B,H,Hk,L,T,parts", SHAPES)
def test_many_pieces_a_cta(B, H, Hk, L, T, parts, D, dtype):
    """All keys; lengths of a full, no, one and a little more than one tile's keys, so that pieces of different lengths and without keys
    follow each other on a CTA; a mask.  NaN and infinities where no key takes part."""
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, dtype, L + D)
    lengths = torch.tensor([T, 0, 65, 129])
    mask = torch.rand(B, T, generator=torch.Generator().manual_seed(L)) < 0.6
    mask[3] = False
    for ln, mk in ((None, None), (lengths, None), (lengths.flip(0), None), (None, mask)):
        live = _live(B, T, ln, mk)
        dead = ~live[:, None, :, None].to(DEV).expand_as(k)
        kk, vv = k.masked_fill(dead, math.nan), v.masked_fill(dead, math.inf)
        got = _run(q, kk, vv, dout, ln, None if mk is None else mk.to(DEV))
        _compare(got, *_exact(q, k, v, live, 1 / math.sqrt(D), dout), dtype)
        assert not got[2][dead].any() and not got[3][dead].any()
        for b in range(B):
            assert live[b].any() or not (got[0][b].any() or got[1][b].any())
    again = _run(q, kk, vv, dout, None, mask.to(DEV), raster=True)
    assert all(torch.equal(x, y) for x, y in zip(got, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 128), (torch.bfloat16, 64), (torch.float16, 64)])
@pytest.mark.parametrize("top", [3.0, 12.0, 30.0])
def test_the_running_maximum_moves_many_times_in_a_piece(dtype, D, top):
    """Keys that grow along a piece of eleven steps of 64.  The accumulated row is moved when its maximum has risen by 8 in base 2: about 1 a step
    (top 3) and 4 (top 12) leave it behind and catch up, 9 (top 30) moves it at every step.  Keys that shrink after the first step, jump
    once, or come in waves.  The rows' statistics, and with them the gradients, follow."""
    B, H, L, T = 1, 40, 1024, 700
    assert _space(0, B, H, H, L, T, D, _lib.VSA_BF16) == 0 and B * H * -(-L // 256) > SMS
    q, k, v, dout = _inputs(B, H, H, L, T, D, dtype, 3)
    ramp = torch.linspace(0, top, T, device=DEV)
    for r in (ramp, ramp.flip(0), top * (ramp > 0.98 * top), top * torch.sin(ramp * 20 / top).abs()):
        kk = (k.float() * r[None, None, :, None]).to(dtype)
        got = _run(q, kk, v, dout)
        # sums where one term carries all: no averaging of the roundings of p and ds, and their cancellation in ds shows
        _compare(got, *_exact(q, kk, v, _live(B, T, None, None), 1 / math.sqrt(D), dout), dtype, slack=2.0)
