"""Backward of cross attention in fp16: gradients far from one, many keys, values of any size, against float64.

Softmax weights of many keys and their gradients are far below fp16's smallest normal number, 2^-14, where its steps are an absolute 2^-24;
what the results may be off is what their own rounding and the relative bound of the other tests allow."""

import ctypes
import math

import pytest
import torch

from simple_vsa_b200 import _lib, video_cross_attn
from tests.test_cross_attn import DEV, _bound, _exact, _inputs, _live, _run


def test_arguments_of_the_c_entry():
    a = _lib.Cross()
    assert _lib.Cross.PACK.size == ctypes.sizeof(a)
    a.B, a.H, a.Hkv, a.Lq, a.Lkv, a.D, a.dtype, a.scale = 1, 1, 1, 4, 4, 64, _lib.VSA_F16, 0.25
    for n in ("q", "k", "v", "dout", "out", "dq", "dk", "dv", "lse2", "delta", "workspace"):
        setattr(a, n, 1 << 20)
    assert _lib.lib.vsa_cross_bwd(a, None) == _lib.ERR_BAD_ARGUMENT and "bounds" in _lib.last_error()      # refused before any launch


def _check(got, want, names=("out", "dq", "dk", "dv")):
    for name, x, y, off in zip(names, got, want, want[4]):
        assert x.dtype == torch.float16
        x = x.detach().double().cpu()
        assert torch.isfinite(x).all(), name
        err = (x - y).norm().item()
        # a result below 2^-14 is rounded to the nearest multiple of 2^-24, off by 2^-25 at most
        allowed = _bound(torch.float16) * y.norm().item() + off + 2.0 ** -25 * math.sqrt(y.numel())
        assert err <= allowed, (name, err, y.norm().item(), allowed)


SHAPES = [  # B, H, Hk, L, T, D
    (1, 2, 1, 300, 512, 128), (2, 2, 2, 130, 1001, 64), (1, 2, 1, 300, 2048, 128), (1, 1, 1, 200, 2048, 72), (1, 2, 2, 200, 16384, 64),
    (1, 1, 1, 130, 65536, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 300.0])
@pytest.mark.parametrize("B,H,Hk,L,T,D", SHAPES)
def test_incoming_gradients_of_any_size(B, H, Hk, L, T, D, size):
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, torch.float16, T + D)
    dout = (dout.float() * size).half()
    _check(_run(q, k, v, dout), _exact(q, k, v, _live(B, T, None, None), 1 / math.sqrt(D), dout))


@pytest.mark.gpu
@pytest.mark.parametrize("values,size", [(1e-3, 1.0), (1e-3, 1000.0), (200.0, 1e-3), (200.0, 10.0), (1000.0, 1e-4)])
def test_values_of_any_size(values, size):
    """Peaked and flat rows: p (dp - delta) as large as the bound on it, and small beside it."""
    B, H, Hk, L, T, D = 1, 2, 1, 300, 700, 128
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, torch.float16, 31)
    q[:, :, ::2] *= 3
    v, dout = (v.float() * values).half(), (dout.float() * size).half()
    _check(_run(q, k, v, dout), _exact(q, k, v, _live(B, T, None, None), 1 / math.sqrt(D), dout))


@pytest.mark.gpu
def test_rows_and_samples_of_different_sizes():
    """Rows of the gradient 2^10 apart, a row of zeros, and samples that share nothing: each with lengths, with a mask, and with an
    encoder state outside them that is infinite."""
    B, H, Hk, L, T, D = 3, 2, 1, 260, 600, 64
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, torch.float16, 32)
    rows = 2.0 ** -(torch.arange(L, device=DEV) % 11).float()
    dout = (dout.float() * rows[None, None, :, None] * torch.tensor([1.0, 1e-3, 50.0], device=DEV).view(3, 1, 1, 1)).half()
    dout[:, :, 7] = 0
    lengths, mask = torch.tensor([T, 333, 0]), torch.rand(B, T, generator=torch.Generator().manual_seed(3)) < 0.5
    for ln, mk in ((lengths, None), (None, mask)):
        live = _live(B, T, ln, mk)
        kk, vv = k.clone(), v.clone()
        dead = ~live[:, None, :, None].to(DEV).expand_as(kk)
        kk[dead], vv[dead] = math.nan, math.inf
        got = _run(q, kk, vv, dout, ln, None if mk is None else mk.to(DEV))
        want = _exact(q, k, v, live, 1 / math.sqrt(D), dout)
        for b in range(B):                            # each sample by its own norms
            if not live[b].any():
                assert all(not x[b].any() for x in got)
                continue
            part = lambda x: x[b:b + 1]
            _check([part(x) for x in got], [*(part(x) for x in want[:4]), _exact(*(part(x) for x in (q, k, v)), part(live), 1 / math.sqrt(D), part(dout))[4]])
        assert not got[1][:, :, 7].any()
        assert all(torch.equal(x, y) for x, y in zip(got, _run(q, kk, vv, dout, ln, None if mk is None else mk.to(DEV))))
        # a row's dQ does not lose digits to larger rows: each row class by itself
        for c in range(11):
            x, y = got[1][0, :, c::11].double().cpu(), want[1][0, :, c::11]
            e = 2 * torch.finfo(torch.float16).eps * (want[0][0, :, c::11] * dout[0, :, c::11].double().cpu()).norm(dim=-1) / math.sqrt(D)
            assert (x - y).norm() <= 2 * _bound(torch.float16) * y.norm() + 8 * e.norm() + 2.0 ** -25 * math.sqrt(y.numel())


@pytest.mark.gpu
def test_more_key_heads_than_a_grid_has_rows():
    B, H, L, T, D = 700, 100, 9, 3, 8                   # 70,000 slices
    q, k, v, dout = _inputs(B, H, H, L, T, D, torch.float16, 33)
    dout = (dout.float() * 1e-3).half()
    got = _run(q, k, v, dout)
    p = torch.softmax(q.double() @ k.double().transpose(2, 3) / math.sqrt(D), dim=-1)
    o, dp = p @ v.double(), dout.double() @ v.double().transpose(2, 3)
    ds = p * (dp - (dout.double() * o).sum(-1, keepdim=True)) / math.sqrt(D)
    for x, y in zip(got, (o, ds @ k.double(), ds.transpose(2, 3) @ q.double(), p.transpose(2, 3) @ dout.double())):
        # delta from the rounded output: with three keys dP - delta is a third of dP and more, so that 2 u of delta are within another bound
        assert (x.double() - y).norm() <= 2 * _bound(torch.float16) * y.norm() + 2.0 ** -25 * math.sqrt(y.numel())


@pytest.mark.gpu
def test_captured_steps_and_side_streams():
    """Two captured steps replayed in turn on gradients of new sizes, and two calls at once on streams of their own: the norms are each
    call's."""
    steps = []
    for L, T in ((300, 200), (140, 3000)):
        q, k, v, dout = _inputs(2, 2, 1, L, T, 64, torch.float16, L)
        leaves = [x.requires_grad_() for x in (q, k, v)]

        def step(leaves=leaves, dout=dout):
            out = video_cross_attn(*leaves)
            return (out.detach(),) + torch.autograd.grad(out, leaves, dout)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        steps.append((graph, res, leaves, dout, step, side))
    for size in (1e-3, 100.0, 1e-4, 1.0):
        for graph, res, leaves, dout, _, _ in steps:
            with torch.no_grad():
                dout.copy_(torch.randn(dout.shape, device=DEV) * size)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(res, _run(*leaves, dout)))
    steps[0][3].mul_(1e-3)
    torch.cuda.synchronize()
    together = []
    for _, _, _, _, step, side in steps:
        with torch.cuda.stream(side):
            together.append(step())
    torch.cuda.synchronize()
    for got, (_, _, leaves, dout, _, _) in zip(together, steps):
        assert all(torch.equal(a, b) for a, b in zip(got, _run(*leaves, dout)))


@pytest.mark.gpu
def test_gradients_of_some_operands_only():
    q, k, v, dout = _inputs(2, 4, 2, 130, 900, 64, torch.float16, 35)
    dout = (dout.float() * 1e-3).half()
    want = _run(q, k, v, dout)[1:]
    for need in ((0,), (1,), (2,), (0, 2)):
        xs = [x.clone().requires_grad_(i in need) for i, x in enumerate((q, k, v))]
        got = torch.autograd.grad(video_cross_attn(*xs), [xs[i] for i in need], dout)
        assert all(torch.equal(g, want[i]) for g, i in zip(got, need))


@pytest.mark.gpu
def test_scores_of_many_thousands():
    """Exponents whose fp32 steps are no longer small beside one: weights may be off by a factor, and stay finite on their way through fp16."""
    q, k, v, dout = _inputs(1, 2, 1, 130, 300, 128, torch.float16, 36)
    for size in (100.0, 1000.0, 4000.0):
        got = _run((q.float() * size).half(), (k.float() * size).half(), v, dout)
        assert all(torch.isfinite(x).all() for x in (got[0], got[3]))
        # At the largest size scores are 1.6e7 apart and more, one key has a row's weight, and exponents of 2^25 and more have steps of 4 and
        # more: the statistic's rounding makes that weight any power of two.  It is held up to 65504 / 2^14 < 4, so that what the values'
        # gradient sums to over the keys is at most four times dout's.
        assert (got[3].double().sum((1, 2)).abs() <= 4 * dout.double().abs().sum((1, 2)) + 1).all()
