"""Rotary positions: the table, the rotation of q and k, and the rotation on the way into tile order, against float64."""

import math

import pytest
import torch

import simple_vsa_b200 as V
from simple_vsa_b200 import ops

DEV = "cuda:0"


# ---- host side ------------------------------------------------------------------------------------------------------
def _angle(pos, pair, dims, theta=10000.0):
    return pos * theta ** (-2.0 * pair / dims)


def test_table_of_a_token_grid():
    T, H, W, R = 3, 4, 5, 16
    meta = V.build_rotary_metadata((T, H, W), R)
    assert meta["cos"].shape == meta["sin"].shape == (T * H * W, R // 2) and meta["interleaved"] is True
    dims = [8, 4, 4]                                       # 8 pairs: the first axis takes what the equal shares leave
    for t, h, w in ((0, 0, 0), (2, 3, 4), (1, 0, 3)):
        row = (t * H + h) * W + w
        want = [_angle(p, i, d) for p, d in zip((t, h, w), dims) for i in range(d // 2)]
        for col, a in enumerate(want):
            assert abs(meta["cos"][row, col].item() - math.cos(a)) <= 2.0 ** -24
            assert abs(meta["sin"][row, col].item() - math.sin(a)) <= 2.0 ** -24
    text = V.build_rotary_metadata((7,), 6, interleaved=False, theta=500.0)
    assert text["cos"].shape == (7, 3) and text["interleaved"] is False
    assert abs(text["sin"][6, 2].item() - math.sin(_angle(6, 2, 6, 500.0))) <= 2.0 ** -24
    own = V.build_rotary_metadata((2, 3, 4), 16, axes_dims=(0, 10, 6))
    assert abs(own["cos"][1 * 12 + 2 * 4 + 3, 5].item() - math.cos(_angle(3, 0, 6))) <= 2.0 ** -24


def test_far_positions_keep_their_angle():
    n = 3_000_001
    meta = V.build_rotary_metadata((n,), 4)
    for pos in (n - 1, 2_000_003):
        assert abs(meta["sin"][pos, 0].item() - math.sin(pos)) <= 2.0 ** -24        # 32-bit angles would be off by 0.1


def test_scaled_tables():
    R, f = 8, 4.0
    plain = V.build_rotary_metadata((64,), R)
    linear = V.build_rotary_metadata((64,), R, scaling={"kind": "linear", "factor": f})
    torch.testing.assert_close(linear["cos"][40], plain["cos"][10], atol=2.0 ** -23, rtol=0)
    ntk = V.build_rotary_metadata((64,), R, scaling={"kind": "ntk", "factor": f})
    assert ntk["sin"][63, 0] == plain["sin"][63, 0]                                  # the fastest pair stays
    assert abs(ntk["sin"][60, 3].item() - math.sin(60 * 10000.0 ** (-6 / 8) / f)) <= 2.0 ** -23      # the slowest: / f
    yarn = V.build_rotary_metadata((64,), R, scaling={"kind": "yarn", "factor": f, "original_length": 400})
    amp = 1.0 + 0.1 * math.log(f)
    for i in range(R // 2):
        freq = 10000.0 ** (-2 * i / R)
        keep = min(1.0, max(0.0, (400 * freq / (2 * math.pi) - 1.0) / 31.0))
        a = 50 * (freq * keep + freq / f * (1 - keep))
        assert abs(yarn["cos"][50, i].item() - amp * math.cos(a)) <= 2.0 ** -22
    mixed = V.build_rotary_metadata((4, 4), R, scaling=[None, {"kind": "linear", "factor": 2.0}])
    assert abs(mixed["sin"][3 * 4 + 2, 2].item() - math.sin(1.0)) <= 2.0 ** -24
    assert abs(mixed["sin"][3 * 4 + 2, 0].item() - math.sin(3.0)) <= 2.0 ** -24


@pytest.mark.parametrize("kwargs,match", [
    (dict(rotary_dim=7), "even"), (dict(rotary_dim=0), "even"), (dict(axes_dims=(4, 4)), "axes_dims"),
    (dict(axes_dims=(3, 3, 2)), "axes_dims"), (dict(axes_dims=(4, 4, 4)), "axes_dims"), (dict(theta=0.0), "theta"),
    (dict(scaling={"kind": "cubic", "factor": 2.0}), "kind"), (dict(scaling={"kind": "linear", "factor": 0.0}), "factor"),
    (dict(scaling={"kind": "yarn", "factor": 2.0}), "original_length"), (dict(scaling=[None]), "axes"),
    (dict(scaling={"kind": "yarn", "factor": 2.0, "original_length": 9, "beta_fast": 1.0}), "beta_fast")])
def test_table_refusals(kwargs, match):
    with pytest.raises(ValueError, match=match):
        V.build_rotary_metadata((2, 3, 4), **{"rotary_dim": 8, **kwargs})
    with pytest.raises(ValueError, match="dit_seq_shape"):
        V.build_rotary_metadata((), 8)


def test_entry_point_refusals_without_a_gpu():
    import simple_vsa_b200._lib as L
    x, rot = torch.zeros(1, 2, 6, 8), V.build_rotary_metadata((6,), 8)
    with pytest.raises(ValueError, match="requires CUDA tensors"):
        V.video_rotary(x, x, rot)
    with pytest.raises(ValueError, match="shape"):
        V.video_rotary_raster(x[0], None, rot)
    with pytest.raises(ValueError, match="requires CUDA tensors"):
        V.tile_heads(x.transpose(1, 2), V.build_vsa_metadata((1, 2, 3), (1, 2, 2)), rot)
    a = L.Rotary()
    a.B, a.rows, a.D, a.rotary_dim, a.dtype = 1, 4, 8, 6, L.VSA_BF16
    a.heads[0] = 1
    for change, rc, match in ((dict(rotary_dim=5), L.ERR_BAD_ARGUMENT, "even"), (dict(rotary_dim=10), L.ERR_BAD_ARGUMENT, "head dim"),
                              (dict(dtype=9), L.ERR_UNSUPPORTED, "dtype"), (dict(rows=-1), L.ERR_BAD_ARGUMENT, "negative"),
                              (dict(), L.ERR_BAD_ARGUMENT, "null")):
        old = {n: getattr(a, n) for n in change}
        for n, v in change.items():
            setattr(a, n, v)
        assert L.lib.vsa_rotary(a, None) == rc and match in L.last_error()
        for n, v in old.items():
            setattr(a, n, v)
    assert L.lib.vsa_rotary(None, None) == L.ERR_BAD_ARGUMENT


# ---- device side ------------------------------------------------------------------------------------------------------
def _turn64(x, cos, sin, interleaved, sign=1.0):
    """``x`` in float64 turned, and the sum of magnitudes each value is made of."""
    x, p = x.double().cpu(), cos.shape[-1]
    first = torch.arange(p) * 2 if interleaved else torch.arange(p)
    second = first + 1 if interleaved else first + p
    a, b = x[..., first], x[..., second]
    y, size = x.clone(), x.abs()
    y[..., first], y[..., second] = a * cos - sign * b * sin, b * cos + sign * a * sin
    size[..., first] = size[..., second] = (a.abs() + b.abs()) * (cos.abs() + sin.abs())
    return y, size


def _check(got, want, size):
    """Half a step of the type for the one rounding, and three fp32 roundings (2^-24 each) of the two products."""
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).smallest_normal * eps          # a step among the subnormals
    tol = eps / 2 * want.abs() * 1.01 + 2.0 ** -22 * size + tiny
    off = (got.detach().double().cpu() - want).abs()
    assert bool((off <= tol).all()), (off - tol).max()


CASES = [  # dtype, B, H, Hk, L, D, R, interleaved, raster, positions
    (torch.bfloat16, 2, 3, 1, 37, 128, 128, True, False, None),
    (torch.float16, 2, 3, 3, 37, 128, 64, True, True, "batch"),
    (torch.float32, 1, 5, 2, 33, 64, 64, True, False, "shared"),
    (torch.bfloat16, 1, 2, 2, 130, 128, 128, False, True, None),           # pieces of 16 bytes
    (torch.float16, 3, 4, 2, 21, 64, 44, False, False, "batch"),           # halves of 22: two at a time
    (torch.float32, 2, 2, 1, 9, 72, 42, False, False, None),               # halves of 21: one at a time
    (torch.bfloat16, 2, 2, 1, 9, 72, 42, False, True, None),
    (torch.bfloat16, 2, 3, 1, 11, 70, 22, False, False, "batch"),          # rows off the 16-byte grid: element by element
    (torch.float16, 2, 3, 1, 11, 71, 70, True, True, None),
    (torch.float32, 1, 1, 1, 5, 3, 2, False, False, None),
    (torch.bfloat16, 8, 40, 8, 1, 128, 128, False, False, "batch"),        # single tokens
    (torch.float16, 1, 1, 1, 1, 256, 256, True, True, None),
    (torch.bfloat16, 1, 2, 2, 4097, 256, 130, False, False, None),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,B,H,Hk,L,D,R,interleaved,raster,positions", CASES)
def test_rotation_and_gradient_match_float64(dtype, B, H, Hk, L, D, R, interleaved, raster, positions):
    g = torch.Generator().manual_seed(L + D + R)
    rows = L + 50
    rot = V.build_rotary_metadata((rows,), R, interleaved=interleaved, device=DEV)
    shape = lambda h: (B, L, h, D) if raster else (B, h, L, D)
    q, k, wq, wk = (torch.randn(shape(h), generator=g).to(dtype).to(DEV) for h in (H, Hk, H, Hk))
    pos = None
    if positions:
        pos = torch.randint(0, rows, (B, L) if positions == "batch" else (L,), generator=g)
    at = pos if pos is not None else torch.arange(L)
    cos, sin = (rot[n].double().cpu()[at] for n in ("cos", "sin"))
    cos, sin = (x.expand(B, L, R // 2).unsqueeze(2 if raster else 1) for x in (cos, sin))
    leaves = [q.requires_grad_(), k.requires_grad_()]
    f = V.video_rotary_raster if raster else V.video_rotary
    outs = f(*leaves, rot, positions=None if pos is None else pos.to(DEV))
    grads = torch.autograd.grad(outs, leaves, (wq, wk))
    for x, y, w, dx in zip(leaves, outs, (wq, wk), grads):
        assert y.shape == x.shape and y.dtype == dtype
        _check(y, *_turn64(x.detach(), cos, sin, interleaved))
        _check(dx, *_turn64(w, cos, sin, interleaved, -1.0))
    # q alone, and int64 / host positions, give the same bits
    alone = f(q.detach(), None, rot, positions=pos)
    assert torch.equal(alone, outs[0])


@pytest.mark.gpu
def test_gradient_against_differences():
    g = torch.Generator().manual_seed(1)
    rot = V.build_rotary_metadata((6,), 10, scaling={"kind": "yarn", "factor": 4.0, "original_length": 50}, interleaved=False)
    x, w = (torch.randn(1, 2, 6, 12, generator=g).to(DEV) for _ in range(2))
    leaf = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad((V.video_rotary(leaf, None, rot).double() * w.double()).sum(), leaf)
    for at in ((0, 0, 3, 2), (0, 1, 5, 9), (0, 1, 0, 11), (0, 0, 4, 7)):
        h = torch.zeros_like(x)
        h[at] = 0.5                                    # the operator is linear: any step gives the derivative
        diff = ((V.video_rotary(x + h, None, rot).double() - V.video_rotary(x - h, None, rot).double()) * w.double()).sum()
        # two outputs of magnitude <= 5 with four fp32 roundings each, two affected values, weights <= 4
        assert abs(diff.item() - dx[at].item()) <= 2 * 2 * 4 * 5 * 4 * 2.0 ** -24


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_positions_outside_the_table_leave_the_token_as_it_is(dtype, interleaved):
    g = torch.Generator().manual_seed(2)
    rot = V.build_rotary_metadata((5,), 16, interleaved=interleaved, device=DEV)
    q = torch.randn(1, 2, 4, 24, generator=g).to(dtype).to(DEV)
    pos = torch.tensor([-1, 5, 2 ** 40 + 1, 1])
    out = V.video_rotary(q, None, rot, positions=pos)
    assert torch.equal(out[:, :, :3], q[:, :, :3])
    assert torch.equal(out[:, :, 3, 16:], q[:, :, 3, 16:]) and not torch.equal(out[:, :, 3, :16], q[:, :, 3, :16])


@pytest.mark.gpu
@pytest.mark.parametrize("interleaved", [True, False])
def test_dims_that_do_not_turn_are_copied_beside_infinities(interleaved):
    """An infinity or NaN in the copied part, or in another pair, reaches no other value."""
    rot = V.build_rotary_metadata((3,), 4, interleaved=interleaved, device=DEV)
    q = torch.ones(1, 1, 3, 8, device=DEV, dtype=torch.bfloat16)
    q[0, 0, 1, 4:] = torch.tensor([math.inf, math.nan, -math.inf, 7.0])
    q[0, 0, 2, 0] = math.inf
    out = V.video_rotary(q, None, rot)[0, 0].float().cpu()
    assert out[1, 4] == math.inf and math.isnan(out[1, 5]) and out[1, 6] == -math.inf and out[1, 7] == 7
    assert torch.isfinite(out[1, :4]).all() and torch.isfinite(out[0]).all()
    pair = [0, 1] if interleaved else [0, 2]
    rest = [i for i in range(8) if i not in pair]
    assert not torch.isfinite(out[2, pair]).any() and torch.isfinite(out[2, rest]).all()


@pytest.mark.gpu
def test_strided_operands_and_gradients():
    """Slices of one projection, transposed views, an expanded gradient, and rows that start off the 16-byte grid."""
    g = torch.Generator().manual_seed(3)
    B, S, H, D = 2, 19, 3, 64
    rot = V.build_rotary_metadata((S,), 32, device=DEV)
    qkv = torch.randn(B, S, 3 * H, D, generator=g).to(torch.bfloat16).to(DEV)
    want = V.video_rotary(*(qkv[:, :, i * H:(i + 1) * H].transpose(1, 2).contiguous() for i in range(2)), rot)
    got = V.video_rotary_raster(qkv[:, :, :H], qkv[:, :, H:2 * H], rot)
    for a, b in zip(got, want):
        assert torch.equal(a.transpose(1, 2), b)
    odd = torch.randn(B * S * H * (D + 3) + 1, generator=g).to(torch.bfloat16).to(DEV)[1:].view(B, H, S, D + 3)[..., 2:D + 2]
    assert torch.equal(V.video_rotary(odd, None, rot), V.video_rotary(odd.contiguous(), None, rot))
    leaf = qkv[:, :, :H].transpose(1, 2).detach().requires_grad_()
    one = torch.ones((), device=DEV, dtype=torch.bfloat16).expand(B, H, S, D)
    (dx,) = torch.autograd.grad(V.video_rotary(leaf, None, rot), leaf, one)
    (dy,) = torch.autograd.grad(V.video_rotary(leaf, None, rot), leaf, one.contiguous())
    assert torch.equal(dx, dy)
    swapped = qkv.permute(0, 3, 2, 1)[:, :32]              # head dim not contiguous: copied first
    assert torch.equal(V.video_rotary(swapped, None, V.build_rotary_metadata((3 * H,), 10)),
                       V.video_rotary(swapped.contiguous(), None, V.build_rotary_metadata((3 * H,), 10)))


def test_outputs_keep_a_contiguous_head_dim():
    """Windows of a longer row have two dims of stride 1; what is made like them is indexed with a contiguous head dim."""
    for n in (5, 64, 137):
        x = torch.zeros(2, 3, n + 63).unfold(-1, 64, 1)
        y = ops._like(x)
        assert y.shape == x.shape and y.stride(3) == 1 and ops._like(x.transpose(1, 2)).stride(3) == 1
    x = torch.zeros(2, 9, 3, 64).transpose(1, 2)
    assert ops._like(x).stride() == x.stride()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [True, False])
def test_windows_of_a_longer_row(dtype, interleaved):
    g = torch.Generator().manual_seed(12)
    rot = V.build_rotary_metadata((5,), 32, device=DEV, interleaved=interleaved)
    x = torch.randn(2, 3, 68, generator=g).to(dtype).to(DEV).unfold(-1, 64, 1)
    want = V.video_rotary(x.contiguous(), None, rot)
    assert torch.equal(V.video_rotary(x, None, rot), want)
    assert torch.equal(V.video_rotary_raster(x.transpose(1, 2), None, rot), want.transpose(1, 2))
    leaf = torch.zeros(2, 3, 5, 64, device=DEV, dtype=dtype, requires_grad=True)
    (dx,) = torch.autograd.grad(V.video_rotary(leaf, None, rot), leaf, x)
    (dy,) = torch.autograd.grad(V.video_rotary(leaf, None, rot), leaf, x.contiguous())
    assert torch.equal(dx, dy)


@pytest.mark.gpu
def test_only_one_gradient_and_empty_tensors():
    g = torch.Generator().manual_seed(4)
    rot = V.build_rotary_metadata((8,), 16, device=DEV)
    q, k = (torch.randn(1, 2, 8, 16, generator=g).to(DEV).requires_grad_() for _ in range(2))
    yq, yk = V.video_rotary(q, k, rot)
    dq, dk = torch.autograd.grad(yk.sum(), (q, k), allow_unused=True)
    assert dk is not None and (dq is None or not dq.any())
    for shape in ((0, 2, 8, 16), (1, 0, 8, 16), (1, 2, 0, 16)):
        e = torch.empty(shape, device=DEV, requires_grad=True)
        out = V.video_rotary(e, None, rot)
        out.sum().backward()
        assert out.shape == e.grad.shape == e.shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,R,interleaved,tile", [(torch.bfloat16, 128, 128, True, (4, 4, 4)), (torch.float16, 64, 44, False, (4, 4, 4)),
                                                        (torch.float32, 24, 16, False, (2, 2, 4))])
def test_tile_heads_turns_on_the_way(dtype, D, R, interleaved, tile):
    g = torch.Generator().manual_seed(5)
    grid, B, H = (3, 5, 6), 2, 3
    meta = V.build_vsa_metadata(grid, tile, device=DEV)
    rot = V.build_rotary_metadata(grid, R, interleaved=interleaved, device=DEV)
    x = torch.randn(B, 90, H, D, generator=g).to(dtype).to(DEV).requires_grad_()
    got = V.tile_heads(x, meta, rot)
    # the same bits as turning first, or as tiling first with the tile map as positions
    assert torch.equal(got, V.tile_heads(V.video_rotary_raster(x.detach(), None, rot), meta))
    assert torch.equal(got, V.video_rotary(V.tile_heads(x.detach(), meta), None, rot, positions=meta["tile_map"]))
    assert not got[:, :, meta["tile_map"] < 0].any()
    w = torch.randn(got.shape, generator=g).to(dtype).to(DEV)
    (dx,) = torch.autograd.grad(got, x, w)
    cos, sin = (rot[n].double().cpu()[None, :, None] for n in ("cos", "sin"))
    _check(dx, *_turn64(V.untile_heads(w, meta), cos, sin, interleaved, -1.0))


@pytest.mark.gpu
@pytest.mark.parametrize("D,topk", [(128, 3), (64, 2)])
def test_raster_operator_with_rotary_is_the_operator_on_turned_activations(D, topk):
    """Both forms (raster-order kernels at head dim 128, separate layout passes at 64): output bit for bit, gradients up to the one
    rounding more that the separate form has no counterpart of, and the order of the sums in dK and dV."""
    g = torch.Generator().manual_seed(6)
    grid, B, H, dtype = (5, 6, 7), 1, 2, torch.bfloat16
    S = 5 * 6 * 7
    meta, rot = V.build_vsa_metadata(grid, (4, 4, 4), device=DEV), V.build_rotary_metadata(grid, D, device=DEV)
    q, k, v, dout = (torch.randn(B, S, H, D, generator=g).to(dtype).to(DEV) for _ in range(4))
    a, b = ([x.clone().requires_grad_() for x in (q, k, v)] for _ in range(2))
    out_a = V.video_sparse_attn_raster(*a, meta, topk, rotary=rot)
    tq, tk = V.video_rotary_raster(b[0], b[1], rot)
    out_b = V.video_sparse_attn_raster(tq, tk, b[2], meta, topk)
    assert torch.equal(out_a, out_b)
    ga, gb = torch.autograd.grad(out_a, a, dout), torch.autograd.grad(out_b, b, dout)
    assert torch.equal(ga[0], gb[0])
    for x, y in zip(ga[1:], gb[1:]):
        torch.testing.assert_close(x.float(), y.float(), atol=2e-2, rtol=2e-2)
    with torch.no_grad():
        assert torch.equal(V.video_sparse_attn_raster(q, k, v, meta, topk, rotary=rot), out_a)
    assert V._lib.device_status() == 0


@pytest.mark.gpu
def test_refusals_on_the_device():
    rot = V.build_rotary_metadata((6,), 8, device=DEV)
    x = torch.zeros(1, 2, 6, 8, device=DEV)
    for bad, match in ((dict(k=torch.zeros(1, 2, 5, 8, device=DEV)), "share"), (dict(k=x.half()), "dtype"),
                       (dict(rotary=V.build_rotary_metadata((5,), 8)), "positions"), (dict(rotary=V.build_rotary_metadata((6,), 10)), "dims of a head"),
                       (dict(positions=torch.zeros(5, dtype=torch.int32)), "positions must have shape"), (dict(positions=torch.zeros(6)), "integers"),
                       (dict(rotary={**rot, "sin": rot["sin"][:3]}), "share the shape"),
                       (dict(rotary={**rot, "sin": rot["sin"].clone().requires_grad_()}), "constant")):
        args = dict(k=None, rotary=rot, positions=None)
        args.update(bad)
        with pytest.raises(ValueError, match=match):
            V.video_rotary(x, args["k"], args["rotary"], positions=args["positions"])
    with pytest.raises(ValueError, match="float"):
        V.video_rotary(x.double(), None, rot)
    with pytest.raises(ValueError, match="256"):
        V.video_rotary(torch.zeros(1, 1, 6, 264, device=DEV), None, rot)
    meta = V.build_vsa_metadata((1, 2, 3), (1, 2, 2), device=DEV)
    with pytest.raises(ValueError, match="grid"):
        V.tile_heads(x.transpose(1, 2), meta, V.build_rotary_metadata((7,), 8))
    with pytest.raises(ValueError, match="tokens"):
        V.tile_heads(x.transpose(1, 2)[:, :5], meta, rot)


@pytest.mark.gpu
def test_side_stream_and_captured_step():
    g = torch.Generator().manual_seed(7)
    rot = V.build_rotary_metadata((64,), 32, device=DEV)
    q, k, w = (torch.randn(1, 2, 64, 32, generator=g).to(torch.bfloat16).to(DEV) for _ in range(3))
    want = V.video_rotary(q, k, rot)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = V.video_rotary(q, k, rot)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    sq, sk = (x.clone().requires_grad_() for x in (q, k))

    def step():
        yq, yk = V.video_rotary(sq, sk, rot)
        return (yq.detach(), yk.detach()) + torch.autograd.grad((yq, yk), (sq, sk), (w, w))

    with torch.cuda.stream(s):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step()
    with torch.no_grad():
        sq.copy_(k)
        sk.copy_(q)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(res[0], V.video_rotary(k, None, rot)) and torch.equal(res[1], V.video_rotary(q, None, rot))


@pytest.mark.gpu
def test_a_table_or_positions_changed_before_the_backward_are_refused():
    rot = V.build_rotary_metadata((6,), 8, device=DEV)
    for change in ("cos", "positions"):
        table = {**rot, "cos": rot["cos"].clone()}
        pos = torch.arange(6, device=DEV, dtype=torch.int32)
        q = torch.randn(1, 2, 6, 8, device=DEV, requires_grad=True)
        out = V.video_rotary(q, None, table, positions=pos)
        (table["cos"] if change == "cos" else pos).add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()
