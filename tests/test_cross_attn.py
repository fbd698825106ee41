"""Cross attention to an encoder's states, against float64: lengths from zero, masks, shared heads, strides, every kernel family."""

import math

import pytest
import torch

import simple_vsa_b200 as V
from simple_vsa_b200 import _lib, ops

DEV = "cuda:0"


# ---- host side ------------------------------------------------------------------------------------------------------
def test_refusals_without_a_gpu():
    q, k = torch.zeros(2, 4, 10, 16), torch.zeros(2, 2, 7, 16)
    for bad, match in ((dict(q=q[0]), "shape"), (dict(k=k[:1], v=k[:1]), "batch"), (dict(v=k[:, :, :6]), "same heads and sequence"),
                       (dict(v=k[:, :1]), "same heads and sequence"), (dict(k=q[:, :3], v=q[:, :3]), "multiple"),
                       (dict(k=k[..., :8], v=k[..., :8]), "head dimension"), (dict(), "requires CUDA tensors")):
        args = dict(q=q, k=k, v=k)
        args.update(bad)
        with pytest.raises(ValueError, match=match):
            V.video_cross_attn(args["q"], args["k"], args["v"])
    with pytest.raises(ValueError, match="1 to 256"):
        V.video_cross_attn(torch.zeros(1, 1, 2, 257), torch.zeros(1, 1, 2, 257), torch.zeros(1, 1, 2, 257))
    with pytest.raises(ValueError, match="head_dim"):
        V.video_cross_attn_raster(q[0], k, k)


def test_c_entry_refusals_and_sizes():
    a = _lib.Cross()
    a.B, a.H, a.Hkv, a.Lq, a.Lkv, a.D, a.dtype, a.scale = 2, 4, 2, 10, 7, 16, _lib.VSA_BF16, 0.25
    for name, value, rc, match in (("Hkv", 3, _lib.ERR_BAD_ARGUMENT, "multiple"), ("Lq", -1, _lib.ERR_BAD_ARGUMENT, "negative"),
                                   ("D", 0, _lib.ERR_BAD_ARGUMENT, "negative"), ("D", 300, _lib.ERR_UNSUPPORTED, "256"),
                                   ("dtype", 5, _lib.ERR_UNSUPPORTED, "dtype"), ("B", 70000, _lib.ERR_UNSUPPORTED, "65535"),
                                   ("scale", 0.5, _lib.ERR_BAD_ARGUMENT, "null")):
        old = getattr(a, name)
        setattr(a, name, value)
        for f in (_lib.lib.vsa_cross_fwd, _lib.lib.vsa_cross_bwd):
            assert f(a, None) == rc and match in _lib.last_error(), (name, _lib.last_error())
        setattr(a, name, old)
    assert _lib.lib.vsa_cross_fwd(None, None) == _lib.ERR_BAD_ARGUMENT
    assert [_lib.lib.vsa_cross_words(n) for n in (-1, 0, 1, 128, 129)] == [-1, 0, 4, 4, 8]
    assert _lib.lib.vsa_cross_workspace_bytes(0, 2, 4, 3, 10, 7, 16, _lib.VSA_BF16, 0) == -1
    assert _lib.lib.vsa_cross_workspace_bytes(1, 2, 4, 2, 10, 7, 16, 9, 0) == -1
    assert _lib.lib.vsa_cross_workspace_bytes(0, 0, 4, 2, 10, 7, 16, _lib.VSA_F32, 0) == 0
    # many rows: nothing is split; a row each against long states: the keys are, and the parts fit what is asked for
    assert _lib.lib.vsa_cross_workspace_bytes(0, 2, 40, 40, 92160, 512, 128, _lib.VSA_BF16, 0) == 0
    n = _lib.lib.vsa_cross_workspace_bytes(0, 1, 2, 2, 1, 8192, 128, _lib.VSA_BF16, 0)
    assert n > 0 and n % (2 * (128 + 1) * 4) == 0
    n = _lib.lib.vsa_cross_workspace_bytes(1, 1, 2, 2, 40000, 77, 64, _lib.VSA_F16, 0)
    assert n > 0 and n % (2 * 2 * 77 * 64 * 4) == 0


# ---- device side ------------------------------------------------------------------------------------------------------
def _exact(q, k, v, live, scale, dout):
    """float64 on the CPU: output and gradients, keys that take no part left out of every sum; and what dq and dk may be off, in
    the 2-norm, because delta_i = out_i . dout_i is formed from the ROUNDED output: ds_ij is p_ij (dp_ij - delta_i), and where the
    two nearly cancel (one key: they are equal) an error e_i of delta is not small beside the result.  Each of the D terms of
    delta_i is off by at most u = eps / 2 of itself, with random signs: e_i <= 2 u |out_i * dout_i| (2-norm of the products; 2^-18 in
    fp32, where the two sums of D products differ by their order).  It moves dq_i by scale e_i (sum_j p_ij k_j) and dk_j by
    scale sum_i e_i p_ij q_i, whose terms have random signs too (factor 2 for their spread)."""
    B, H, L, D = q.shape
    G = H // max(1, k.shape[1])
    e = max(2 * torch.finfo(q.dtype).eps / 2, 2.0 ** -18)
    off = [0.0, 0.0, 0.0, 0.0]
    q, k, v, dout = (x.detach().double().cpu() for x in (q, k, v, dout))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        at = live[b].nonzero().flatten()
        if at.numel() == 0:
            continue
        for h in range(H):
            kk, vv = k[b, h // G, at], v[b, h // G, at]
            p = torch.softmax(q[b, h] @ kk.T * scale, dim=-1)
            o = p @ vv
            ds = p * (dout[b, h] @ vv.T - (dout[b, h] * o).sum(-1, keepdim=True)) * scale
            out[b, h], dq[b, h] = o, ds @ kk
            dk[b, h // G, at] += ds.T @ q[b, h]
            dv[b, h // G, at] += p.T @ dout[b, h]
            ei = e * (o * dout[b, h]).norm(dim=-1) * abs(scale)
            off[1] += (ei * (p @ kk).norm(dim=-1)).square().sum().item()
            off[2] += 4 * (p.square().T @ (ei * q[b, h].norm(dim=-1)).square()).sum().item()
    return out, dq, dk, dv, [x ** 0.5 for x in off]


def _bound(dtype):
    """2-norm of the error over that of the result.  16-bit: the result is rounded (half a step, u = eps / 2, 0.58 u in the root
    mean square) and so are p and ds on their way into the second product, one rounding per term each, whose errors add up like
    random signs: at most u of the terms' 2-norm, and the gradients' sums cancel no more than by a factor two for these
    inputs.  Together below 4 u.  fp32: scores of magnitude up to 2^4 rounded to 2^-20 in the exponent, sums of up to some
    thousand terms in pieces: 2^-18."""
    return 2.0 ** -18 if dtype == torch.float32 else 4 * torch.finfo(dtype).eps / 2


def _inputs(B, H, Hk, L, T, D, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda h, n: torch.randn(B, h, n, D, generator=g).to(dtype).to(DEV)
    return make(H, L), make(Hk, T), make(Hk, T), make(H, L)


def _compare(got, want, dtype, names=("out", "dq", "dk", "dv"), slack=1.0):
    for name, x, y, off in zip(names, got, want, want[4]):
        x = x.detach().double().cpu()
        assert torch.isfinite(x).all(), name
        err = (x - y).norm().item()
        assert err <= slack * _bound(dtype) * y.norm().item() + off, (name, err, y.norm().item(), off)


def _run(q, k, v, dout, lengths=None, mask=None, scale=None, f=None):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = (f or V.video_cross_attn)(*leaves, lengths, kv_mask=mask, sm_scale=scale)
    grads = torch.autograd.grad(out, leaves, dout)
    assert _lib.device_status() == 0
    return (out.detach(),) + grads


def _live(B, T, lengths, mask):
    live = torch.ones(B, T, dtype=torch.bool)
    if lengths is not None:
        live &= torch.arange(T)[None] < lengths.cpu()[:, None]
    return live & mask.cpu() if mask is not None else live


SHAPES = [  # B, H, Hk, L, T, D
    (1, 1, 1, 1, 1, 128), (2, 3, 3, 1, 300, 64), (2, 2, 1, 5, 127, 128), (1, 2, 2, 128, 128, 128), (2, 6, 2, 129, 129, 64),
    (1, 3, 1, 257, 77, 128), (1, 2, 2, 640, 512, 128), (3, 2, 2, 300, 1001, 64), (1, 4, 2, 511, 260, 72), (1, 2, 2, 100, 90, 8),
    (2, 2, 1, 70, 200, 120), (1, 1, 1, 2000, 33, 96),
]
ODD = [(1, 2, 1, 67, 70, 20), (2, 2, 2, 33, 65, 200), (1, 1, 1, 130, 100, 256), (1, 2, 2, 40, 50, 1), (1, 1, 1, 65, 64, 133)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,Hk,L,T,D", SHAPES + ODD)
def test_output_and_gradients_match_float64(dtype, B, H, Hk, L, T, D):
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, dtype, L + T + D)
    got = _run(q, k, v, dout)
    _compare(got, _exact(q, k, v, _live(B, T, None, None), 1 / math.sqrt(D), dout), dtype)
    with torch.no_grad():
        assert torch.equal(V.video_cross_attn(q, k, v), got[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,H,Hk,L,T,D", [(3, 2, 2, 1, 1, 64), (3, 2, 1, 1, 255, 128), (3, 4, 1, 1, 257, 72), (3, 4, 2, 2, 5000, 128),
                                          (3, 4, 1, 2, 700, 64), (3, 3, 1, 3, 130, 128), (3, 160, 160, 1, 500, 128), (3, 5, 5, 7, 40, 8)])
def test_few_rows(dtype, B, H, Hk, L, T, D):
    """Up to eight and just above eight rows a key head, keys cut into parts or not, with lengths and a mask, and a sample without
    keys; the gradient of such a call."""
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, dtype, T + H)
    g = torch.Generator().manual_seed(T)
    mask = torch.rand(B, T, generator=g) < 0.7
    mask[0] = True
    mask[2] = False
    for ln, mk in ((None, None), (torch.tensor([T, max(1, T // 3), 0]), None), (None, mask), (torch.tensor([T // 2, T, T]), mask)):
        live = _live(B, T, ln, mk)
        kk, vv = k.clone(), v.clone()
        dead = ~live[:, None, :, None].to(DEV).expand_as(kk)
        kk[dead], vv[dead] = math.nan, math.nan
        got = _run(q, kk, vv, dout, ln, None if mk is None else mk.to(DEV))
        _compare(got, _exact(q, k, v, live, 1 / math.sqrt(D), dout), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,D", [(300, 128), (512, 64), (129, 72), (1, 64), (70, 20)])
def test_lengths_and_masks(dtype, T, D):
    """Prompts of zero, one, full and odd lengths; masks with holes, whole tiles and whole samples gone; both together.  What stands
    in keys that take no part is NaN and infinite, and reaches nothing; their gradients are zero."""
    B, H, Hk, L = 5, 2, 1, 200
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, dtype, T + D)
    g = torch.Generator().manual_seed(9)
    lengths = torch.tensor([0, 1, T, max(1, T - 37), T + 50])
    mask = torch.rand(B, T, generator=g) < 0.6
    mask[1] = False
    mask[2, :min(T, 200)] = False
    mask[3] = True
    for ln, mk in ((lengths, None), (None, mask), (lengths, mask)):
        live = _live(B, T, ln, mk)
        kk, vv = k.clone(), v.clone()
        dead = ~live[:, None, :, None].to(DEV).expand_as(kk)
        kk[dead], vv[dead] = math.nan, math.inf
        got = _run(q, kk, vv, dout, None if ln is None else ln.to(DEV), None if mk is None else mk.to(DEV))
        want = _exact(q, k, v, live, 1 / math.sqrt(D), dout)
        _compare(got, want, dtype)
        assert not got[2][dead].any() and not got[3][dead].any()
        for b in range(B):
            if not live[b].any():
                assert not got[0][b].any() and not got[1][b].any()
    # lengths on the host, as int32 / int64, and the mask that says the same give the same bits
    live = _live(B, T, lengths, None)
    a = V.video_cross_attn(q, k, v, lengths)
    assert torch.equal(a, V.video_cross_attn(q, k, v, lengths.to(DEV).int()))
    assert torch.equal(a, V.video_cross_attn(q, k, v, kv_mask=live.to(DEV)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64), (torch.float16, 36)])
def test_scores_that_grow_and_shrink_along_the_keys(dtype, D):
    """The running maximum moves at every tile, by more and by less than the range of the type; whole tiles weigh nothing beside
    one key."""
    B, H, L, T = 1, 2, 150, 700
    q, k, v, dout = _inputs(B, H, H, L, T, D, dtype, 3)
    ramp = torch.linspace(0, 6, T, device=DEV)
    for r in (ramp, ramp.flip(0), 6 * (ramp > 5.9)):
        kk = (k.float() * r[None, None, :, None]).to(dtype)
        got = _run(q, kk, v, dout)
        # sums where one term carries all: no averaging of the roundings of p and ds, and their cancellation in ds shows
        _compare(got, _exact(q, kk, v, _live(B, T, None, None), 1 / math.sqrt(D), dout), dtype, slack=2.0 if dtype != torch.float32 else 8.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 24)])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1.5])
def test_any_scale(dtype, D, scale):
    q, k, v, dout = _inputs(1, 2, 2, 140, 150, D, dtype, 4)
    s = 0.3 if scale > 1 else 1.0                 # keep the softmax from collapsing to one key
    q = q * s
    got = _run(q, k, v, dout, scale=scale)
    _compare(got, _exact(q, k, v, _live(1, 150, None, None), scale, dout), dtype, slack=2.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides_and_layouts(dtype):
    """Raster layout, slices of one projection, keys shared by the batch (expanded), rows off the 16-byte grid, a head dim that is
    not contiguous, an expanded gradient."""
    B, H, L, T, D = 2, 3, 150, 140, 64
    q, k, v, dout = _inputs(B, H, H, L, T, D, dtype, 5)
    want = _run(q, k, v, dout)
    tr = lambda x: x.transpose(1, 2).contiguous()
    got = _run(tr(q), tr(k), tr(v), tr(dout), f=V.video_cross_attn_raster)
    assert got[0].is_contiguous() and all(torch.equal(tr(a), b) for a, b in zip(got, want))
    kv = torch.cat((tr(k), tr(v)), dim=2)                    # [B, T, 2H, D]
    got = _run(tr(q), kv[:, :, :H], kv[:, :, H:], tr(dout), f=V.video_cross_attn_raster)
    assert all(torch.equal(tr(a), b) for a, b in zip(got, want))
    shared = [x[:1].expand(B, H, T, D) for x in (k, v)]
    leaf = k[:1].clone().requires_grad_()
    out = V.video_cross_attn(q, leaf.expand(B, H, T, D), shared[1])
    (dk,) = torch.autograd.grad(out, leaf, dout)
    full = _run(q, *(x.contiguous() for x in shared), dout)
    assert torch.equal(out, full[0])
    torch.testing.assert_close(dk.float(), full[2].float().sum(0, keepdim=True), atol=2e-2 if dtype == torch.bfloat16 else 1e-5, rtol=1e-2)
    off = torch.empty(q.numel() + 1, device=DEV, dtype=dtype)[1:].view(q.shape).copy_(q)
    assert torch.equal(V.video_cross_attn(off, k, v), want[0])
    flipped = q.transpose(2, 3).contiguous().transpose(2, 3)
    assert torch.equal(V.video_cross_attn(flipped, k, v), want[0])
    one = torch.ones((), device=DEV, dtype=dtype).expand_as(q)
    for a, b in zip(_run(q, k, v, one), _run(q, k, v, one.contiguous())):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 20), (torch.float32, 64)])
def test_windows_of_a_longer_row(dtype, D):
    """Rows that overlap by an element: two dims of stride 1."""
    B, H, n = 2, 3, 5
    rows = [torch.randn(B, H, n + D - 1, generator=torch.Generator().manual_seed(20 + i)).to(dtype).to(DEV) for i in range(4)]
    q, k, v, dout = (x.unfold(-1, D, 1) for x in rows)
    dense = [x.contiguous() for x in (q, k, v)]
    want = _run(*dense, dout.contiguous())
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = V.video_cross_attn(*leaves)
    got = (out, *torch.autograd.grad(out, leaves, dout))
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_empty_extents(dtype):
    for B, H, Hk, L, T in ((0, 2, 2, 5, 5), (2, 2, 1, 0, 5), (2, 2, 1, 5, 0), (1, 0, 0, 5, 5), (1, 0, 2, 5, 5)):
        q, k, v, dout = _inputs(B, H, Hk, L, T, 64, dtype, 6)
        got = _run(q, k, v, dout)
        assert all(x.shape == y.shape and not x.any() for x, y in zip(got, (q, q, k, v)))
        got = V.video_cross_attn(q, k, v, torch.zeros(B, dtype=torch.int32), kv_mask=torch.ones(B, T, dtype=torch.bool, device=DEV))
        assert not got.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 24)])
def test_gradients_of_some_operands_only(dtype, D):
    q, k, v, dout = _inputs(2, 4, 2, 130, 140, D, dtype, 11)
    mask = torch.ones(2, 140, dtype=torch.bool, device=DEV)
    mask[0, 3:70] = False
    for kw in (dict(), dict(kv_mask=mask)):
        leaves = [x.clone().requires_grad_() for x in (q, k, v)]
        want = torch.autograd.grad(V.video_cross_attn(*leaves, **kw), leaves, dout)
        for need in ((0,), (1,), (2,), (0, 2)):
            xs = [x.clone().requires_grad_(i in need) for i, x in enumerate((q, k, v))]
            got = torch.autograd.grad(V.video_cross_attn(*xs, **kw), [xs[i] for i in need], dout)
            assert all(torch.equal(g, want[i]) for g, i in zip(got, need))


@pytest.mark.gpu
def test_refusals_on_the_device():
    q, k, v, _ = _inputs(2, 2, 2, 6, 5, 16, torch.bfloat16, 7)
    for bad, match in ((dict(k=k.half(), v=v.half()), "dtype"), (dict(kv_lengths=torch.tensor([5])), "2 integers"),
                       (dict(kv_lengths=torch.tensor([5.0, 5.0])), "integers"), (dict(kv_mask=torch.ones(2, 5)), "bool"),
                       (dict(kv_mask=torch.ones(2, 6, dtype=torch.bool)), "shape"), (dict(sm_scale=math.inf), "finite")):
        args = dict(k=k, v=v, kv_lengths=None, kv_mask=None, sm_scale=None)
        args.update(bad)
        with pytest.raises(ValueError, match=match):
            V.video_cross_attn(q, args["k"], args["v"], args["kv_lengths"], kv_mask=args["kv_mask"], sm_scale=args["sm_scale"])
    with pytest.raises(ValueError, match="supports"):
        V.video_cross_attn(q.double(), k.double(), v.double())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 128), (torch.float16, 64), (torch.float32, 64)])
def test_gradients_against_differences(dtype, D):
    """A step along the gradient changes the output's weighted sum as the gradient says (central differences in float64 on the
    formula, the kernels' gradient in between)."""
    B, H, L, T = 1, 2, 130, 140
    q, k, v, dout = _inputs(B, H, 1, L, T, D, dtype, 8)
    _, *grads = _run(q, k, v, dout)
    live = _live(B, T, None, None)
    f = lambda *x: (_exact(*x, live, 1 / math.sqrt(D), dout)[0] * dout.double().cpu()).sum()
    base = [x.double().cpu() for x in (q, k, v)]
    for i in range(3):
        step = grads[i].double().cpu()
        step = step * (1e-3 / step.abs().max())
        up, down = ([x + s * step if j == i else x for j, x in enumerate(base)] for s in (1, -1))
        diff = (f(*up) - f(*down)) / 2
        assert abs(diff - (grads[i].double().cpu() * step).sum()) <= (4 * _bound(dtype) + 1e-5) * abs(diff)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_inputs_same_bits_and_side_streams(dtype):
    q, k, v, dout = _inputs(2, 4, 2, 1000, 600, 64, dtype, 10)
    want = _run(q, k, v, dout)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = _run(q, k, v, dout)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, dout), want))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_whole_step_replays_from_a_cuda_graph(dtype):
    """Two captured steps of their own sizes, replayed in turn on new numbers and new lengths."""
    steps = []
    for L, T in ((300, 200), (1, 2000)):
        q, k, v, dout = _inputs(2, 2, 2, L, T, 64, dtype, L)
        leaves = [x.requires_grad_() for x in (q, k, v)]
        lengths = torch.tensor([T, T // 2], dtype=torch.int32, device=DEV)

        def step(leaves=leaves, dout=dout, lengths=lengths):
            out = V.video_cross_attn(*leaves, lengths)
            return (out.detach(),) + torch.autograd.grad(out, leaves, dout)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            res = step()
        steps.append((graph, res, leaves, dout, lengths, T))
    for n in range(2):
        for graph, res, leaves, dout, lengths, T in steps:
            with torch.no_grad():
                for x in leaves:
                    x.mul_(-1).add_(0.01 * n)
                lengths.copy_(torch.tensor([T - 7 * n, 3]))
            graph.replay()
            torch.cuda.synchronize()
            want = _run(*leaves, dout, lengths)
            assert all(torch.equal(a, b) for a, b in zip(res, want))


def test_lengths_and_positions_of_types_that_would_wrap_are_refused():
    for dtype in (torch.uint32, torch.uint64, torch.bool, torch.float32):
        assert not ops._integers(torch.zeros(2, dtype=dtype))
    for dtype in (torch.int32, torch.int64, torch.int16, torch.int8, torch.uint8):
        assert ops._integers(torch.zeros(2, dtype=dtype))


@pytest.mark.gpu
def test_integer_types_of_lengths_and_positions():
    q, k, v, _ = _inputs(2, 2, 2, 6, 5, 16, torch.bfloat16, 21)
    rot = V.build_rotary_metadata((9,), 16, device=DEV)
    lengths, positions = torch.tensor([5, 2]), torch.tensor([0, 8, 3, 4, 1, 2])
    want, turned = V.video_cross_attn(q, k, v, lengths), V.video_rotary(q, None, rot, positions=positions)
    for dtype in (torch.int32, torch.int16, torch.int8, torch.uint8):
        assert torch.equal(V.video_cross_attn(q, k, v, lengths.to(dtype)), want)
        assert torch.equal(V.video_rotary(q, None, rot, positions=positions.to(dtype)), turned)
    for dtype in (torch.uint32, torch.uint64):
        with pytest.raises(ValueError, match="signed"):
            V.video_cross_attn(q, k, v, lengths.to(dtype))
        with pytest.raises(ValueError, match="signed"):
            V.video_rotary(q, None, rot, positions=positions.to(dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D,L", [(torch.bfloat16, 128, 300), (torch.float16, 64, 2), (torch.bfloat16, 20, 70), (torch.float32, 64, 70)])
def test_offsets_beyond_32_bits(dtype, D, L):
    """Samples of one buffer more than 2^31 elements apart, and a sample's keys that reach as far."""
    B, H, T, far, row = 2, 2, 140, (1 << 31) + (1 << 23), 1 << 24
    pool = torch.empty(far + T * row, device=DEV, dtype=dtype)
    dense = _inputs(B, H, H, L, T, D, dtype, 22)
    want = _run(*dense)
    places = [pool.as_strided((B, H, x.shape[2], D), (far, 4096, row if i == 1 else 8192, 1), 512 * i) for i, x in enumerate(dense)]
    for p, x in zip(places, dense):
        p.copy_(x)
    q, k, v, dout = places
    mask = torch.ones(B, T, dtype=torch.bool, device=DEV)
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    for kw in (dict(), dict(kv_mask=mask)):
        out = V.video_cross_attn(*leaves, **kw)
        got = (out.detach(), *torch.autograd.grad(out, leaves, dout))
        if not kw:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        else:                                            # keys gathered first: the same sums, up to their order
            for a, b in zip(got, want):
                torch.testing.assert_close(a.float(), b.float(), rtol=4 * torch.finfo(dtype).eps, atol=4 * torch.finfo(dtype).eps * b.abs().max().item())
    rot = V.build_rotary_metadata((max(L, T),), D if D % 4 == 0 else D - D % 4, device=DEV)
    assert torch.equal(V.video_rotary(k, None, rot), V.video_rotary(dense[1], None, rot))


def _cuda_core_tiles(D):
    """Which passes of [2, 4 + 2, 1300, D] x 333 run on the large tiles of the CUDA-core kernels: at least 300 tiles of scores
    (forward, dK/dV), 74 of query rows (dQ), and no more than a quarter of padding."""
    heads, Lq, Lkv = 8, 1300, 333
    tiles = lambda n, edge: -(-n // edge)
    rows, cols, keys, queries = (64, 64, 64, 32) if D > 128 else (128, 64, 128 if D <= 64 else 96, 64)
    fits = lambda n, large, small: 4 * tiles(n, large) * large <= 5 * tiles(n, small) * small
    small = 32 if D > 128 else 64
    return (fits(Lq, rows, small) and heads * tiles(Lq, rows) * tiles(Lkv, cols) >= 300, fits(Lq, rows, small) and heads * tiles(Lq, rows) >= 74,
            fits(Lkv, keys, small) and heads * tiles(Lkv, keys) * tiles(Lq, queries) >= 300)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.float32, 128), (torch.float32, 256), (torch.float32, 61), (torch.bfloat16, 100),
                                     (torch.float16, 200)])
def test_large_tiles_of_the_cuda_core_kernels(dtype, D):
    """Problems that fill the GPU with large tiles; lengths and masks, values that must not be read."""
    assert all(_cuda_core_tiles(D))
    B, H, Hk, L, T = 2, 4, 2, 1300, 333
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, dtype, D)
    lengths = torch.tensor([T, 190])
    mask = torch.rand(B, T, generator=torch.Generator().manual_seed(1)) < 0.7
    for ln, mk in ((None, None), (lengths, None), (lengths, mask)):
        live = _live(B, T, ln, mk)
        kk, vv = k.clone(), v.clone()
        dead = ~live[:, None, :, None].to(DEV).expand_as(kk)
        kk[dead], vv[dead] = math.nan, math.inf
        got = _run(q, kk, vv, dout, None if ln is None else ln.to(DEV), None if mk is None else mk.to(DEV))
        _compare(got, _exact(q, k, v, live, 1 / math.sqrt(D), dout), dtype)
        assert not got[2][dead].any() and not got[3][dead].any()


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 200])
def test_few_rows_of_queries_against_long_states_in_fp32(D):
    """dQ cut over the keys: parts without a live key, and a sample without one."""
    B, H, Hk, L, T = 2, 1, 1, 70, 1900
    q, k, v, dout = _inputs(B, H, Hk, L, T, D, torch.float32, D + 1)
    for lengths in (None, torch.tensor([1900, 100]), torch.tensor([0, 65])):
        live = _live(B, T, lengths, None)
        got = _run(q, k, v, dout, None if lengths is None else lengths.to(DEV))
        _compare(got, _exact(q, k, v, live, 1 / math.sqrt(D), dout), torch.float32)
        assert all(torch.equal(a, b) for a, b in zip(got, _run(q, k, v, dout, None if lengths is None else lengths.to(DEV))))
