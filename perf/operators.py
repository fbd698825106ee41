"""Performance cases of the operators that stand beside Video Sparse Attention in a transformer layer.

* ``cross``: ``video_cross_attn`` / ``video_cross_attn_raster``: the video tokens attend to an encoder's states of another
  length (every key that is live for the sample, no routing), forward alone or with the gradients of q, k and v;
* ``rotary``: ``video_rotary`` / ``video_rotary_raster``: rotary positions of q and k in one call, the first ``rotary_dim``
  dims of each head, pairs interleaved or in halves, rows of the table by token or by a position of the caller;
* ``tile_rotary``: ``tile_heads(x, meta, rotary)``: raster-order activations rotated on their way into tile order.

``run`` computes the same operators from elementary torch operations in 32 bits while ``own`` is false.  Inputs are N(0,1)
like a normalised layer's activations; the angles are those of a (t, h, w) token grid.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ELEMENT = {"bf16": 2, "fp16": 2, "fp32": 4}
BLOCKS = {64: (4, 4, 4), 128: (4, 4, 8), 256: (4, 8, 8)}
CHUNK = 1 << 29                  # scores that the plain form holds at once (2 GB in 32 bits)


def _cross(name, dtype, batch, heads, kv_heads, tokens, keys, dim, **more):
    c = dict(name=name, op="cross", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, tokens=tokens, keys=keys, dim=dim,
             ragged=False, mask=False, raster=False, train=False)
    c.update(more)
    return c


def _rotary(name, dtype, batch, heads, kv_heads, tokens, dim, rotary_dim, **more):
    c = dict(name=name, op="rotary", dtype=dtype, batch=batch, heads=heads, kv_heads=kv_heads, tokens=tokens, dim=dim,
             rotary_dim=rotary_dim, interleaved=True, raster=False, positions=False, train=False)
    c.update(more)
    return c


def _tile_rotary(name, dtype, batch, heads, grid, dim, rotary_dim, block, **more):
    c = dict(name=name, op="tile_rotary", dtype=dtype, batch=batch, heads=heads, grid_t=grid[0], grid_h=grid[1], grid_w=grid[2],
             dim=dim, rotary_dim=rotary_dim, block=block, interleaved=True, train=False)
    c.update(more)
    return c


def listed():
    return [
        # one new token of each of eight samples against the encoder's states: a pass over K and V, latency counts
        _cross("cross_token", "bf16", 8, 40, 40, 1, 512, 128, ragged=True),
        # a sampling step on a thumbnail-sized latent with a short prompt of odd length
        _cross("cross_infer_4k_77", "bf16", 1, 12, 12, 4096, 77, 128),
        # numerics check in fp32, both lengths odd
        _cross("cross_train_1k_fp32_d64", "fp32", 1, 2, 2, 1025, 333, 64, ragged=True, train=True),
        # a training batch of two clips at head dim 64, keys and values shared by three heads each, keys masked one by one
        _cross("cross_train_8k_d64_mask", "fp16", 2, 12, 4, 8190, 1001, 64, mask=True, train=True),
        # the 16k-token training configuration; prompts of two samples padded to 512
        _cross("cross_train_16k", "bf16", 2, 12, 12, 16384, 512, 128, ragged=True, train=True),
        # one eight-head shard of the 92k-token shape, activations as the projections leave them
        _cross("cross_train_92k_h8_raster", "bf16", 1, 8, 8, 92160, 512, 128, raster=True, train=True),
        # sampling at 92k tokens with all forty heads
        _cross("cross_infer_92k", "bf16", 1, 40, 40, 92160, 512, 128),
        # a decoding step: one token of each sample at a position of its own, half of the head rotated
        _rotary("rotary_token_half", "fp16", 8, 40, 8, 1, 128, 64, interleaved=False, positions=True),
        # q and k of the 16k-token training configuration
        _rotary("rotary_train_16k", "bf16", 1, 12, 12, 16384, 128, 128, train=True),
        # raster-order activations at the 92k-token shape, two samples
        _rotary("rotary_92k_raster", "bf16", 2, 40, 40, 92160, 128, 128, raster=True),
        # the layer that tiles its activations (tiles clipped on two axes), with the rotation on the way
        _tile_rotary("tile_rotary_train_81k", "bf16", 1, 8, (20, 45, 90), 128, 128, 64, train=True),
        # the same pass in sampling at head dim 64, in fp16, the two axes of a frame rotated
        _tile_rotary("tile_rotary_40k_d64", "fp16", 2, 12, (13, 48, 64), 64, 44, 256, interleaved=False),
    ]


LARGEST_CROSS_PAIRS = 40 * 92160 * 512            # scores of the largest listed attention
LARGEST_ROTARY_VALUES = 2 * 80 * 92160 * 128      # values of q and k of the largest listed rotation


def _log_uniform(rng, low, high):
    return math.exp(rng.uniform(math.log(low), math.log(high)))


def draw(rng):
    """One more case: lengths, heads, shared heads, head dims, masks, types, layouts and directions vary."""
    while True:
        op = rng.choice(("cross", "cross", "cross", "rotary", "rotary", "tile_rotary"))
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp16", "fp32"))
        dim = rng.choice((128, 128, 128, 64, 64))
        kv_heads = round(_log_uniform(rng, 1, 40))
        heads = kv_heads * rng.choice((1, 1, 1, 2, 3))
        batch = rng.choice((1, 1, 2, 3))
        train = rng.random() < 0.6
        if op == "cross":
            few = rng.random() < 0.15
            tokens = rng.randint(1, 16) if few else round(_log_uniform(rng, 64, 100000))
            keys = round(_log_uniform(rng, 16, 2048))
            if few:
                batch, train = rng.randint(1, 8), False
            if dtype == "fp32":                       # the numerics mode: small problems only
                tokens, heads, kv_heads = min(tokens, rng.randint(500, 2000)), min(heads, 8), 1
                heads = max(1, heads)
            masks = rng.choice(("none", "ragged", "mask"))
            c = _cross("", dtype, batch, heads, kv_heads, tokens, keys, dim, ragged=masks == "ragged", mask=masks == "mask",
                       raster=rng.random() < 0.4, train=train)
            fits = batch * heads * tokens * keys * (3 if train else 1) <= LARGEST_CROSS_PAIRS
        elif op == "rotary":
            tokens = 1 if rng.random() < 0.15 else round(_log_uniform(rng, 2, 100000))
            c = _rotary("", dtype, batch, heads, kv_heads, tokens, dim, rng.choice((dim, dim, dim // 2, dim - 20)),
                        interleaved=rng.random() < 0.5, raster=rng.random() < 0.5, positions=tokens == 1 or rng.random() < 0.3,
                        train=train and tokens > 1)
            fits = batch * (heads + kv_heads) * tokens * dim * (2 if train else 1) * ELEMENT[dtype] <= 2 * LARGEST_ROTARY_VALUES
        else:
            grid = (rng.randint(2, 24), rng.randint(8, 60), rng.randint(8, 90))
            c = _tile_rotary("", dtype, batch, kv_heads, grid, dim, rng.choice((dim, dim, dim // 2, dim - 20)),
                             rng.choice((64, 64, 128, 256)), interleaved=rng.random() < 0.5, train=train)
            fits = batch * kv_heads * math.prod(grid) * dim * ELEMENT[dtype] <= LARGEST_ROTARY_VALUES
        del c["name"]
        if fits:
            return c


# ---- inputs -------------------------------------------------------------------------------------------------------
def _normal(shape, dtype, gen):
    return torch.empty(shape, device="cuda", dtype=dtype).normal_(generator=gen)


def _grid_of(tokens):
    """A (t, h, w) grid of at least ``tokens`` positions, the frames at most 48 x 80."""
    h = max(1, min(48, round(math.sqrt(tokens / 2))))
    w = max(1, min(80, -(-tokens // h)))
    return -(-tokens // (h * w)), h, w


def _angles(grid, rotary_dim, theta=10000.0):
    """cos and sin ``[t*h*w, rotary_dim/2]`` in 32 bits of a token grid's angles, the pairs of a head dealt to the three axes."""
    pairs = rotary_dim // 2
    share = [pairs - 2 * (pairs // 3), pairs // 3, pairs // 3]
    parts = []
    for axis, (n, p) in enumerate(zip(grid, share)):
        at = torch.arange(n, device="cuda", dtype=torch.float64)
        a = at[:, None] * theta ** (-torch.arange(p, device="cuda", dtype=torch.float64) / max(1, p))[None, :]
        shape = [1, 1, 1, p]
        shape[axis] = n
        parts.append(a.view(shape).expand(*grid, p))
    angle = torch.cat(parts, dim=-1).reshape(-1, pairs)
    return angle.cos().float(), angle.sin().float()


def _tile_rows(case):
    """Raster index of every tile-order token, -1 for padding: tiles in raster order, a clipped tile's tokens at its front."""
    grid, (a, b, c) = (case["grid_t"], case["grid_h"], case["grid_w"]), BLOCKS[case["block"]]
    ids = torch.arange(math.prod(grid)).view(grid)
    rows = []
    for t in range(0, grid[0], a):
        for h in range(0, grid[1], b):
            for w in range(0, grid[2], c):
                live = ids[t:t + a, h:h + b, w:w + c].reshape(-1)
                rows.append(torch.nn.functional.pad(live, (0, case["block"] - live.numel()), value=-1))
    return torch.cat(rows).cuda()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, D, dtype = case["batch"], case["dim"], DTYPES[case["dtype"]]
    state = {"case": case}

    def heads_of(n, tokens):
        return _normal((B, tokens, n, D) if case.get("raster") else (B, n, tokens, D), dtype, gen)

    if case["op"] == "cross":
        H, Hk, L, T = case["heads"], case["kv_heads"], case["tokens"], case["keys"]
        tensors = {"q": heads_of(H, L), "k": heads_of(Hk, T), "v": heads_of(Hk, T)}
        if case["ragged"]:
            # prompts between a quarter and all of the padded length; the first sample's fills it
            state["lengths"] = torch.randint(max(1, T // 4), T + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
            state["lengths"][0] = T
        if case["mask"]:
            state["mask"] = torch.rand((B, T), device="cuda", generator=gen) < 0.8
        if case["train"]:
            state["dout"] = heads_of(H, L)
    elif case["op"] == "rotary":
        H, Hk, L, R = case["heads"], case["kv_heads"], case["tokens"], case["rotary_dim"]
        tensors = {"q": heads_of(H, L), "k": heads_of(Hk, L)}
        rows = L
        if case["positions"]:
            rows = max(4096, L)
            state["positions"] = torch.randint(0, rows, (B, L), device="cuda", generator=gen, dtype=torch.int32)
        cos, sin = _angles(_grid_of(rows), R)
        state["rotary"] = {"cos": cos[:rows].contiguous(), "sin": sin[:rows].contiguous(), "interleaved": case["interleaved"]}
        if case["train"]:
            state["dq"], state["dk"] = heads_of(H, L), heads_of(Hk, L)
    else:
        grid = (case["grid_t"], case["grid_h"], case["grid_w"])
        tensors = {"x": _normal((B, math.prod(grid), case["heads"], D), dtype, gen)}
        state["rows"] = _tile_rows(case)
        cos, sin = _angles(grid, case["rotary_dim"])
        state["rotary"] = {"cos": cos, "sin": sin, "interleaved": case["interleaved"]}
        if case["train"]:
            state["dout"] = _normal((B, case["heads"], state["rows"].numel(), D), dtype, gen)
        if own:
            import simple_vsa_b200 as vsa
            state["meta"] = vsa.build_vsa_metadata(grid, BLOCKS[case["block"]], "cuda")
    if own and case["train"]:
        for t in tensors.values():
            t.requires_grad_()
    state["tensors"] = tensors
    return state


# ---- the framework's calls -----------------------------------------------------------------------------------------
def _own_call(state):
    import simple_vsa_b200 as vsa
    case, t = state["case"], state["tensors"]
    if case["op"] == "cross":
        f = vsa.video_cross_attn_raster if case["raster"] else vsa.video_cross_attn
        return (f(t["q"], t["k"], t["v"], state.get("lengths"), kv_mask=state.get("mask")),)
    if case["op"] == "rotary":
        f = vsa.video_rotary_raster if case["raster"] else vsa.video_rotary
        return f(t["q"], t["k"], state["rotary"], positions=state.get("positions"))
    return (vsa.tile_heads(t["x"], state["meta"], rotary=state["rotary"]),)


NAMES = {"cross": (("out",), ("dq", "dk", "dv")), "rotary": (("q", "k"), ("dq", "dk")), "tile_rotary": (("out",), ("dx",))}


def _own_run(state):
    case = state["case"]
    names, grad_names = NAMES[case["op"]]
    if not case["train"]:
        with torch.no_grad():
            return dict(zip(names, _own_call(state)))
    outs = _own_call(state)
    douts = (state["dq"], state["dk"]) if case["op"] == "rotary" else (state["dout"],)
    grads = torch.autograd.grad(outs, list(state["tensors"].values()), douts)
    result = {n: o.detach() for n, o in zip(names, outs)}
    result.update(zip(grad_names, grads))
    return result


# ---- the plain form ------------------------------------------------------------------------------------------------
def _plain_cross(state):
    """softmax over the live keys, 32 bits; samples and heads in chunks that bound the scores' memory."""
    case, t = state["case"], state["tensors"]
    B, H, Hk, L, T, D = (case[n] for n in ("batch", "heads", "kv_heads", "tokens", "keys", "dim"))
    dtype, scale, group = DTYPES[case["dtype"]], 1.0 / math.sqrt(case["dim"]), case["heads"] // case["kv_heads"]
    tensors = dict(t, dout=state["dout"]) if case["train"] else t
    if case["raster"]:
        tensors = {n: x.transpose(1, 2) for n, x in tensors.items()}
    live = torch.ones((B, T), device="cuda", dtype=torch.bool)
    if "lengths" in state:
        live = torch.arange(T, device="cuda")[None, :] < state["lengths"][:, None]
    if "mask" in state:
        live = live & state["mask"]

    def empty_like(x):                                   # in the memory order of the operand
        return torch.empty_like(x, memory_format=torch.preserve_format)

    res = {"out": empty_like(tensors["q"])}
    if case["train"]:
        res.update({"d" + n: empty_like(tensors[n]) for n in "qkv"})
    per_batch = H * L * T
    batches = max(1, min(B, CHUNK // per_batch))
    groups = Hk if per_batch <= CHUNK else max(1, min(Hk, CHUNK // (L * T * group)))
    for b in range(0, B, batches):
        for g in range(0, Hk, groups):
            bs, ks, hs = slice(b, b + batches), slice(g, g + groups), slice(g * group, (g + groups) * group)
            dead = ~live[bs][:, None, None, :]
            k, v = (tensors[n][bs, ks].float().masked_fill(dead.transpose(2, 3), 0.0) for n in "kv")
            n, h = k.shape[:2]
            # the heads that share a key head lie one after another: one product over their rows together
            q = tensors["q"][bs, hs].float().reshape(n, h, group * L, D)
            s = torch.matmul(q, k.transpose(2, 3)).mul_(scale).masked_fill_(dead, -math.inf)
            top = s.amax(dim=-1, keepdim=True)
            p = s.sub_(top.masked_fill(top == -math.inf, 0.0)).exp_()
            total = p.sum(dim=-1, keepdim=True)
            p = p.div_(total.masked_fill(total == 0, 1.0))
            out = torch.matmul(p, v)
            res["out"][bs, hs] = out.reshape(n, h * group, L, D).to(dtype)
            if case["train"]:
                do = tensors["dout"][bs, hs].float().reshape(n, h, group * L, D)
                res["dv"][bs, ks] = torch.matmul(p.transpose(2, 3), do).to(dtype)
                ds = torch.matmul(do, v.transpose(2, 3)).sub_((do * out).sum(dim=-1, keepdim=True)).mul_(p).mul_(scale)
                res["dq"][bs, hs] = torch.matmul(ds, k).reshape(n, h * group, L, D).to(dtype)
                res["dk"][bs, ks] = torch.matmul(ds.transpose(2, 3), q).to(dtype)
    return {n: x.transpose(1, 2) for n, x in res.items()} if case["raster"] else res


def _plain_rotate(x, cos, sin, interleaved):
    """``x[..., :2p]`` rotated by the angles whose ``cos`` and ``sin`` ``[..., p]`` broadcast against it, in 32 bits."""
    p = cos.shape[-1]
    y = x.float()
    head, rest = y[..., :2 * p], y[..., 2 * p:]
    if interleaved:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), dim=-1).flatten(-2)
    else:
        a, b = head[..., :p], head[..., p:]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)
    return torch.cat((turned, rest), dim=-1).to(x.dtype)


def _plain_rotary(state):
    case, rot = state["case"], state["rotary"]
    cos, sin = rot["cos"], rot["sin"]
    if "positions" in state:
        cos, sin = cos[state["positions"].long()], sin[state["positions"].long()]
    else:
        cos, sin = cos[None], sin[None]
    cos, sin = (x.unsqueeze(2 if case["raster"] else 1) for x in (cos, sin))
    res = {n: _plain_rotate(x, cos, sin, case["interleaved"]) for n, x in state["tensors"].items()}
    if case["train"]:
        res.update({n: _plain_rotate(state[n], cos, -sin, case["interleaved"]) for n in ("dq", "dk")})
    return res


def _plain_tile_rotary(state):
    case, rot, rows = state["case"], state["rotary"], state["rows"]
    x, live = state["tensors"]["x"], state["rows"] >= 0
    cos, sin = (r[None, :, None, :] for r in (rot["cos"], rot["sin"]))
    turned = _plain_rotate(x, cos, sin, case["interleaved"])
    tiled = turned.new_zeros((x.shape[0], rows.numel()) + x.shape[2:])
    tiled[:, live] = turned[:, rows[live]]
    res = {"out": tiled.transpose(1, 2).contiguous()}
    if case["train"]:
        back = torch.empty_like(x)
        back[:, rows[live]] = state["dout"].transpose(1, 2)[:, live]
        res["dx"] = _plain_rotate(back, cos, -sin, case["interleaved"])
    return res


def run(state):
    if own:
        return _own_run(state)
    return {"cross": _plain_cross, "rotary": _plain_rotary, "tile_rotary": _plain_tile_rotary}[state["case"]["op"]](state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    """Each operand read once, each result written once.  Attention: 2 products of 2 D flops per score forward and 5
    backward; a rotation: 6 flops per pair of values."""
    B, D, e = case["batch"], case["dim"], ELEMENT[case["dtype"]]
    if case["op"] == "cross":
        H, Hk, L, T = case["heads"], case["kv_heads"], case["tokens"], case["keys"]
        live = 0.625 * (1 + 0.6 / B) if case["ragged"] else 0.8 if case["mask"] else 1.0
        pairs = B * H * L * T * live
        q, kv = B * H * L * D * e, 2 * B * Hk * T * D * e * (1 if case["train"] else live)
        moved = (2 * q + kv) + ((2 * q + kv) if case["train"] else 0)     # backward: dout in, dq, dk, dv out
        return {"bytes": float(moved), "flops": (14.0 if case["train"] else 4.0) * pairs * D}
    directions = 2 if case["train"] else 1
    if case["op"] == "rotary":
        rows = B * case["tokens"] if case["positions"] else case["tokens"]
        values = B * (case["heads"] + case["kv_heads"]) * case["tokens"]
        moved = directions * 2 * values * D * e + rows * case["rotary_dim"] * 4 + (rows * 4 if case["positions"] else 0)
        return {"bytes": float(moved), "flops": 3.0 * directions * values * case["rotary_dim"]}
    grid = (case["grid_t"], case["grid_h"], case["grid_w"])
    tokens, padded = math.prod(grid), case["block"] * math.prod(-(-n // s) for n, s in zip(grid, BLOCKS[case["block"]]))
    values = B * case["heads"] * tokens
    moved = B * case["heads"] * D * e * (tokens + padded + (2 * tokens if case["train"] else 0)) + tokens * case["rotary_dim"] * 4 + padded * 4
    return {"bytes": float(moved), "flops": 3.0 * directions * values * case["rotary_dim"]}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------
def _exact_cross(case, state):
    """Head by head: softmax and its gradient by autograd, in float64."""
    B, H, Hk, T = case["batch"], case["heads"], case["kv_heads"], case["keys"]
    order = (lambda x: x.transpose(1, 2)) if case["raster"] else (lambda x: x)
    t = {n: order(x.detach()) for n, x in state["tensors"].items()}
    live = torch.ones((B, T), device="cuda", dtype=torch.bool)
    if "lengths" in state:
        live = torch.arange(T, device="cuda")[None, :] < state["lengths"][:, None]
    if "mask" in state:
        live = live & state["mask"]
    res = {"out": torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64)}
    if case["train"]:
        res.update({"d" + n: torch.zeros(t[n].shape, device="cuda", dtype=torch.float64) for n in "qkv"})
    for b in range(B):
        at = live[b].nonzero().flatten()
        if at.numel() == 0:
            continue
        for h in range(H):
            g = h // (H // Hk)
            step = max(1, (1 << 27) // at.numel())
            for r in range(0, t["q"].shape[2], step):
                q, k, v = (x.double().requires_grad_(case["train"]) for x in (t["q"][b, h, r:r + step], t["k"][b, g, at], t["v"][b, g, at]))
                o = torch.softmax((q @ k.T) / math.sqrt(case["dim"]), dim=-1) @ v
                res["out"][b, h, r:r + step] = o.detach()
                if case["train"]:
                    dq, dk, dv = torch.autograd.grad(o, (q, k, v), order(state["dout"])[b, h, r:r + step].double())
                    res["dq"][b, h, r:r + step] = dq
                    res["dk"][b, g, at] += dk
                    res["dv"][b, g, at] += dv
    return {n: order(x) for n, x in res.items()}


def _exact_turn(x, angle, interleaved):
    """A pair of values as a complex number, times ``angle`` (complex128, broadcast against the pairs)."""
    p = angle.shape[-1]
    y = x.double()
    pairs = y[..., :2 * p]
    pairs = pairs.unflatten(-1, (p, 2)) if interleaved else torch.stack(pairs.chunk(2, dim=-1), dim=-1)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * angle)
    y[..., :2 * p] = turned.flatten(-2) if interleaved else torch.cat(turned.unbind(-1), dim=-1)
    return y


def exact(case, seed):
    """``run``'s outputs in float64 from the definitions."""
    state = prepare(case, seed)
    if case["op"] == "cross":
        with torch.enable_grad():
            return _exact_cross(case, state)
    rot = state["rotary"]
    angle = torch.complex(rot["cos"].double(), rot["sin"].double())
    t = {n: x.detach() for n, x in state["tensors"].items()}
    if case["op"] == "rotary":
        angle = angle[state["positions"].long()] if "positions" in state else angle[None]
        angle = angle.unsqueeze(2 if case["raster"] else 1)
        res = {n: _exact_turn(x, angle, case["interleaved"]) for n, x in t.items()}
        if case["train"]:
            res.update({n: _exact_turn(state[n], angle.conj(), case["interleaved"]) for n in ("dq", "dk")})
        return res
    rows, live = state["rows"], state["rows"] >= 0
    out = torch.zeros((t["x"].shape[0], case["heads"], rows.numel(), case["dim"]), device="cuda", dtype=torch.float64)
    source = rows[live]
    out[:, :, live] = _exact_turn(t["x"][:, source].transpose(1, 2), angle[source], case["interleaved"])
    res = {"out": out}
    if case["train"]:
        dx = torch.zeros(t["x"].shape, device="cuda", dtype=torch.float64)
        dx[:, source] = _exact_turn(state["dout"][:, :, live], angle[source].conj(), case["interleaved"]).transpose(1, 2)
        res["dx"] = dx
    return res
