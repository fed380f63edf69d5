"""Cases of two operator pairs of the encoder's attention path, with their plain forms.

* ``qk``: the norm of every query and key head of a packed projection output and the rotary position rotation, in one
  pass, and its gradient (``vit_amd.ops.qk_norm_rope`` / ``qk_norm_rope_backward``).
* ``rel``: attention with a learned relative position bias by buckets, and its gradient, the table's included
  (``vit_amd.ops.attention_rel_bias`` / ``_train`` / ``_backward``).

``run`` computes the plain form (elementary torch operations in 32 bits) while ``own`` is false and calls the package
while it is true. The packed layout is the encoder's: ``[batch, tokens, q heads | k heads | v heads]``.
"""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def _qk(name, direction, batch, grid_h, grid_w, prefix, heads, kv_heads, head_dim, rot_dim, interleaved, norm, given_positions, dtype):
    return {"name": name, "op": "qk", "direction": direction, "batch": batch, "grid_h": grid_h, "grid_w": grid_w, "prefix": prefix,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "rot_dim": rot_dim, "interleaved": interleaved,
            "norm": norm, "given_positions": given_positions, "dtype": dtype}


def _rel(name, direction, batch, grid_h, grid_w, prefix, heads, kv_heads, head_dim, log_buckets, ragged, dtype):
    return {"name": name, "op": "rel", "direction": direction, "batch": batch, "grid_h": grid_h, "grid_w": grid_w, "prefix": prefix,
            "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "log_buckets": log_buckets, "ragged": ragged, "dtype": dtype}


def listed():
    return [
        # one 224-pixel image through a base-size encoder: latency of an interactive embedding call
        _qk("qk one image", "forward", 1, 14, 14, 1, 12, 12, 64, 64, False, "rms", False, "bf16"),
        # the batch of the throughput benchmark (256 images of 197 tokens), inference and the training step's backward
        _qk("qk base batch", "forward", 256, 14, 14, 1, 12, 12, 64, 64, False, "rms", False, "bf16"),
        _qk("qk base batch gradient", "backward", 256, 14, 14, 1, 12, 12, 64, 64, False, "rms", False, "bf16"),
        # 448-pixel images through a huge-size encoder (head_dim 80), part of each head rotated, neighbours paired, full
        # LayerNorm on the heads, fp32: the numerics-checking mode of the gradient
        _qk("qk huge fp32 gradient", "backward", 3, 32, 32, 1, 16, 16, 80, 64, True, "layer", False, "f32"),
        # a packed batch of crops, every token with its own position, keys shared by groups of query heads
        _qk("qk packed crops", "forward", 9, 1, 331, 0, 12, 4, 96, 96, False, "layer", True, "bf16"),
        # one 224-pixel image: latency
        _rel("rel one image", "forward", 1, 14, 14, 1, 12, 12, 64, 0, False, "bf16"),
        # the throughput batch, inference and one training step (forward and backward)
        _rel("rel base batch", "forward", 256, 14, 14, 1, 12, 12, 64, 0, False, "bf16"),
        _rel("rel base batch training", "training", 256, 14, 14, 1, 12, 12, 64, 0, False, "bf16"),
        # 336-pixel images through a large-size tower (577 tokens)
        _rel("rel large batch", "forward", 32, 24, 24, 1, 16, 16, 64, 0, False, "bf16"),
        # 448-pixel images through a huge-size encoder (1025 tokens, head_dim 80): fine-tuning at high resolution
        _rel("rel huge training", "training", 4, 32, 32, 1, 16, 16, 80, 0, False, "bf16"),
        # a padded batch of one-dimensional sequences of different lengths, logarithmic buckets, shared key heads
        _rel("rel padded sequences", "forward", 6, 1, 1777, 0, 16, 4, 128, 32, True, "bf16"),
        # the fp32 mode that checks numerics against a CPU run
        _rel("rel fp32", "forward", 4, 14, 14, 1, 12, 12, 64, 0, False, "f32"),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["qk", "rel"])
    direction = rng.choice(["forward", "backward"] if op == "qk" else ["forward", "training"])
    dtype = rng.choice(["bf16", "bf16", "f32"] if direction != "training" else ["bf16"])
    heads = rng.choice([3, 4, 6, 8, 12, 16])
    kv_heads = rng.choice([heads, heads, heads // 2 if heads % 2 == 0 else 1])
    head_dim = rng.choice([32, 48, 64, 64, 64, 80, 96, 128])
    if rng.random() < 0.7:
        grid_h, grid_w, prefix = _log_int(rng, 2, 36), _log_int(rng, 2, 36), rng.choice([0, 1, 1, 5])
    else:
        grid_h, grid_w, prefix = 1, _log_int(rng, 2, 2000), 0
    n = grid_h * grid_w + prefix
    if op == "qk":
        most = 50432 * 24 * 64 // (n * (heads + kv_heads) * head_dim)
        batch = _log_int(rng, 1, max(1, min(256, most // (2 if dtype == "f32" else 1))))
        rot_dim = rng.choice([head_dim, head_dim, 16 * rng.randint(1, head_dim // 16)])
        c = _qk("", direction, batch, grid_h, grid_w, prefix, heads, kv_heads, head_dim, rot_dim, rng.random() < 0.5,
                rng.choice(["rms", "layer"]), rng.random() < 0.3, dtype)
    else:
        most = int(256 * 12 * 197 * 197 * 64 / (heads * n * n * head_dim) / (8 if dtype == "f32" else 1))
        batch = _log_int(rng, 1, max(1, min(256, most)))
        c = _rel("", direction, batch, grid_h, grid_w, prefix, heads, kv_heads, head_dim,
                 rng.choice([8, 32, 48]) if grid_h == 1 else 0, rng.random() < 0.4, dtype)
    del c["name"]
    return c


def _tokens(case):
    return case["grid_h"] * case["grid_w"] + case["prefix"]


def _width(case):
    return (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]


def _rope_table(case):
    """[grid tokens, rot_dim / 2, 2] (cos, sin), angles in 64 bits: half the pairs turn with the row and half with the
    column of the grid, or all of them with the place in a sequence."""
    pairs = case["rot_dim"] // 2
    f64 = dict(dtype=torch.float64, device="cuda")
    if case["grid_h"] == 1:
        freq = 10000.0 ** (-torch.arange(pairs, **f64) / pairs)
        angle = torch.arange(case["grid_w"], **f64)[:, None] * freq
    else:
        half = pairs // 2
        freq = 100.0 ** (-torch.arange(half, **f64) / half)
        y = torch.arange(case["grid_h"], **f64)[:, None, None].expand(-1, case["grid_w"], half) * freq
        x = torch.arange(case["grid_w"], **f64)[None, :, None].expand(case["grid_h"], -1, half) * freq
        angle = torch.cat([y, x], dim=-1).reshape(-1, pairs)
    return torch.stack([angle.cos(), angle.sin()], dim=-1).float().contiguous()


def _offset_buckets(case):
    """int64 [offsets]: the bucket of every key place minus... query place minus key place, from -(n-1) to n-1: exact up to
    a quarter of the buckets in each direction, logarithmic to a distance of 128 behind that."""
    n, half = case["grid_w"], case["log_buckets"] // 2
    exact_to = half // 2
    d = torch.arange(-(n - 1), n, dtype=torch.float64, device="cuda")  # query - key
    a = d.abs().clamp(min=1.0)
    far = exact_to + torch.floor(torch.log(a / exact_to) / math.log(128 / exact_to) * (half - exact_to) + 1e-9).clamp(max=half - exact_to - 1)
    b = torch.where(d.abs() < exact_to, d.abs(), far)
    return (b + half * (d < 0)).to(torch.int64)


def _bucket_index(case, offset_buckets):
    """int64 [tokens, tokens]: the bucket of every (query, key). A grid has one bucket for every (row, column) offset, then
    three for the tokens before it: from one of them, to one of them, among them."""
    gh, gw, p = case["grid_h"], case["grid_w"], case["prefix"]
    g = torch.arange(gh * gw, device="cuda")
    dy = g[:, None] // gw - g[None, :] // gw + gh - 1
    dx = g[:, None] % gw - g[None, :] % gw + gw - 1
    offset = dy * (2 * gw - 1) + dx
    if offset_buckets is not None:
        return offset_buckets[offset]
    offsets = (2 * gh - 1) * (2 * gw - 1)
    index = torch.full((_tokens(case), _tokens(case)), offsets + 2, dtype=torch.int64, device="cuda")
    index[:p, p:] = offsets
    index[p:, :p] = offsets + 1
    index[p:, p:] = offset
    return index


def _buckets(case):
    if case["log_buckets"]:
        return case["log_buckets"]
    return (2 * case["grid_h"] - 1) * (2 * case["grid_w"] - 1) + (3 if case["prefix"] else 0)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(*shape, dtype=torch.float32, by=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * by).to(dtype)

    b, n, dt = case["batch"], _tokens(case), DT[case["dtype"]]
    s = {"case": case, "qkv": randn(b, n, _width(case), dtype=dt)}
    if case["op"] == "qk":
        dh = case["head_dim"]
        s["qkv"] *= 1.5
        s["eps"] = 1e-6
        s["q_weight"], s["k_weight"] = 1 + randn(dh, by=0.2), 1 + randn(dh, by=0.2)
        layer = case["norm"] == "layer"
        s["q_bias"], s["k_bias"] = (randn(dh, by=0.1), randn(dh, by=0.1)) if layer else (None, None)
        s["rope"] = _rope_table(case)
        grid = s["rope"].shape[0]
        if case["given_positions"]:  # every token of every sample has a place of its own
            s["positions"] = torch.randint(0, grid, (b, n), generator=g, device="cuda", dtype=torch.int32)
        else:  # the tokens before the grid are not turned
            s["positions"] = torch.arange(-case["prefix"], grid, dtype=torch.int32, device="cuda").clamp(min=-1)
        if case["direction"] == "backward":
            s["d_out"] = randn(b, n, _width(case), dtype=dt)
        return s
    offsets = _offset_buckets(case) if case["log_buckets"] else None
    s["index"] = _bucket_index(case, offsets)
    s["table"] = randn(_buckets(case), case["heads"], by=0.7)
    s["lengths"] = torch.randint(max(1, n // 5), n + 1, (b,), generator=g, device="cuda", dtype=torch.int32) if case["ragged"] else None
    s["scale"] = case["head_dim"] ** -0.5
    if case["direction"] == "training":
        s["d_out"] = randn(b, n, case["heads"] * case["head_dim"], dtype=dt)
    if own:
        from vit_amd.rel_pos import RelPosBuckets
        s["buckets"] = RelPosBuckets((case["grid_h"], case["grid_w"]), prefix=case["prefix"], bucket_of=offsets,
                                     num_buckets=_buckets(case), device="cuda")
    return s


# ------------------------------------------------------------------------------------------------- plain forms
def _turn(x, s, sign):
    """The first rot_dim values of every head turned by sign * the angle of the token's position; -1: not turned."""
    c = s["case"]
    rot, pos = c["rot_dim"], s["positions"].long()
    cs = s["rope"][pos.clamp(min=0)]
    turned = (pos >= 0)[..., None]
    cos = torch.where(turned, cs[..., 0], 1.0).unsqueeze(-2)
    sin = torch.where(turned, cs[..., 1], 0.0).unsqueeze(-2) * sign
    if c["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        out = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2:rot]
        out = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([out, x[..., rot:]], dim=-1)


def _heads(x, c):
    """Packed rows in 32 bits as (q [b, n, h, dh], k [b, n, hk, dh], v)."""
    b, n, _ = x.shape
    h, hk, dh = c["heads"], c["kv_heads"], c["head_dim"]
    x = x.float().view(b, n, h + 2 * hk, dh)
    return x[:, :, :h], x[:, :, h:h + hk], x[:, :, h + hk:]


def _normed(x, c, eps):
    """(normalised heads, 1 / their deviation)"""
    if c["norm"] == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def _plain_qk_forward(s):
    c, x = s["case"], s["qkv"]
    q, k, _ = _heads(x, c)
    q = _normed(q, c, s["eps"])[0] * s["q_weight"]
    k = _normed(k, c, s["eps"])[0] * s["k_weight"]
    if s["q_bias"] is not None:
        q, k = q + s["q_bias"], k + s["k_bias"]
    out = x.clone()
    qk = torch.cat([_turn(q, s, 1.0), _turn(k, s, 1.0)], dim=2).flatten(2)
    out[..., : qk.shape[-1]] = qk.to(x.dtype)
    return out


def _plain_qk_part(x, dy, weight, s):
    c = s["case"]
    xh, r = _normed(x, c, s["eps"])
    t = _turn(dy, s, -1.0)
    u = t * xh
    g = t * weight
    dx = g - xh * (g * xh).mean(-1, keepdim=True)
    if c["norm"] == "layer":
        dx = dx - g.mean(-1, keepdim=True)
    return dx * r, u.double().sum((0, 1, 2)).float(), t.double().sum((0, 1, 2)).float()


def _plain_qk_backward(s):
    c, x = s["case"], s["qkv"]
    q, k, _ = _heads(x, c)
    dq, dk, _ = _heads(s["d_out"], c)
    dq, dq_weight, dq_bias = _plain_qk_part(q, dq, s["q_weight"], s)
    dk, dk_weight, dk_bias = _plain_qk_part(k, dk, s["k_weight"], s)
    out = s["d_out"].clone()
    qk = torch.cat([dq, dk], dim=2).flatten(2)
    out[..., : qk.shape[-1]] = qk.to(x.dtype)
    got = {"dqkv": out, "dq_weight": dq_weight, "dk_weight": dk_weight}
    if s["q_bias"] is not None:
        got["dq_bias"], got["dk_bias"] = dq_bias, dk_bias
    return got


def _plain_rel(s):
    """(out, softmax, q, k, v, rows in use): heads grouped as [b, key heads, query heads of each, tokens, ...]"""
    c = s["case"]
    b, n, _ = s["qkv"].shape
    h, hk, dh = c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = _heads(s["qkv"], c)
    q = q.reshape(b, n, hk, h // hk, dh).permute(0, 2, 3, 1, 4).contiguous()
    k = k.permute(0, 2, 1, 3).unsqueeze(2).contiguous()
    v = v.permute(0, 2, 1, 3).unsqueeze(2).contiguous()
    p = torch.matmul(q, k.transpose(-1, -2)) * s["scale"]
    p += s["table"][s["index"]].permute(2, 0, 1).reshape(hk, h // hk, n, n)
    rows = None
    if s["lengths"] is not None:
        rows = torch.arange(n, device="cuda") < s["lengths"][:, None]
        p.masked_fill_(~rows[:, None, None, None, :], -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    out = torch.matmul(p, v)
    if rows is not None:
        out = torch.where(rows[:, None, None, :, None], out, 0.0)
    return out, p, q, k, v, rows


def _plain_rel_forward(s):
    b, n, _ = s["qkv"].shape
    out = _plain_rel(s)[0]
    return out.permute(0, 3, 1, 2, 4).reshape(b, n, -1).to(s["qkv"].dtype)


def _plain_rel_training(s):
    c = s["case"]
    b, n, _ = s["qkv"].shape
    h, hk, dh = c["heads"], c["kv_heads"], c["head_dim"]
    out, p, q, k, v, rows = _plain_rel(s)
    do = s["d_out"].float().view(b, n, hk, h // hk, dh).permute(0, 2, 3, 1, 4)
    if rows is not None:
        do = torch.where(rows[:, None, None, :, None], do, 0.0)
        p = torch.where(rows[:, None, None, :, None], p, 0.0)
    do = do.contiguous()
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = torch.matmul(do, v.transpose(-1, -2))
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    d_bias = ds.sum(0).reshape(h, n * n)
    d_table = torch.zeros(s["table"].shape, dtype=torch.float64, device="cuda")
    d_table.index_add_(0, s["index"].flatten(), d_bias.t().double())
    dq = torch.matmul(ds, k) * s["scale"]
    dk = (torch.matmul(ds.transpose(-1, -2), q) * s["scale"]).sum(2)
    dqkv = torch.cat([dq.permute(0, 3, 1, 2, 4).reshape(b, n, h * dh), dk.permute(0, 2, 1, 3).reshape(b, n, hk * dh),
                      dv.permute(0, 2, 1, 3).reshape(b, n, hk * dh)], dim=-1).to(s["qkv"].dtype)
    out = out.permute(0, 3, 1, 2, 4).reshape(b, n, h * dh).to(s["qkv"].dtype)
    return {"out": out, "dqkv": dqkv, "d_table": d_table.float()}


# ------------------------------------------------------------------------------------------------- the package's calls
def _own(s):
    from vit_amd import ops
    c = s["case"]
    if c["op"] == "qk":
        more = dict(eps=s["eps"], rope=s["rope"], positions=s["positions"], interleaved=c["interleaved"], norm=c["norm"],
                    num_kv_heads=c["kv_heads"])
        if c["direction"] == "forward":
            return ops.qk_norm_rope(s["qkv"], c["heads"], s["q_weight"], s["k_weight"], q_bias=s["q_bias"], k_bias=s["k_bias"], **more)
        dqkv, dqw, dkw, dqb, dkb = ops.qk_norm_rope_backward(s["qkv"], s["d_out"], c["heads"], s["q_weight"], s["k_weight"], **more)
        got = {"dqkv": dqkv, "dq_weight": dqw, "dk_weight": dkw}
        if s["q_bias"] is not None:
            got["dq_bias"], got["dk_bias"] = dqb, dkb
        return got
    more = dict(lengths=s["lengths"], num_kv_heads=c["kv_heads"], scale=s["scale"])
    if c["direction"] == "forward":
        return ops.attention_rel_bias(s["qkv"], c["heads"], s["table"], s["buckets"], **more)
    out, saved = ops.attention_rel_bias_train(s["qkv"], c["heads"], s["table"], s["buckets"], **more)
    dqkv, d_table = ops.attention_rel_bias_backward(s["qkv"], out, s["d_out"], saved, c["heads"], s["table"], s["buckets"], **more)
    return {"out": out, "dqkv": dqkv, "d_table": d_table}


def run(state):
    if own:
        return _own(state)
    c = state["case"]
    if c["op"] == "qk":
        return _plain_qk_forward(state) if c["direction"] == "forward" else _plain_qk_backward(state)
    return _plain_rel_forward(state) if c["direction"] == "forward" else _plain_rel_training(state)


def work(case):
    n, size = _tokens(case), 2 if case["dtype"] == "bf16" else 4
    rows, dh = case["batch"] * n, case["head_dim"]
    packed = rows * _width(case) * size
    qk = rows * (case["heads"] + case["kv_heads"]) * dh
    if case["op"] == "qk":
        rope = (n - case["prefix"]) * case["rot_dim"] * 4
        back = case["direction"] == "backward"
        # forward: the packed rows in and out; backward: their gradient in and out, the queries and keys in
        return {"bytes": 2 * packed + (qk * size if back else 0) + rope, "flops": qk * (22 if back else 10)}
    out = rows * case["heads"] * dh * size
    product = 2 * case["batch"] * case["heads"] * dh * n * n * (0.4 if case["ragged"] else 1.0)  # mean of squared lengths
    table = _buckets(case) * case["heads"] * 4
    if case["direction"] == "forward":
        return {"bytes": packed + out + table, "flops": 2 * product}
    # forward: 2 products; backward: 5. The packed rows and the output once each way, the output's gradient in
    return {"bytes": 2 * packed + 2 * out + 2 * table, "flops": 7 * product}


# ------------------------------------------------------------------------------------------------- in 64 bits
def _exact_qk(s):
    c = s["case"]
    h, hk, dh, rot = c["heads"], c["kv_heads"], c["head_dim"], c["rot_dim"]
    x = s["qkv"].double()
    layer = s["q_bias"] is not None
    leaves = [t.double().requires_grad_() for t in (s["q_weight"], s["k_weight"])]
    leaves += [t.double().requires_grad_() for t in (s["q_bias"], s["k_bias"])] if layer else []
    back = c["direction"] == "backward"
    x.requires_grad_(back)
    z = torch.view_as_complex(s["rope"].double())  # e^(i angle)
    z = torch.cat([z, torch.ones_like(z[:1])])[s["positions"].long()].unsqueeze(-2)  # position -1: the last row, no turn

    def part(heads, w, b):
        mean = heads.mean(-1, keepdim=True) if c["norm"] == "layer" else 0.0
        y = (heads - mean) * torch.rsqrt(((heads - mean) ** 2).mean(-1, keepdim=True) + s["eps"]) * w
        y = y if b is None else y + b
        pair = y[..., :rot].unflatten(-1, (rot // 2, 2) if c["interleaved"] else (2, rot // 2))
        pair = pair if c["interleaved"] else pair.transpose(-1, -2)
        turned = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * z)
        turned = turned if c["interleaved"] else turned.transpose(-1, -2)
        return torch.cat([turned.flatten(-2), y[..., rot:]], dim=-1).flatten(2)

    with torch.set_grad_enabled(back):
        e = x.unflatten(-1, (h + 2 * hk, dh))
        out = torch.cat([part(e[:, :, :h], leaves[0], leaves[2] if layer else None),
                         part(e[:, :, h:h + hk], leaves[1], leaves[3] if layer else None), e[:, :, h + hk:].flatten(2)], dim=-1)
    if not back:
        return out.detach()
    grads = torch.autograd.grad(out, [x] + leaves, s["d_out"].double())
    return dict(zip(["dqkv", "dq_weight", "dk_weight", "dq_bias", "dk_bias"], grads))


def _exact_rel(s):
    c = s["case"]
    b, n, _ = s["qkv"].shape
    h, hk, dh = c["heads"], c["kv_heads"], c["head_dim"]
    train = c["direction"] == "training"
    x, table = s["qkv"].double().requires_grad_(train), s["table"].double().requires_grad_(train)
    used = torch.ones(b, n, dtype=torch.bool, device="cuda")
    if s["lengths"] is not None:
        used = torch.arange(n, device="cuda")[None] < s["lengths"][:, None].long()
    with torch.set_grad_enabled(train):
        e = x.unflatten(-1, (h + 2 * hk, dh)).transpose(1, 2)
        q, k, v = e[:, :h], e[:, h:h + hk].repeat_interleave(h // hk, 1), e[:, h + hk:].repeat_interleave(h // hk, 1)
        logits = (q * s["scale"]) @ k.transpose(-1, -2) + table.t()[:, s["index"]]
        logits = torch.where(used[:, None, None, :], logits, -math.inf)
        out = torch.softmax(logits, -1) @ v * used[:, None, :, None]
        out = out.transpose(1, 2).flatten(2)
    if not train:
        return out.detach()
    dx, d_table = torch.autograd.grad(out, [x, table], s["d_out"].double())
    return {"out": out.detach(), "dqkv": dx, "d_table": d_table}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_qk(s) if case["op"] == "qk" else _exact_rel(s)
