"""GPU parity tests of the head norm + rotation and its gradient against plain torch in 64 bits on the same inputs.

Bars, from the arithmetic. fp32 values: every step rounds by 2^-24, and a value passes fewer than 40 of them (a sum of 128
squares in a tree, the square root, the weight, the turn), each relative to the row's largest term
``r max|x| max|w| + max|b|``. bf16 outputs: that, and one rounding of the result by at most 2^-8 of it. Parameter gradients:
fewer than 128 rounded additions deep at these sizes, relative to the sum of the terms' magnitudes."""
import pytest
import torch

from vit_amd import ops, synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U32 = 2.0 ** -24


def make(b, n, h, hk, dh, dtype, seed=5, mean=0.3):
    x = synth.normal((b, n, (h + 2 * hk) * dh), seed, "qkv", std=1.4, mean=mean).to(dtype)
    w = [1 + synth.normal((dh,), seed, f"w{i}", std=0.3) for i in range(2)]
    bias = [synth.normal((dh,), seed, f"b{i}", std=0.2) for i in range(2)]
    return x, w, bias


def reference(x, w, bias, h, hk, eps, rope, pos, interleaved, norm, g=None):
    """(out, grads) in 64 bits by autograd; the turn is a complex product."""
    x = x.double().requires_grad_(True)
    w = [v.double().requires_grad_(True) for v in w]
    bias = [v.double().requires_grad_(True) for v in bias]
    dh = x.shape[-1] // (h + 2 * hk)
    e = x.unflatten(-1, (h + 2 * hk, dh))

    def part(t, wt, bt):
        if norm == "layer":
            t = t - t.mean(-1, keepdim=True)
        y = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + eps) * wt
        if norm == "layer":
            y = y + bt
        if rope is None:
            return y
        p, rot = rope.shape[0], 2 * rope.shape[1]
        z = torch.cat([torch.view_as_complex(rope.double()), torch.ones(1, rot // 2, dtype=torch.complex128)])
        at = torch.where((pos >= 0) & (pos < p), pos, p).long()
        z = z[at].unsqueeze(-2)
        a, c = (y[..., 0:rot:2], y[..., 1:rot:2]) if interleaved else (y[..., :rot // 2], y[..., rot // 2:rot])
        v = torch.complex(a, c) * z
        turned = torch.stack([v.real, v.imag], -1).flatten(-2) if interleaved else torch.cat([v.real, v.imag], -1)
        return torch.cat([turned, y[..., rot:]], -1)

    out = torch.cat([part(e[..., :h, :], w[0], bias[0]), part(e[..., h:h + hk, :], w[1], bias[1]), e[..., h + hk:, :]], -2).flatten(-2)
    grads = None
    if g is not None:
        grads = torch.autograd.grad(out, [x] + w + bias, g.double(), allow_unused=True)
    return out.detach(), grads


def head_scale(x, h, hk, eps, norm):
    """r max|x| of every head, broadcast over its values"""
    e = x.double().unflatten(-1, (h + 2 * hk, -1))
    t = e - e.mean(-1, keepdim=True) if norm == "layer" else e
    r = torch.rsqrt((t * t).mean(-1, keepdim=True) + eps)
    return r, r * e.abs().amax(-1, keepdim=True)


CASES = [  # b, n, h, hk, dh, rot, interleaved, norm, dtype, positions
    (1, 1, 1, 1, 16, 16, False, "rms", torch.bfloat16, None),
    (2, 5, 3, 3, 32, 16, True, "rms", torch.float32, "token"),
    (3, 197, 12, 12, 64, 64, False, "rms", torch.bfloat16, "shared"),
    (2, 50, 12, 4, 96, 96, False, "layer", torch.bfloat16, "token"),
    (1, 33, 16, 16, 80, 64, True, "layer", torch.float32, "shared"),
    (2, 17, 5, 1, 128, 128, False, "layer", torch.float32, "token"),
    (4, 9, 7, 7, 48, 48, True, "layer", torch.bfloat16, None),
    (2, 7, 4, 2, 112, 32, False, "rms", torch.float32, "shared"),
    (2, 40, 6, 3, 64, 0, False, "rms", torch.bfloat16, None),
]


def setup_case(case):
    b, n, h, hk, dh, rot, il, norm, dtype, places = case
    x, w, bias = make(b, n, h, hk, dh, dtype)
    rope = ops.rope_table((1, n + 3), rot, device="cpu") if rot else None
    pos, given = torch.arange(n), None
    if places == "shared":  # leading tokens unturned, one position past the table
        given = torch.arange(-2, n - 2, dtype=torch.int32)
        given[-1] = n + 3
        pos = given
    elif places == "token":
        given = torch.randint(-1, n + 4, (b, n), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
        pos = given
    return x, w, bias, rope, pos, given


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v).replace("torch.", "") for v in c))
def test_forward_and_gradient(case):
    b, n, h, hk, dh, rot, il, norm, dtype, places = case
    eps = 1e-6
    x, w, bias, rope, pos, given = setup_case(case)
    g = synth.normal(tuple(x.shape), 6, "g").to(dtype)
    layer = norm == "layer"
    ref, grads = reference(x, w, bias, h, hk, eps, rope, pos, il, norm, g)
    dev = lambda t: None if t is None else t.to(DEV)  # noqa: E731
    kw = dict(eps=eps, rope=dev(rope), positions=dev(given), interleaved=il, norm=norm, num_kv_heads=hk)
    got = ops.qk_norm_rope(dev(x), h, dev(w[0]), dev(w[1]), *([dev(bias[0]), dev(bias[1])] if layer else []), **kw)
    assert got.dtype == dtype and got.shape == x.shape
    qk = (h + hk) * dh
    assert torch.equal(got[..., qk:].cpu(), x[..., qk:])
    r, s = head_scale(x, h, hk, eps, norm)
    wmax, bmax = max(v.abs().max() for v in w), max(v.abs().max() for v in bias)
    out_round = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
    tol = out_round * ref.abs() + (40 * U32 * (s * wmax + bmax) * torch.ones(dh)).flatten(-2)
    err = (got.cpu().double() - ref).abs()
    assert (err <= tol).all(), (err / tol).max()

    res = ops.qk_norm_rope_backward(dev(x), dev(g), h, dev(w[0]), dev(w[1]), **kw)
    dx = res[0].cpu()
    assert torch.equal(dx[..., qk:], g[..., qk:])
    xh = s[..., :h + hk, :]
    gmax = g.double().unflatten(-1, (h + 2 * hk, dh)).abs().amax(-1, keepdim=True)[..., :h + hk, :] * 2 * wmax
    tol = out_round * grads[0].abs()[..., :qk] + (64 * U32 * r[..., :h + hk, :] * gmax * (1 + xh * xh) * torch.ones(dh)).flatten(-2)
    err = (dx.double() - grads[0])[..., :qk].abs()
    assert (err <= tol).all(), (err / tol).max()
    terms_w = (gmax / wmax * xh).sum() * torch.ones(dh)  # bounds sum |t xh| of any column
    for k in range(4 if layer else 2):
        ref_k = grads[1 + k]
        tol = 128 * U32 * (terms_w if k < 2 else gmax.sum() / wmax)
        assert ((res[1 + k].cpu().double() - ref_k).abs() <= tol).all(), k
    if not layer:
        assert res[3] is None and res[4] is None


def test_in_place_equals_new_tensor():
    case = CASES[3]
    b, n, h, hk, dh, rot, il, norm, dtype, places = case
    x, w, bias, rope, pos, given = setup_case(case)
    kw = dict(rope=rope.to(DEV), positions=given.to(DEV), norm=norm, num_kv_heads=hk)
    wd, bd = [v.to(DEV) for v in w], [v.to(DEV) for v in bias]
    a = ops.qk_norm_rope(x.to(DEV), h, *wd, *bd, **kw)
    y = x.to(DEV)
    assert ops.qk_norm_rope(y, h, *wd, *bd, out=y, **kw) is y and torch.equal(a, y)
    g = synth.normal(tuple(x.shape), 6, "g").to(dtype).to(DEV)
    r1 = ops.qk_norm_rope_backward(x.to(DEV), g, h, *wd, **kw)
    r2 = ops.qk_norm_rope_backward(x.to(DEV), g, h, *wd, out=g, **kw)
    assert r2[0] is g and all(torch.equal(p, q) for p, q in zip(r1, r2))


def test_big_batch_is_reproducible_and_exact_in_the_sums():
    """More tokens than the launch has waves: sums of 50 thousand rows, the same bits twice, against 64 bits."""
    b, n, h, hk, dh = 64, 197, 12, 12, 64
    x, w, _ = make(b, n, h, hk, dh, torch.bfloat16)
    g = synth.normal(tuple(x.shape), 6, "g").to(torch.bfloat16)
    rope = ops.rope_table((14, 14), dh, device=DEV)
    pos = torch.arange(-1, 196, dtype=torch.int32, device=DEV)
    args = (x.to(DEV), g.to(DEV), h, w[0].to(DEV), w[1].to(DEV))
    r1 = ops.qk_norm_rope_backward(*args, rope=rope, positions=pos)
    r2 = ops.qk_norm_rope_backward(*args, rope=rope, positions=pos)
    assert all(torch.equal(p, q) for p, q in zip(r1[:3], r2[:3]))
    _, grads = reference(x, w, [torch.zeros(dh)] * 2, h, hk, 1e-6, rope.cpu(), pos.cpu(), False, "rms", g)
    for k in (1, 2):
        # random signs: rounding errors add as a random walk, far below 2e-5 of the result's norm
        assert ((r1[k].cpu().double() - grads[k]).norm() / grads[k].norm()) < 2e-6


def test_noncontiguous_and_constant_rows():
    """A strided qkv is taken as its values; a head of equal values has variance 0 (r = eps^-1/2) and stays finite."""
    b, n, h, dh = 2, 6, 2, 32
    x, w, bias = make(b, n, h, h, dh, torch.float32)
    x[0, 0, :dh] = 2.5
    x[0, 1] = 0.0
    wide = torch.zeros(b, n, 2 * x.shape[-1])
    wide[..., ::2] = x
    kw = dict(norm="layer", eps=1e-5)
    a = ops.qk_norm_rope(wide.to(DEV)[..., ::2], h, w[0].to(DEV), w[1].to(DEV), bias[0].to(DEV), bias[1].to(DEV), **kw)
    ref, _ = reference(x, w, bias, h, h, 1e-5, None, None, False, "layer")
    assert torch.isfinite(a).all()
    # eps^-1/2 = 316 times the rounding of 2.5 and of its mean: 316 * 40 * 2^-24 * 2.5
    assert ((a.cpu().double() - ref).abs().max()) < 316 * 40 * U32 * 2.5 + 1e-5


def test_graph_replays_equal_eager():
    b, n, h, dh = 3, 50, 4, 64
    x, w, _ = make(b, n, h, h, dh, torch.bfloat16)
    x, w = x.to(DEV), [v.to(DEV) for v in w]
    g = torch.randn_like(x)
    rope = ops.rope_table((5, 10), dh, device=DEV)

    def step():
        y = ops.qk_norm_rope(x, h, *w, rope=rope)
        return (y,) + ops.qk_norm_rope_backward(x, g, h, *w, rope=rope)[:3]

    step()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        x.copy_(torch.randn_like(x) + k)
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(captured, step()):
            assert torch.equal(a, e)


def test_other_stream():
    b, n, h, dh = 8, 300, 8, 64
    x, w, _ = make(b, n, h, h, dh, torch.bfloat16)
    x, w = x.to(DEV), [v.to(DEV) for v in w]
    ref = ops.qk_norm_rope(x, h, *w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = ops.qk_norm_rope(x * 1.0, h, *w)
    s.synchronize()
    assert torch.equal(got, ref)


def test_refusals_on_device():
    x, w, bias = make(1, 4, 2, 2, 32, torch.bfloat16)
    x, w, bias = x.to(DEV), [v.to(DEV) for v in w], [v.to(DEV) for v in bias]
    rope = ops.rope_table((1, 4), 32, device=DEV)
    for kw in (dict(norm="batch"), dict(positions=torch.zeros(4, dtype=torch.int32, device=DEV)), dict(rope=rope[..., 0]),
               dict(rope=rope, positions=torch.zeros(3, dtype=torch.int32, device=DEV)),
               dict(rope=rope, positions=torch.zeros(4, dtype=torch.int64, device=DEV)), dict(num_kv_heads=3),
               dict(rope=rope, positions=torch.zeros(4, dtype=torch.int32)), dict(q_bias=bias[0])):
        with pytest.raises(ValueError):
            ops.qk_norm_rope(x, 2, *w, **kw)
    from vit_amd._lib import VitError
    for kw in (dict(eps=0.0), dict(eps=float("nan")), dict(rope=ops.rope_table((1, 4), 24, device=DEV))):
        with pytest.raises(VitError):
            ops.qk_norm_rope(x, 2, *w, **kw)
    with pytest.raises(TypeError):
        ops.qk_norm_rope(x.half(), 2, *w)
    with pytest.raises(ValueError):
        ops.qk_norm_rope(x, 2, w[0][:16], w[1])
    flat = torch.zeros(x.numel() + 64, dtype=x.dtype, device=DEV)
    with pytest.raises(VitError, match="overlap"):
        ops.qk_norm_rope(flat[:x.numel()].view(x.shape), 2, *w, out=flat[64:].view(x.shape))
    with pytest.raises(VitError, match="aligned"):
        ops.qk_norm_rope(flat[1:1 + x.numel()].view(x.shape), 2, *w)
