"""GPU tests: what is not finite in the gradient of qk_norm_rope stays with the heads that it belongs to."""
import pytest
import torch

from vit_amd import ops, synth

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("where", ["query", "key"])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype,h,hk,dh", [(torch.bfloat16, 12, 12, 64), (torch.bfloat16, 5, 1, 96), (torch.float32, 4, 2, 80), (torch.float32, 2, 2, 16)])
def test_parameter_gradients_of_the_other_heads(dtype, h, hk, dh, norm, where, bad):
    """One value of a query head's gradient that is not finite leaves the keys' parameter gradients as they were, bit for bit, and the
    reverse."""
    b, n = 3, 37
    x = synth.normal((b, n, (h + 2 * hk) * dh), 1, "x").to(dtype).to(DEV)
    g = synth.normal((b, n, (h + 2 * hk) * dh), 1, "g").to(dtype).to(DEV)
    qw, kw = (1 + synth.normal((dh,), 1, k, std=0.2).to(DEV) for k in ("qw", "kw"))
    rope = ops.rope_table((1, n), 16, device=DEV)

    def grads(g):
        d = ops.qk_norm_rope_backward(x, g, h, qw, kw, rope=rope, norm=norm, num_kv_heads=hk)
        return (d[1], d[3]), (d[2], d[4])

    clean = grads(g)
    worse = g.clone()
    worse[1, 5, 3 if where == "query" else h * dh + 3] = bad
    got = grads(worse)
    hit, kept = (0, 1) if where == "query" else (1, 0)
    for a, c in zip(got[kept], clean[kept]):
        assert (a is None and c is None) or torch.equal(a, c)
    for a in got[hit]:
        assert a is None or not torch.isfinite(a).all()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", ["rms", "layer"])
@pytest.mark.parametrize("dtype,dh,rot", [(torch.bfloat16, 64, 64), (torch.bfloat16, 96, 32), (torch.float32, 80, 64), (torch.float32, 32, 16)])
def test_values_that_are_not_turned_stay_apart(dtype, dh, rot, norm, interleaved):
    """A gradient value that is not finite in a token without a rotation, or behind the rotated part of a head, reaches the parameter sums
    of its own place alone; in a turned pair those of both of its places."""
    h, n = 4, 20
    x = synth.normal((1, n, 3 * h * dh), 1, "x").to(dtype).to(DEV)
    g = synth.normal((1, n, 3 * h * dh), 1, "g").to(dtype).to(DEV)
    w = torch.ones(dh, device=DEV)
    rope = ops.rope_table((1, n), rot, device=DEV)
    pos = torch.arange(-2, n - 2, dtype=torch.int32, device=DEV)  # two tokens without a rotation

    def hit(token, place):
        bad = g.clone()
        bad[0, token, place] = float("nan")
        d = ops.qk_norm_rope_backward(x, bad, h, w, w, rope=rope, positions=pos, interleaved=interleaved, norm=norm)
        sets = [set(torch.isnan(v).nonzero().flatten().tolist()) for v in (d[1], d[3]) if v is not None]
        assert torch.isfinite(d[2]).all() and all(s == sets[0] for s in sets)
        return sets[0]

    for place in (0, 5, rot // 2, rot - 1):
        assert hit(1, place) == {place}
        pair = place ^ 1 if interleaved else (place + rot // 2) % rot
        assert hit(7, place) == {place, pair}
    if rot < dh:
        for place in (rot, rot + 5, dh - 1):
            assert hit(7, place) == {place} and hit(0, place) == {place}
