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
