"""GPU parity of attention with a relative position bias where there are rows enough for the kernels that share staged keys or queries
between a workgroup's waves (fewer go to kernels whose waves share one tile), at the bars of test_gpu_attention_rel."""
import pytest
import torch

from vit_amd import ops, synth
from vit_amd.rel_pos import RelPosBuckets

from .test_gpu_attention_rel import BF, DEV, SLACK, U, Ref, make, plan

pytestmark = pytest.mark.gpu

CASES = [  # b, grid, prefix, h, hk, dh, mapped, with lengths
    (50, (14, 14), 1, 3, 3, 64, False, False),
    (50, (14, 14), 1, 3, 3, 64, False, True),
    (40, (1, 105), 0, 7, 7, 64, True, False),
    (30, (6, 20), 32, 8, 8, 64, False, True),
    (40, (15, 14), 5, 4, 4, 64, True, False),
    (90, (13, 10), 1, 4, 2, 64, False, True),
    (65, (9, 11), 1, 4, 2, 32, True, True),
    (90, (1, 97), 0, 4, 2, 128, False, False),
    (66, (5, 7), 5, 8, 8, 16, False, False),
    (66, (5, 7), 5, 8, 8, 48, True, True),
    (66, (1, 40), 0, 8, 8, 80, False, False),
    (90, (6, 6), 2, 8, 4, 96, False, False),
    (66, (33, 1), 0, 8, 8, 112, False, True),
    (32, (16, 16), 1, 8, 8, 80, False, False),
    (9, (24, 24), 1, 6, 6, 64, False, False),
    (4, (32, 32), 1, 8, 8, 64, False, False),
]
IDS = lambda c: "-".join(str(v).replace(" ", "") for v in c)  # noqa: E731


def setup_case(case, dtype=BF):
    b, grid, prefix, h, hk, dh, mapped, ragged = case
    pl = plan(grid, prefix, mapped)
    qkv, table = make(b, pl.seq, h, hk, dh, pl.num_buckets, dtype)
    ln = torch.tensor([(37 * i * i + 11 * i) % (pl.seq + 1) for i in range(b)], dtype=torch.int32) if ragged else None
    return pl, qkv, table, ln


def check(pl, qkv, table, ln, h, hk, dh, d_out):
    ref = Ref(qkv, table, pl.index(), h, hk, ln, dh ** -0.5, d_out)
    kw = dict(lengths=None if ln is None else ln.to(DEV), num_kv_heads=hk)
    q, t, g = qkv.to(DEV), table.to(DEV), d_out.to(DEV)
    out, lse = ops.attention_rel_bias_train(q, h, t, pl, **kw)
    assert torch.equal(out, ops.attention_rel_bias(q, h, t, pl, **kw))
    dqkv, dt = ops.attention_rel_bias_backward(q, out, g, lse, h, t, pl, **kw)
    assert torch.equal(torch.isinf(lse).cpu(), ref.empty)
    assert ((lse.cpu().double() - ref.lse)[~ref.empty].abs() <= 2.0 ** -18 * (1 + ref.lse[~ref.empty].abs())).all()
    err, tol = (out.cpu().double() - ref.out).abs(), SLACK * U * (ref.out_mag + ref.out.abs()) + 1e-30
    assert (err <= tol).all(), (err / tol).max()
    err, tol = (dqkv.cpu().double() - ref.dqkv).abs(), SLACK * (ref.dmag + U * ref.dqkv.abs()) + 2.0 ** -16 * ref.dqkv.abs().max() + 1e-30
    assert (err <= tol).all(), (err / tol).max()
    err, tol = (dt.cpu().double() - ref.dtable).abs(), 2.0 ** -16 * ref.dtable_mag + 1e-30
    assert (err <= tol).all(), (err / tol).max()
    again = ops.attention_rel_bias_backward(q, out, g, lse, h, t, pl, **kw)
    assert torch.equal(dqkv, again[0]) and torch.equal(dt, again[1])


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_forward_and_gradient(case):
    b, grid, prefix, h, hk, dh, mapped, ragged = case
    pl, qkv, table, ln = setup_case(case)
    check(pl, qkv, table, ln, h, hk, dh, synth.normal((b, pl.seq, h * dh), 4, "d_out").to(BF))


@pytest.mark.parametrize("case", [CASES[0], CASES[5], CASES[7], CASES[11], CASES[14]], ids=IDS)
def test_fp32_forward(case):
    b, grid, prefix, h, hk, dh, mapped, ragged = case
    pl, qkv, table, ln = setup_case(case, torch.float32)
    ref = Ref(qkv, table, pl.index(), h, hk, ln, dh ** -0.5)
    got = ops.attention_rel_bias(qkv.to(DEV), h, table.to(DEV), pl, lengths=None if ln is None else ln.to(DEV), num_kv_heads=hk)
    err, tol = (got.cpu().double() - ref.out).abs(), 2.0 ** -16 * ref.out_mag + 1e-30
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min, -2e30])
def test_entries_that_mask(value):
    """Offsets masked by the table, down to queries that keep no key, and prefix tokens that see only each other."""
    b, h, dh = 60, 6, 64
    pl = RelPosBuckets((1, 110), prefix=2, device=DEV)
    qkv, table = make(b, pl.seq, h, h, dh, pl.num_buckets)
    table[109:219] = value         # keys at or before the query
    table[:, 1][100:109] = value   # second head: only keys 10 or more behind the query
    table[219, 2] = value          # third head: prefix queries on grid keys
    table[220] = value             # grid queries on prefix keys
    check(pl, qkv, table, None, h, h, dh, synth.normal((b, pl.seq, h * dh), 4, "d").to(BF))


@pytest.mark.parametrize("grid,hk,dh", [((14, 14), 4, 64), ((14, 14), 2, 64), ((8, 5), 4, 80)])
def test_padding_is_never_read(grid, hk, dh):
    """NaN and infinities behind each sample's length reach nothing."""
    b, h = 150, 4
    pl = plan(grid, 1, False)
    n = pl.seq
    ln = [(37 * i * i + 11 * i) % (n + 1) for i in range(b)]
    qkv, table = make(b, n, h, hk, dh, pl.num_buckets)
    d_out = synth.normal((b, n, h * dh), 4, "d").to(BF)
    t, lens = table.to(DEV), torch.tensor(ln, dtype=torch.int32, device=DEV)

    def run(x, g):
        out, lse = ops.attention_rel_bias_train(x.to(DEV), h, t, pl, lengths=lens, num_kv_heads=hk)
        return (out, lse) + ops.attention_rel_bias_backward(x.to(DEV), out, g.to(DEV), lse, h, t, pl, lengths=lens, num_kv_heads=hk)

    clean = run(qkv, d_out)
    bad, badg = qkv.clone(), d_out.clone()
    for i, m in enumerate(ln):
        bad[i, m:] = float("nan")
        bad[i, m::2] = float("inf")
        badg[i, m:] = float("nan")
    for p, q in zip(clean, run(bad, badg)):
        assert torch.equal(p, q)
    f = [ops.attention_rel_bias(x.float().to(DEV), h, t, pl, lengths=lens, num_kv_heads=hk) for x in (qkv, bad)]
    assert torch.equal(*f)


def test_graph_replays_equal_eager():
    pl = plan((14, 14), 1, True)
    qkv, table = make(60, 197, 4, 4, 64, pl.num_buckets)
    x, t = qkv.to(DEV), table.to(DEV)
    g = torch.randn(60, 197, 256, device=DEV).to(BF)

    def step():
        out, lse = ops.attention_rel_bias_train(x, 4, t, pl)
        return (out,) + ops.attention_rel_bias_backward(x, out, g, lse, 4, t, pl)

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        x.copy_(torch.randn_like(x))
        t.copy_(torch.randn_like(t))
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(captured, step()):
            assert torch.equal(a, e)


@pytest.mark.parametrize("b,grid,h,hk,dh", [(2, (14, 14), 4, 4, 64), (150, (14, 14), 4, 4, 64), (150, (14, 14), 4, 2, 64), (150, (8, 5), 4, 4, 80)])
def test_nan_stays_in_its_sample(b, grid, h, hk, dh):
    """A sample whose last row in use is not finite: rows behind it are zeros all the same, the other samples' results keep their bits."""
    pl = plan(grid, 1, False)
    n = pl.seq
    lens = torch.full((b,), n - 5, dtype=torch.int32, device=DEV)
    qkv, table = make(b, n, h, hk, dh, pl.num_buckets)
    g, t = synth.normal((b, n, h * dh), 4, "d").to(BF).to(DEV), table.to(DEV)

    def run(x, fwd):
        out, lse = ops.attention_rel_bias_train(x, h, t, pl, lengths=lens, num_kv_heads=hk)
        if fwd is not None:  # the gradient from the same forward but for that sample
            out, lse = torch.cat([out[:1], fwd[0][1:]]), torch.cat([lse[:1], fwd[1][1:]])
        return out, lse, ops.attention_rel_bias_backward(x, out, g, lse, h, t, pl, lengths=lens, num_kv_heads=hk)[0]

    clean = run(qkv.to(DEV), None)
    bad = qkv.clone()
    bad[0, n - 6] = float("nan")
    got = run(bad.to(DEV), clean)
    for p, q in zip(clean, got):
        assert torch.equal(p[1:], q[1:])
    assert not got[0][0, n - 5:].any() and not got[2][0, n - 5:].any() and torch.isnan(got[2][0, :n - 5]).any()


@pytest.mark.parametrize("b", [3, 400])
@pytest.mark.parametrize("n,dh", [(1, 16), (2, 64), (3, 128), (13, 64), (32, 80)])
def test_few_keys(b, n, dh):
    """With one chunk of keys dQ has the roundings of dS and its own alone (bars of test_gpu_attention_rel without the part for the rounded
    out): with a handful of keys the rest would be the most of it."""
    h = 4
    pl = plan((1, n), 0, False)
    qkv, table = make(b, n, h, h, dh, pl.num_buckets)
    d_out = synth.normal((b, n, h * dh), 4, "d").to(BF)
    ref = Ref(qkv, table, pl.index(), h, h, None, dh ** -0.5, d_out)
    q, t = qkv.to(DEV), table.to(DEV)
    out, lse = ops.attention_rel_bias_train(q, h, t, pl)
    dq = ops.attention_rel_bias_backward(q, out, d_out.to(DEV), lse, h, t, pl)[0].cpu().double()[..., :h * dh]
    e = qkv.double().unflatten(-1, (3 * h, dh)).transpose(1, 2)
    do = d_out.double().unflatten(-1, (h, dh)).transpose(1, 2)
    s = e[:, :h] @ e[:, h:2 * h].transpose(-1, -2) * dh ** -0.5 + table.double()[pl.index()].permute(2, 0, 1)
    p, dp = torch.softmax(s, -1), do @ e[:, 2 * h:].transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    size = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True))  # fp32 terms: arguments of exp2 below 64 (2^-18 each)
    tol = SLACK * U * (ds.abs() @ e[:, h:2 * h].abs()) * dh ** -0.5 + 2.0 ** -16 * (size @ e[:, h:2 * h].abs()) * dh ** -0.5
    want = ref.dqkv[..., :h * dh]
    tol = tol.transpose(1, 2).flatten(2) + SLACK * U * want.abs() + 1e-30
    assert ((dq - want).abs() <= tol).all(), ((dq - want).abs() / tol).max()
