"""GPU tests of single rows of attention_rel_bias that are unlike the others: rows whose scores all lie far from zero, rows of a handful of
keys in a batch of long ones, rows that are not finite.

A softmax does not change when a number is added to all scores of a row, so rows whose every key carries a large entry of the table (a
finite mask, say) have ordinary probabilities. The inputs are such that fp32 holds every score exactly (queries of zero, or products of
small integers that stay below 2^24 with the entry), so the bars of test_gpu_attention_rel hold unchanged."""
import pytest
import torch

from vit_amd import _lib, ops, synth
from vit_amd.rel_pos import RelPosBuckets

from .test_gpu_attention_rel import BF, DEV, SLACK, U, Ref, plan

pytestmark = pytest.mark.gpu

ROUTES = [  # b, tokens, h, hk, dh, with lengths: the kernels for few rows, one pass, chunks, chunks with lengths and shared keys
    (2, 70, 3, 3, 64, False),
    (1, 33, 3, 3, 128, False),
    (60, 110, 6, 6, 64, False),
    (60, 110, 6, 6, 64, True),
    (60, 110, 6, 6, 80, False),
    (120, 100, 6, 3, 64, True),
    (100, 97, 6, 3, 128, False),
]
IDS = lambda c: "-".join(str(v) for v in c)  # noqa: E731


def far_inputs(route, value, integers):
    b, n, h, hk, dh, ragged = route
    pl = RelPosBuckets((1, n), device=DEV)
    qkv = synth.normal((b, n, (h + 2 * hk) * dh), 9, "qkv")
    table = synth.normal((pl.num_buckets, h), 9, "table", std=0.8)
    if integers:
        qkv[..., :(h + hk) * dh] = qkv[..., :(h + hk) * dh].round().clamp(-2, 2)
    else:
        qkv[..., :h * dh] = 0
    table[n - 1:] = value             # keys at or before the query: the last query has no other
    table[:, 1][n - 11:n - 1] = value  # second head: only keys more than 10 behind the query are ordinary
    table[:, 2] = value               # third head: every key
    ln = torch.tensor([(37 * i * i + 11 * i) % (n + 1) for i in range(b)], dtype=torch.int32) if ragged else None
    return pl, qkv.to(BF), table, ln


def run(route, value, integers, train):
    b, n, h, hk, dh, ragged = route
    compare(*far_inputs(route, value, integers), h, hk, dh, train)


def compare(pl, qkv, table, ln, h, hk, dh, train):
    d_out = synth.normal((*qkv.shape[:2], h * dh), 4, "d_out").to(BF)
    ref = Ref(qkv, table, pl.index(), h, hk, ln, 0.125, d_out)
    kw = dict(lengths=None if ln is None else ln.to(DEV), num_kv_heads=hk, scale=0.125)
    q, t, g = qkv.to(DEV), table.to(DEV), d_out.to(DEV)
    out, lse = ops.attention_rel_bias_train(q, h, t, pl, **kw)
    if not train:
        assert torch.equal(torch.isinf(lse).cpu(), ref.empty)
        assert ((lse.cpu().double() - ref.lse)[~ref.empty].abs() <= 2.0 ** -18 * (1 + ref.lse[~ref.empty].abs())).all()
        for got in (out, ops.attention_rel_bias(q, h, t, pl, **kw)):
            err, tol = (got.cpu().double() - ref.out).abs(), SLACK * U * (ref.out_mag + ref.out.abs()) + 1e-30
            assert (err <= tol).all(), (err / tol).max()
        f = ops.attention_rel_bias(q.float(), h, t, pl, **kw)
        err, tol = (f.cpu().double() - ref.out).abs(), 2.0 ** -16 * ref.out_mag + 1e-30
        assert (err <= tol).all(), (err / tol).max()
        return
    dqkv, dt = ops.attention_rel_bias_backward(q, out, g, lse, h, t, pl, **kw)
    err, tol = (dqkv.cpu().double() - ref.dqkv).abs(), SLACK * (ref.dmag + U * ref.dqkv.abs()) + 2.0 ** -16 * ref.dqkv.abs().max() + 1e-30
    assert (err <= tol).all(), (err / tol).max()
    err, tol = (dt.cpu().double() - ref.dtable).abs(), 2.0 ** -16 * ref.dtable_mag + 1e-30
    assert (err <= tol).all(), (err / tol).max()
    again = ops.attention_rel_bias_backward(q, out, g, lse, h, t, pl, **kw)
    assert torch.equal(dqkv, again[0]) and torch.equal(dt, again[1])


VALUES = [-300.0, -1e4, -1e6, -1e9, -1e12, -9e29, 1e9, 1e20]


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("route", ROUTES, ids=IDS)
def test_far_entries_forward(route, value):
    run(route, value, False, False)


@pytest.mark.parametrize("value", [-2.0 ** 10, -2.0 ** 20, 2.0 ** 20])
@pytest.mark.parametrize("route", ROUTES, ids=IDS)
def test_far_entries_with_products_forward(route, value):
    run(route, value, True, False)


def test_far_entries_of_two_sizes():
    """A row whose keys carry two entries, both far from zero: the larger takes all, also where the running maximum meets it last."""
    n, h = 200, 2
    pl = RelPosBuckets((1, n), device=DEV)
    qkv = synth.normal((2, n, 3 * h * 64), 9, "qkv").to(BF)
    qkv[..., :h * 64] = 0
    table = torch.full((pl.num_buckets, h), -2e12)
    table[:n - 100, 0] = -1e12  # keys more than 99 behind the query
    table[n + 99:, 1] = -1e12   # keys more than 99 before it
    ref = Ref(qkv, table, pl.index(), h, h, None, 0.125)
    for b in (1, 40):  # few rows, the ring
        x = qkv[:1].repeat(b, 1, 1).to(DEV)
        got = ops.attention_rel_bias(x, h, table.to(DEV), pl)
        want = ref.out[:1]
        assert ((got.cpu().double() - want).abs() <= SLACK * U * (ref.out_mag[:1] + want.abs())).all()
    f = ops.attention_rel_bias(qkv.float().to(DEV), h, table.to(DEV), pl)
    assert ((f.cpu().double() - ref.out).abs() <= 2.0 ** -16 * ref.out_mag).all()


@pytest.mark.parametrize("value", VALUES)
@pytest.mark.parametrize("route", ROUTES, ids=IDS)
def test_far_entries_gradient(route, value):
    run(route, value, False, True)


@pytest.mark.parametrize("value", [-2.0 ** 10, -2.0 ** 20, 2.0 ** 20])
@pytest.mark.parametrize("route", ROUTES, ids=IDS)
def test_far_entries_with_products_gradient(route, value):
    run(route, value, True, True)


@pytest.mark.parametrize("value", [-2.0 ** 20, 2.0 ** 18, -2.0 ** 9])
@pytest.mark.parametrize("b,grid,prefix,h,hk,dh,mapped,ragged", [
    (2, (7, 9), 2, 4, 2, 48, True, False), (3, (14, 14), 1, 4, 4, 64, False, True), (60, (10, 11), 32, 6, 6, 64, False, False),
    (60, (10, 11), 1, 6, 6, 64, True, True), (60, (9, 11), 5, 6, 3, 80, False, True), (70, (5, 13), 1, 8, 4, 128, True, False),
    (1, (24, 24), 1, 4, 4, 64, False, False), (60, (3, 3), 2, 8, 8, 32, False, True)])
def test_far_tables_on_a_grid(b, grid, prefix, h, hk, dh, mapped, ragged, value):
    """Every entry far from zero, each at its own distance, prefix tokens' entries among them; products of small integers."""
    pl = plan(grid, prefix, mapped)
    n = pl.seq
    qkv = synth.normal((b, n, (h + 2 * hk) * dh), 9, "qkv")
    qkv[..., :(h + hk) * dh] = qkv[..., :(h + hk) * dh].round().clamp(-2, 2)
    table = value + synth.normal((pl.num_buckets, h), 9, "table", std=2.0).round()
    ln = torch.tensor([(37 * i * i + 11 * i) % (n + 1) for i in range(b)], dtype=torch.int32) if ragged else None
    compare(pl, qkv.to(BF), table, ln, h, hk, dh, True)
    compare(pl, qkv.to(BF), table, ln, h, hk, dh, False)


@pytest.mark.parametrize("b,n,h,hk,dh", [(100, 197, 4, 4, 64), (100, 97, 4, 4, 64), (2, 197, 4, 4, 64), (100, 197, 4, 2, 64)])
def test_few_keys_of_a_ragged_batch(b, n, h, hk, dh):
    """Samples of at most one chunk of keys have the dQ that whole sequences of their length have, whatever the batch is padded to: the
    roundings of dS and its own alone (bars of test_few_keys)."""
    pl = RelPosBuckets((1, n), device=DEV)
    ln = torch.tensor([(1, 2, 3, 13, 32)[i % 5] for i in range(b)], dtype=torch.int32)
    qkv = synth.normal((b, n, (h + 2 * hk) * dh), 9, "qkv").to(BF)
    table = synth.normal((pl.num_buckets, h), 9, "table", std=0.8)
    d_out = synth.normal((b, n, h * dh), 4, "d_out").to(BF)
    q, t, kw = qkv.to(DEV), table.to(DEV), dict(lengths=ln.to(DEV), num_kv_heads=hk)
    out, lse = ops.attention_rel_bias_train(q, h, t, pl, **kw)
    dq = ops.attention_rel_bias_backward(q, out, d_out.to(DEV), lse, h, t, pl, **kw)[0].cpu().double()[..., :h * dh]
    for i in range(b):
        m = int(ln[i])
        e = qkv[i, :m].double().unflatten(-1, (h + 2 * hk, dh)).transpose(0, 1)
        k, v = (x.repeat_interleave(h // hk, 0) for x in (e[h:h + hk], e[h + hk:]))
        do = d_out[i, :m].double().unflatten(-1, (h, dh)).transpose(0, 1)
        s = e[:h] @ k.transpose(-1, -2) * dh ** -0.5 + table.double()[pl.index()[:m, :m]].permute(2, 0, 1)
        p, dp = torch.softmax(s, -1), do @ v.transpose(-1, -2)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        size = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True))
        want = (ds @ k * dh ** -0.5).transpose(0, 1).flatten(1)
        tol = (SLACK * U * ds.abs() + 2.0 ** -16 * size) @ k.abs() * dh ** -0.5
        tol = tol.transpose(0, 1).flatten(1) + SLACK * U * want.abs() + 1e-30
        assert ((dq[i, :m] - want).abs() <= tol).all(), (m, ((dq[i, :m] - want).abs() / tol).max())
        assert not dq[i, m:].any()


@pytest.mark.parametrize("what", ["q", "v", "d_out"])
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("b,grid,prefix,h,hk,dh", [(2, (1, 197), 0, 4, 4, 64), (150, (14, 14), 1, 4, 4, 64), (150, (1, 101), 0, 4, 2, 80), (2, (17, 18), 2, 2, 2, 128)])
def test_nan_of_a_last_row_stays_with_its_pairs(b, grid, prefix, h, hk, dh, ragged, what):
    """A last row in use that is not finite: of d_table exactly the entries of its pairs are not finite (with values that are not, all pairs
    of its sample), those that only rows and keys behind it would reach are."""
    pl = RelPosBuckets(grid, prefix=prefix, device=DEV)
    n = pl.seq
    m = n - 5 if ragged else n
    kw = dict(lengths=torch.full((b,), m, dtype=torch.int32, device=DEV) if ragged else None, num_kv_heads=hk)
    qkv = synth.normal((b, n, (h + 2 * hk) * dh), 9, "qkv").to(BF)
    table = synth.normal((pl.num_buckets, h), 9, "table", std=0.8).to(DEV)
    d_out = synth.normal((b, n, h * dh), 4, "d_out").to(BF)
    if what == "q":
        qkv[0, m - 1, :h * dh] = float("nan")
    elif what == "v":
        qkv[0, m - 1, (h + hk) * dh:] = float("nan")
    else:
        d_out[0, m - 1] = float("nan")
    x = qkv.to(DEV)
    out, lse = ops.attention_rel_bias_train(x, h, table, pl, **kw)
    dt = ops.attention_rel_bias_backward(x, out, d_out.to(DEV), lse, h, table, pl, **kw)[1]
    index = pl.index()
    hit = torch.zeros(pl.num_buckets, dtype=torch.bool)
    hit[(index[:m, :m] if what == "v" else index[m - 1, :m]).flatten()] = True
    assert torch.equal(torch.isfinite(dt).cpu(), ~hit[:, None].expand(-1, h))


@pytest.mark.parametrize("grid", [(1, 15872), (89, 89)])
def test_refused_gradient_writes_nothing(grid):
    """One size past the limit with d_table: refused, and neither dqkv nor the workspace is touched. Without d_table the call is taken."""
    pl = RelPosBuckets(grid, device=DEV)
    n, lib, c = pl.seq, _lib.load(), pl._c()
    x = synth.normal((1, n, 48), 1, "x").to(BF).to(DEV)
    t = torch.zeros(pl.num_buckets, 1, device=DEV)
    out, lse = ops.attention_rel_bias_train(x, 1, t, pl)
    need = lib.vit_attention_rel_bwd_workspace_bytes(c, 1, 1, 16)
    ws, dqkv, dt = torch.full((need,), 77, dtype=torch.uint8, device=DEV), torch.full_like(x, 7), torch.full_like(t, 7)
    args = [x.data_ptr(), t.data_ptr(), None, out.data_ptr(), out.data_ptr(), lse.data_ptr(), dqkv.data_ptr()]
    rest = [ws.data_ptr(), need, 1, 1, 1, 16, 0.25, torch.cuda.current_stream().cuda_stream]
    assert lib.vit_attention_rel_bwd(c, *args, dt.data_ptr(), *rest) == -1
    torch.cuda.synchronize()
    assert (ws == 77).all() and (dqkv == 7).all() and (dt == 7).all()
    assert lib.vit_attention_rel_bwd(c, *args, None, *rest) == 0
    torch.cuda.synchronize()
    assert torch.isfinite(dqkv.float()).all() and not (dqkv == 7).all()


@pytest.mark.parametrize("b,n,h,hk,dh", [(60, 110, 6, 6, 64), (2, 70, 3, 3, 64), (100, 97, 6, 3, 128)])
def test_far_rows_come_and_go_in_a_graph(b, n, h, hk, dh):
    """A captured step whose table gets and loses entries far from zero between its replays, against the eager call each time."""
    pl = RelPosBuckets((1, n), device=DEV)
    x = synth.normal((b, n, (h + 2 * hk) * dh), 9, "qkv").to(BF).to(DEV)
    t = synth.normal((pl.num_buckets, h), 9, "table", std=0.8).to(DEV)
    g = synth.normal((b, n, h * dh), 4, "d_out").to(BF).to(DEV)

    def step():
        out, lse = ops.attention_rel_bias_train(x, h, t, pl, num_kv_heads=hk)
        return (out, lse) + ops.attention_rel_bias_backward(x, out, g, lse, h, t, pl, num_kv_heads=hk)

    step()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    ordinary = t.clone()
    for value in (None, -1e9, None, 1e12, -400.0, None):
        t.copy_(ordinary)
        if value is not None:
            t[n - 1:, 1] = value
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(captured, step()):
            assert torch.equal(a, e) and torch.isfinite(e.float()).all()
