"""GPU tests of the ends of what qk_norm_rope and attention_rel_bias take: the longest sequences and largest grids, tensors past 2^31
elements, views, other streams, tables with entries that no offset names."""
import pytest
import torch

from vit_amd import _lib, ops, synth
from vit_amd._lib import VitError
from vit_amd.rel_pos import RelPosBuckets

from .test_gpu_attention_rel import BF, DEV, SLACK, U, Ref, make, plan

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("grid,prefix,dh", [((1, 15000), 0, 16), ((88, 88), 1, 16), ((1, 5000), 0, 128)])
def test_longest(grid, prefix, dh):
    """Some rows of the output and of dQ, some of dK and dV, and some entries of the table's gradient, from their formulas in 64 bits
    (rounded bars as in test_gpu_attention_rel; scores within +-8 here, arguments of exp2 below 16: 2^-19)."""
    h, scale = 1, dh ** -0.5
    pl = RelPosBuckets(grid, prefix=prefix, device=DEV)
    n = pl.seq
    qkv, table = make(1, n, h, h, dh, pl.num_buckets)
    d_out = synth.normal((1, n, dh), 4, "d").to(BF)
    x, t, g = qkv.to(DEV), table.to(DEV), d_out.to(DEV)
    out, lse = ops.attention_rel_bias_train(x, h, t, pl)
    dqkv, dt = ops.attention_rel_bias_backward(x, out, g, lse, h, t, pl)
    q, k, v = (e.to(DEV).double() for e in qkv[0].split(dh, dim=-1))
    go, tab = g[0].double(), t[:, 0].double()
    cells = torch.arange(n - prefix, device=DEV)
    gh, gw = grid

    def bias(rows, cols):  # [rows, cols] from the definition
        def place(i):
            p = (i - prefix).clamp(min=0)
            return p // gw, p % gw
        (yi, xi), (yj, xj) = place(rows[:, None]), place(cols[None])
        at = (yi - yj + gh - 1) * (2 * gw - 1) + xi - xj + gw - 1
        pi, pj = rows[:, None] < prefix, cols[None] < prefix
        at = torch.where(pi & pj, pl.offsets + 2, torch.where(pj, pl.offsets + 1, torch.where(pi, pl.offsets, at)))
        return tab[at]

    every = torch.arange(n, device=DEV)
    del cells
    some = torch.tensor(sorted({0, 1, prefix, 31, 32, 257, n // 2, n - 33, n - 2, n - 1}), device=DEV)
    s = q[some] @ k.T * scale + bias(some, every)
    p = torch.softmax(s, -1)
    o = p @ v
    assert ((out[0, some].double() - o).abs() <= SLACK * U * (p @ v.abs() + o.abs())).all()
    want = torch.logsumexp(s, -1) / torch.log(torch.tensor(2.0, dtype=torch.float64, device=DEV))
    assert ((lse[0, 0, some].double() - want).abs() <= 2.0 ** -18 * (1 + want.abs())).all()
    # every row's statistics, blockwise: lse and delta
    full, delta = torch.empty(n, dtype=torch.float64, device=DEV), torch.empty(n, dtype=torch.float64, device=DEV)
    for i in range(0, n, 1024):
        r = every[i:i + 1024]
        si = q[r] @ k.T * scale + bias(r, every)
        full[r] = torch.logsumexp(si, -1)
        delta[r] = (torch.exp(si - full[r, None]) * (go[r] @ v.T)).sum(-1)
    dp = go[some] @ v.T
    ds = p * (dp - delta[some, None])
    dq = ds @ k * scale
    mag = ds.abs() * U + p * (2 * U * (p @ v.abs() * go[some].abs()).sum(-1, keepdim=True))
    assert ((dqkv[0, some, :dh].double() - dq).abs() <= SLACK * (mag @ k.abs() * scale + U * dq.abs()) + 2.0 ** -16 * dq.abs().max()).all()
    s = q @ k[some].T * scale + bias(every, some)  # all queries on some keys
    p = torch.exp(s - full[:, None])
    ds = p * (go @ v[some].T - delta[:, None])
    dk, dv = ds.T @ q * scale, p.T @ go
    assert ((dqkv[0, some, dh:2 * dh].double() - dk).abs() <= SLACK * U * (ds.abs().T @ q.abs() * scale + dk.abs()) + 2.0 ** -16 * dk.abs().max()).all()
    assert ((dqkv[0, some, 2 * dh:].double() - dv).abs() <= SLACK * U * (p.T @ go.abs() + dv.abs()) + 2.0 ** -16 * dv.abs().max()).all()
    if gh == 1:  # an offset's pairs are a diagonal
        for off in (0, 1, -1, 31, -32, 1000, -n // 2, n - 1, -(n - 1)):
            i = every[max(off, 0):n + min(off, 0)]
            j = i - off
            pij = torch.exp((q[i] * k[j]).sum(-1) * scale + tab[off + n - 1] - full[i])
            dpij = (go[i] * v[j]).sum(-1)
            # (each row's delta is a sum over the row: its magnitude in fp32 terms)
            tol = 2.0 ** -16 * (pij * (dpij.abs() + go[i].abs() @ v.abs().amax(0))).sum() + 1e-30
            assert (dt[off + n - 1, 0].double() - (pij * (dpij - delta[i])).sum()).abs() <= tol, off
    # the softmax's gradient sums to zero over each row, so the table's does
    assert dt.double().sum().abs() <= 2.0 ** -16 * n * 8


def test_limits():
    def call(grid, train):
        pl = RelPosBuckets(grid, device=DEV)
        x = torch.zeros(1, pl.seq, 48, device=DEV, dtype=BF)
        t = torch.zeros(pl.num_buckets, 1, device=DEV)
        if not train:
            return ops.attention_rel_bias(x, 1, t, pl)
        out = torch.zeros(1, pl.seq, 16, device=DEV, dtype=BF)
        return ops.attention_rel_bias_backward(x, out, out, torch.zeros(1, 1, pl.seq, device=DEV), 1, t, pl)

    call((1, 15871), True)
    call((1, 16127), False)
    pl = RelPosBuckets((1, 16127), device=DEV)
    x = synth.normal((1, pl.seq, 384), 1, "x").to(DEV)
    out = ops.attention_rel_bias(x, 1, torch.zeros(pl.num_buckets, 1, device=DEV), pl, lengths=torch.tensor([5], dtype=torch.int32, device=DEV))
    want = torch.softmax(x[0, :5, :128] @ x[0, :5, 128:256].T * 128 ** -0.5, -1) @ x[0, :5, 256:]
    assert (out[0, :5] - want).abs().max() < 2.0 ** -14 and not out[0, 5:].any()
    for grid in ((1, 16200), (128, 128)):
        with pytest.raises(VitError, match="bias entries"):
            call(grid, False)
        with pytest.raises(VitError, match="bias entries"):
            call(grid, True)


def test_past_32_bits():
    """The last samples of tensors of more than 2^31 elements, against calls on those samples alone."""
    b, n, h, dh, m = 5000, 197, 12, 64, 60
    pl = plan((14, 14), 1, False)
    gen = torch.Generator(device=DEV).manual_seed(3)
    x = torch.empty(b, n, 3 * h * dh, device=DEV, dtype=BF).normal_(generator=gen)
    assert x.numel() > 2 ** 31
    w = 1 + 0.1 * torch.randn(dh, device=DEV, generator=gen)
    rope, pos = ops.rope_table((14, 14), dh, device=DEV), torch.arange(-1, 196, dtype=torch.int32, device=DEV)
    y = ops.qk_norm_rope(x, h, w, w, rope=rope, positions=pos)
    assert torch.equal(y[-m:], ops.qk_norm_rope(x[-m:].contiguous(), h, w, w, rope=rope, positions=pos))
    dx = ops.qk_norm_rope_backward(x, y, h, w, w, rope=rope, positions=pos)[0]
    assert torch.equal(dx[-m:], ops.qk_norm_rope_backward(x[-m:].contiguous(), y[-m:].contiguous(), h, w, w, rope=rope, positions=pos)[0])
    del dx
    t = torch.randn(pl.num_buckets, h, device=DEV, generator=gen)
    out, lse = ops.attention_rel_bias_train(y, h, t, pl)
    ys = y[-m:].contiguous()
    outs, lses = ops.attention_rel_bias_train(ys, h, t, pl)
    assert torch.equal(out[-m:], outs) and torch.equal(lse[-m:], lses)
    g = torch.randn_like(out)
    d, dt = ops.attention_rel_bias_backward(y, out, g, lse, h, t, pl)
    ds, _ = ops.attention_rel_bias_backward(ys, outs, g[-m:].contiguous(), lses, h, t, pl)
    assert torch.equal(d[-m:], ds)
    assert torch.isfinite(dt).all() and dt.double().sum(0).abs().max() < 2.0 ** -16 * b * n


def test_views_and_strides():
    """Arguments that are views of something larger give what their copies give."""
    pl = plan((6, 6), 1, True)
    h, dh = 4, 64
    wide = synth.normal((3, 40, 3 * h * dh + 64), 1, "w").to(BF).to(DEV)
    x = wide[:, :37, 32:-32]
    t = synth.normal((h, pl.num_buckets + 5), 1, "t").to(DEV)[:, 2:-3].t()
    lens = torch.tensor([[37, 1], [30, 1], [2, 1]], dtype=torch.int32, device=DEV)[:, 0]
    g = synth.normal((3, 37, 2 * h * dh), 1, "g").to(BF).to(DEV)[..., ::2]
    assert not any(v.is_contiguous() for v in (x, t, lens, g))

    def run(*a):
        x, t, lens, g = a
        out, lse = ops.attention_rel_bias_train(x, h, t, pl, lengths=lens)
        return (out, lse) + ops.attention_rel_bias_backward(x, out, g, lse, h, t, pl, lengths=lens)

    for p, q in zip(run(x, t, lens, g), run(*(v.contiguous() for v in (x, t, lens, g)))):
        assert torch.equal(p, q)


def test_entries_without_an_offset():
    """More buckets than offset indices, and buckets that the map does not name: their gradient is zero."""
    h, dh = 2, 32
    qkv, _ = make(2, 12, h, h, dh, 1)
    g = synth.normal((2, 12, h * dh), 1, "g").to(BF)
    plain, more = RelPosBuckets((3, 4), device=DEV), RelPosBuckets((3, 4), num_buckets=50, device=DEV)
    table = synth.normal((50, h), 1, "t").to(DEV)
    x, gd = qkv.to(DEV), g.to(DEV)
    res = []
    for pl, t in ((plain, table[:35].contiguous()), (more, table)):
        out, lse = ops.attention_rel_bias_train(x, h, t, pl)
        res.append((out,) + ops.attention_rel_bias_backward(x, out, gd, lse, h, t, pl))
    assert torch.equal(res[0][0], res[1][0]) and torch.equal(res[0][1], res[1][1])
    assert torch.equal(res[0][2], res[1][2][:35]) and not res[1][2][35:].any()
    mapped = RelPosBuckets((3, 4), bucket_of=[2 * (i % 5) for i in range(35)], num_buckets=16, device=DEV)
    t = table[:16].contiguous()
    out, lse = ops.attention_rel_bias_train(x, h, t, mapped)
    dt = ops.attention_rel_bias_backward(x, out, gd, lse, h, t, mapped)[1]
    assert not dt[1::2].any() and not dt[10:].any() and dt[0:10:2].all()


def test_another_stream():
    """A plan made on one stream and calls on another, behind that stream's own work."""
    h, dh = 4, 64
    qkv, _ = make(2, 150, h, h, dh, 1)
    table = synth.normal((32, h), 1, "t")
    s = torch.cuda.Stream()
    pl = RelPosBuckets.sequence(150, device=DEV)
    with torch.cuda.stream(s):
        x = qkv.to(DEV, non_blocking=True)
        y = x * 2
        got = ops.attention_rel_bias(y, h, table.to(DEV), pl)
    s.synchronize()
    ref = Ref((qkv.float() * 2).to(BF), table, pl.index(), h, h, None, dh ** -0.5)
    assert ((got.cpu().double() - ref.out).abs() <= SLACK * U * (ref.out_mag + ref.out.abs())).all()


@pytest.mark.parametrize("b,grid,h,hk,dh", [(2, (5, 7), 4, 2, 32), (40, (14, 14), 4, 4, 64), (60, (10, 10), 4, 2, 48)])
def test_gradient_without_the_table(b, grid, h, hk, dh):
    """d_table NULL: the same dqkv; the workspace it writes ends where it says."""
    pl = plan(grid, 1, False)
    n = pl.seq
    qkv, table = make(b, n, h, hk, dh, pl.num_buckets)
    x, t = qkv.to(DEV), table.to(DEV)
    g = synth.normal((b, n, h * dh), 4, "d").to(BF).to(DEV)
    out, lse = ops.attention_rel_bias_train(x, h, t, pl, num_kv_heads=hk)
    want, dt = ops.attention_rel_bias_backward(x, out, g, lse, h, t, pl, num_kv_heads=hk)
    lib, c = _lib.load(), pl._c()
    need = lib.vit_attention_rel_bwd_workspace_bytes(c, b, h, dh)
    ws = torch.full((need + 4096,), 77, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    for table_grad in (None, torch.empty_like(dt)):
        got = torch.empty_like(x)
        _lib.check(lib.vit_attention_rel_bwd(c, x.data_ptr(), t.data_ptr(), None, out.data_ptr(), g.data_ptr(), lse.data_ptr(), got.data_ptr(),
                                             None if table_grad is None else table_grad.data_ptr(), ws.data_ptr(), need, b, h, hk, dh,
                                             dh ** -0.5, stream))
        assert torch.equal(got, want) and (ws[need:] == 77).all()
        assert table_grad is None or torch.equal(table_grad, dt)
    assert lib.vit_attention_rel_bwd(c, x.data_ptr(), t.data_ptr(), None, out.data_ptr(), g.data_ptr(), lse.data_ptr(), got.data_ptr(), None,
                                     ws.data_ptr(), need - 1, b, h, hk, dh, dh ** -0.5, stream) != 0


@pytest.mark.parametrize("grid,prefix,h,dh", [((1, 4096), 0, 12, 64), ((64, 64), 1, 12, 64), ((1, 4096), 0, 12, 80), ((64, 64), 1, 12, 112)])
def test_long_with_many_rows(grid, prefix, h, dh):
    """The kernels for many rows at thousands of tokens, whole and with lengths, against the fp32 form (2^-16 of the magnitudes)."""
    pl = RelPosBuckets(grid, prefix=prefix, device=DEV)
    n = pl.seq
    qkv, table = make(1, n, h, h, dh, pl.num_buckets)
    x, t = qkv.to(DEV), table.to(DEV)
    f = x.float()
    want = ops.attention_rel_bias(f, h, t, pl)
    mag = ops.attention_rel_bias(torch.cat([f[..., :2 * h * dh], f[..., 2 * h * dh:].abs()], -1), h, t, pl)
    tol = SLACK * U * (mag + want.abs()) + 2.0 ** -16 * mag
    assert ((ops.attention_rel_bias(x, h, t, pl).float() - want).abs() <= tol).all()
    full, part = (torch.tensor([m], dtype=torch.int32, device=DEV) for m in (n, n - 37))
    assert ((ops.attention_rel_bias(x, h, t, pl, lengths=full).float() - want).abs() <= tol).all()
    want = ops.attention_rel_bias(f, h, t, pl, lengths=part)
    mag = ops.attention_rel_bias(torch.cat([f[..., :2 * h * dh], f[..., 2 * h * dh:].abs()], -1), h, t, pl, lengths=part)
    got = ops.attention_rel_bias(x, h, t, pl, lengths=part).float()
    assert ((got - want).abs() <= SLACK * U * (mag + want.abs()) + 2.0 ** -16 * mag).all() and not got[:, n - 37:].any()


def test_two_graphs():
    """Two captured steps, replayed in turns without a wait between them, keep out of each other's memory; one is captured at its first call."""
    def make_step(grid, b, h, dh, seed):
        pl = plan(grid, 1, True)
        x = synth.normal((b, pl.seq, 3 * h * dh), seed, "x").to(BF).to(DEV)
        t = synth.normal((pl.num_buckets, h), seed, "t").to(DEV)
        g = synth.normal((b, pl.seq, h * dh), seed, "g").to(BF).to(DEV)
        w = torch.ones(dh, device=DEV)

        def step():
            y = ops.qk_norm_rope(x, h, w, w)
            out, lse = ops.attention_rel_bias_train(y, h, t, pl)
            dy, dt = ops.attention_rel_bias_backward(y, out, g, lse, h, t, pl)
            return (out, dt) + ops.qk_norm_rope_backward(x, dy, h, w, w)[:3]
        return step

    steps = [make_step((14, 14), 60, 4, 64, 1), make_step((3, 11), 3, 2, 112, 2)]
    graphs, outs = [], []
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s())
        graphs.append(g)
    eager = [s() for s in steps]
    for _ in range(3):
        for o in outs:
            for v in o:
                v.zero_()
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert all(torch.equal(a, c) for a, c in zip(o, e))
        steps[0]()  # (eager work between the replays)
