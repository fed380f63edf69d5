"""GPU parity tests of attention with a bucketed relative position bias and its gradient against plain torch in 64 bits.

Bars, from the arithmetic. bf16: the probabilities are rounded by at most 2^-8 of themselves before they meet the values, so
a result is off by at most 2^-8 sum_j P_j |V_j|, and by 2^-8 of itself when it is stored (likewise dQ by 2^-8 scale sum
|dS| |K|, dK, dV); a further eighth covers the fp32 steps (exponent arguments of some tens rounded by 2^-24: 2^-17) and, in
dQ and dK, the rounded out in delta: 2^-8 sum_j P_j |V_j| |dO| of each row times P. The bias gradient and the fp32 mode round
in fp32 only: arguments of up to 64 by 2^-24 each give 2^-16 of a probability at worst (2^-16 sum |terms|)."""
import pytest
import torch

from vit_amd import ops, synth
from vit_amd.rel_pos import RelPosBuckets

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
U = 2.0 ** -8
SLACK = 1 + 2.0 ** -3


def make(b, n, h, hk, dh, nb, dtype=BF, seed=9):
    qkv = synth.normal((b, n, (h + 2 * hk) * dh), seed, "qkv").to(dtype)
    return qkv, synth.normal((nb, h), seed, "table", std=0.8)


class Ref:
    """Everything in 64 bits from the definition, the gradients by the formulas (autograd agrees: test_formulas)."""

    def __init__(self, qkv, table, index, h, hk, lengths, scale, d_out=None):
        b, n, w = qkv.shape
        dh = w // (h + 2 * hk)
        e = qkv.double().unflatten(-1, (h + 2 * hk, dh)).transpose(1, 2)
        grp = h // hk
        q, k, v = e[:, :h], e[:, h:h + hk].repeat_interleave(grp, 1), e[:, h + hk:].repeat_interleave(grp, 1)
        bias = table.double()[index].permute(2, 0, 1)
        bias = torch.where(bias < -1e30, -torch.inf, bias)
        s = q @ k.transpose(-1, -2) * scale + bias
        used = torch.ones(b, n, dtype=torch.bool) if lengths is None else torch.arange(n)[None] < lengths[:, None].clamp(0, n)
        s = torch.where(used[:, None, None, :], s, -torch.inf)
        m = s.amax(-1, keepdim=True)
        self.empty = (m == -torch.inf)[..., 0] | ~used[:, None, :]
        p = torch.exp(s - torch.where(m == -torch.inf, 0.0, m))
        z = p.sum(-1, keepdim=True)
        self.lse = torch.where(self.empty, torch.inf, ((m + z.log()) / torch.log(torch.tensor(2.0, dtype=torch.float64)))[..., 0])
        p = torch.where(self.empty[..., None], 0.0, p / z)
        pack = lambda t: t.transpose(1, 2).flatten(2)  # noqa: E731
        self.out, self.out_mag = pack(p @ v), pack(p @ v.abs())
        if d_out is None:
            return
        do = d_out.double().unflatten(-1, (h, dh)).transpose(1, 2)
        dp = do @ v.transpose(-1, -2)
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        # rounding of delta: out by U (sum P |V|) and U |out|, times |dO|
        ddel = 2 * U * ((p @ v.abs()) * do.abs()).sum(-1, keepdim=True)
        mag = ds.abs() * U + p * ddel
        fold = lambda t: pack(t.unflatten(1, (hk, grp)).sum(2))  # noqa: E731
        self.dqkv = torch.cat([pack(ds @ k) * scale, fold(ds.transpose(-1, -2) @ q) * scale, fold(p.transpose(-1, -2) @ do)], -1)
        self.dmag = torch.cat([pack(mag @ k.abs()) * scale, fold((U * ds.abs()).transpose(-1, -2) @ q.abs()) * scale,
                               fold((U * p).transpose(-1, -2) @ do.abs())], -1)
        add = lambda t: torch.zeros_like(table, dtype=torch.float64).index_add_(0, index.flatten(), t.sum(0).flatten(1).t())  # noqa: E731
        self.dtable = add(ds)
        self.dtable_mag = add(p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True)))


def plan(grid, prefix, mapped):
    if not mapped:
        return RelPosBuckets(grid, prefix=prefix, device=DEV)
    gh, gw = grid
    total = (2 * gh - 1) * (2 * gw - 1) + (3 if prefix else 0)
    return RelPosBuckets(grid, prefix=prefix, bucket_of=[(7 * i * i + i // 3) % 11 for i in range(total)], num_buckets=12, device=DEV)


CASES = [  # b, grid, prefix, h, hk, dh, mapped, lengths
    (1, (1, 1), 0, 1, 1, 16, False, None),
    (2, (1, 1), 1, 2, 1, 32, False, None),
    (3, (14, 14), 1, 3, 3, 64, False, None),
    (2, (5, 7), 5, 4, 2, 48, False, None),
    (2, (1, 130), 0, 4, 1, 80, True, None),
    (2, (9, 1), 0, 2, 2, 112, False, None),
    (5, (6, 11), 2, 2, 2, 64, True, [68, 0, 1, 33, 64]),
    (4, (1, 97), 0, 3, 1, 128, False, [97, 5, 96, 32]),
    (2, (17, 19), 1, 2, 2, 64, False, None),
    (1, (3, 67), 32, 2, 1, 96, False, [201]),
    (33, (4, 4), 1, 2, 2, 32, False, None),
    (2, (24, 24), 1, 1, 1, 64, False, [577, 400]),
]
IDS = lambda c: "-".join(str(v).replace(" ", "") for v in c)  # noqa: E731


def setup_case(case, dtype=BF):
    b, grid, prefix, h, hk, dh, mapped, lengths = case
    pl = plan(grid, prefix, mapped)
    qkv, table = make(b, pl.seq, h, hk, dh, pl.num_buckets, dtype)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return pl, qkv, table, ln


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_bf16_forward(case):
    b, grid, prefix, h, hk, dh, mapped, lengths = case
    pl, qkv, table, ln = setup_case(case)
    ref = Ref(qkv, table, pl.index(), h, hk, ln, dh ** -0.5)
    kw = dict(lengths=None if ln is None else ln.to(DEV), num_kv_heads=hk)
    got = ops.attention_rel_bias(qkv.to(DEV), h, table.to(DEV), pl, **kw)
    tol = SLACK * U * (ref.out_mag + ref.out.abs()) + 1e-30
    err = (got.cpu().double() - ref.out).abs()
    assert (err <= tol).all(), (err / tol).max()
    out, lse = ops.attention_rel_bias_train(qkv.to(DEV), h, table.to(DEV), pl, **kw)
    assert torch.equal(out, got)
    lse = lse.cpu().double()
    assert torch.equal(torch.isinf(lse), ref.empty)
    fin = ~ref.empty
    assert ((lse - ref.lse)[fin].abs() <= 2.0 ** -18 * (1 + ref.lse[fin].abs())).all()


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_fp32_forward(case):
    b, grid, prefix, h, hk, dh, mapped, lengths = case
    pl, qkv, table, ln = setup_case(case, torch.float32)
    ref = Ref(qkv, table, pl.index(), h, hk, ln, dh ** -0.5)
    got = ops.attention_rel_bias(qkv.to(DEV), h, table.to(DEV), pl, lengths=None if ln is None else ln.to(DEV), num_kv_heads=hk)
    err = (got.cpu().double() - ref.out).abs()
    tol = 2.0 ** -16 * ref.out_mag + 1e-30
    assert (err <= tol).all(), (err / tol).max()


@pytest.mark.parametrize("case", CASES, ids=IDS)
def test_gradient(case):
    b, grid, prefix, h, hk, dh, mapped, lengths = case
    pl, qkv, table, ln = setup_case(case)
    d_out = synth.normal((b, pl.seq, h * dh), 4, "d_out").to(BF)
    ref = Ref(qkv, table, pl.index(), h, hk, ln, dh ** -0.5, d_out)
    kw = dict(lengths=None if ln is None else ln.to(DEV), num_kv_heads=hk)
    q, t = qkv.to(DEV), table.to(DEV)
    out, saved = ops.attention_rel_bias_train(q, h, t, pl, **kw)
    dqkv, dt = ops.attention_rel_bias_backward(q, out, d_out.to(DEV), saved, h, t, pl, **kw)
    tol = SLACK * (ref.dmag + U * ref.dqkv.abs()) + 2.0 ** -16 * ref.dqkv.abs().max() + 1e-30
    err = (dqkv.cpu().double() - ref.dqkv).abs()
    assert (err <= tol).all(), (err / tol).max()
    tol = 2.0 ** -16 * ref.dtable_mag + 1e-30
    err = (dt.cpu().double() - ref.dtable).abs()
    assert (err <= tol).all(), (err / tol).max()
    again = ops.attention_rel_bias_backward(q, out, d_out.to(DEV), saved, h, t, pl, **kw)
    assert torch.equal(dqkv, again[0]) and torch.equal(dt, again[1])


def test_formulas():
    """The reference's gradients are autograd's, and the bias gradient is the difference quotient of the loss."""
    pl = plan((3, 4), 2, True)
    qkv, table = make(2, pl.seq, 4, 2, 16, pl.num_buckets, torch.float64)
    g = synth.normal((2, pl.seq, 64), 3, "g").double()
    ln = torch.tensor([14, 9])
    ref = Ref(qkv, table, pl.index(), 4, 2, ln, 0.3, g)
    x, t = qkv.double().requires_grad_(), table.double().requires_grad_()
    e = x.unflatten(-1, (8, 16)).transpose(1, 2)
    s = e[:, :4] @ e[:, 4:6].repeat_interleave(2, 1).transpose(-1, -2) * 0.3 + t[pl.index()].permute(2, 0, 1)
    used = torch.arange(14)[None] < ln[:, None]
    s = s.masked_fill(~used[:, None, None], -torch.inf)
    o = (torch.softmax(s, -1) @ e[:, 6:].repeat_interleave(2, 1) * used[:, None, :, None]).transpose(1, 2).flatten(2)
    dx, dt = torch.autograd.grad(o, [x, t], g)
    assert torch.allclose(dx, ref.dqkv, atol=1e-12) and torch.allclose(dt, ref.dtable, atol=1e-12)
    step = torch.zeros_like(table, dtype=torch.float64)
    step[3, 1] = 1e-5
    up, dn = (Ref(qkv, table.double() + k * step, pl.index(), 4, 2, ln, 0.3).out for k in (1, -1))
    assert abs(((up - dn) * g).sum() / 2e-5 - ref.dtable[3, 1]) < 1e-7


@pytest.mark.parametrize("value", [float("-inf"), torch.finfo(torch.float32).min, -2e30])
def test_entries_that_mask(value):
    """Offsets masked by the table, down to queries that keep no key (rows of zeros, no gradient from them)."""
    pl = RelPosBuckets((1, 70), device=DEV)
    h, dh = 2, 64
    qkv, table = make(2, 70, h, h, dh, pl.num_buckets)
    table[69:] = value          # keys at or before the query: query 69 sees nothing
    table[:, 1][60:69] = value  # second head: only keys 10 or more behind the query
    d_out = synth.normal((2, 70, h * dh), 4, "d").to(BF)
    ref = Ref(qkv, table, pl.index(), h, h, None, dh ** -0.5, d_out)
    assert ref.empty[:, 0].sum() == 2 and ref.empty[:, 1].sum() == 20
    q, t = qkv.to(DEV), table.to(DEV)
    out, lse = ops.attention_rel_bias_train(q, h, t, pl)
    dqkv, dt = ops.attention_rel_bias_backward(q, out, d_out.to(DEV), lse, h, t, pl)
    assert torch.equal(torch.isinf(lse).cpu(), ref.empty)
    assert ((out.cpu().double() - ref.out).abs() <= SLACK * U * (ref.out_mag + ref.out.abs()) + 1e-30).all()
    tol = SLACK * (ref.dmag + U * ref.dqkv.abs()) + 2.0 ** -16 * ref.dqkv.abs().max()
    assert ((dqkv.cpu().double() - ref.dqkv).abs() <= tol).all()
    assert ((dt.cpu().double() - ref.dtable).abs() <= 2.0 ** -16 * ref.dtable_mag + 1e-30).all()
    f = ops.attention_rel_bias(q.float(), h, t, pl)
    assert ((f.cpu().double() - ref.out).abs() <= 2.0 ** -16 * ref.out_mag + 1e-30).all()


def test_padding_is_never_read():
    """NaN and infinities behind each sample's length reach nothing."""
    b, h, hk, dh, ln = 4, 4, 2, 64, [70, 1, 0, 37]
    pl = plan((10, 7), 1, False)
    qkv, table = make(b, 71, h, hk, dh, pl.num_buckets)
    d_out = synth.normal((b, 71, h * dh), 4, "d").to(BF)
    t, lens = table.to(DEV), torch.tensor(ln, dtype=torch.int32, device=DEV)

    def run(x, g):
        out, lse = ops.attention_rel_bias_train(x.to(DEV), h, t, pl, lengths=lens, num_kv_heads=hk)
        return (out, lse) + ops.attention_rel_bias_backward(x.to(DEV), out, g.to(DEV), lse, h, t, pl, lengths=lens, num_kv_heads=hk)

    clean = run(qkv, d_out)
    bad, badg = qkv.clone(), d_out.clone()
    for i, n in enumerate(ln):
        bad[i, n:] = float("nan")
        bad[i, n::2] = float("inf")
        badg[i, n:] = float("nan")
    for p, q in zip(clean, run(bad, badg)):
        assert torch.equal(p, q)
    assert not clean[0][2].any() and not clean[2][1, 1:].any()
    f = [ops.attention_rel_bias(x.float().to(DEV), h, t, pl, lengths=lens, num_kv_heads=hk) for x in (qkv, bad)]
    assert torch.equal(*f)


def test_lengths_outside_the_range_are_clamped():
    pl = plan((4, 8), 0, False)
    qkv, table = make(2, 32, 2, 2, 32, pl.num_buckets)
    x, t = qkv.to(DEV), table.to(DEV)
    a = ops.attention_rel_bias(x, 2, t, pl, lengths=torch.tensor([-3, 1000], dtype=torch.int32, device=DEV))
    c = ops.attention_rel_bias(x, 2, t, pl, lengths=torch.tensor([0, 32], dtype=torch.int32, device=DEV))
    assert torch.equal(a, c) and not a[0].any()


def test_zero_table_is_plain_attention():
    pl = plan((14, 14), 1, False)
    qkv, _ = make(4, 197, 12, 12, 64, 1)
    x = qkv.to(DEV)
    got = ops.attention_rel_bias(x, 12, torch.zeros(pl.num_buckets, 12, device=DEV), pl)
    ref = Ref(qkv, torch.zeros(pl.num_buckets, 12), pl.index(), 12, 12, None, 0.125)
    for y in (got, ops.attention(x, 12)):  # the stand-in for each other: both within the same bound of the exact result
        assert ((y.cpu().double() - ref.out).abs() <= SLACK * U * (ref.out_mag + ref.out.abs())).all()


def test_large_scores_and_scale():
    """Scores of several hundred (a one-hot softmax), another scale, and a running maximum that keeps rising."""
    pl = plan((1, 150), 0, False)
    qkv, table = make(1, 150, 2, 2, 64, pl.num_buckets, torch.float32)
    qkv[..., :256] *= 4
    qkv[0, :, 128:192] = qkv[0, :, 128:192] * torch.linspace(0.1, 3, 150)[:, None]
    x = qkv.to(BF)
    ref = Ref(x, table, pl.index(), 2, 2, None, 0.5)
    got = ops.attention_rel_bias(x.to(DEV), 2, table.to(DEV), pl, scale=0.5)
    # arguments of up to ~1500 rounded by 2^-24: 2^-13 of a probability
    assert ((got.cpu().double() - ref.out).abs() <= (SLACK * U + 2.0 ** -12) * (ref.out_mag + ref.out.abs())).all()


def test_sequence_buckets_long():
    """A long ragged sequence with logarithmic buckets: offsets sum into few buckets, many tiles on both sides."""
    pl = RelPosBuckets.sequence(700, num_buckets=32, max_distance=128, device=DEV)
    h, hk, dh, ln = 4, 2, 64, torch.tensor([700, 411], dtype=torch.int32)
    qkv, table = make(2, 700, h, hk, dh, 32)
    d_out = synth.normal((2, 700, h * dh), 4, "d").to(BF)
    ref = Ref(qkv, table, pl.index(), h, hk, ln, 0.125, d_out)
    x, t, kw = qkv.to(DEV), table.to(DEV), dict(lengths=ln.to(DEV), num_kv_heads=hk)
    out, lse = ops.attention_rel_bias_train(x, h, t, pl, **kw)
    dqkv, dt = ops.attention_rel_bias_backward(x, out, d_out.to(DEV), lse, h, t, pl, **kw)
    assert ((out.cpu().double() - ref.out).abs() <= SLACK * U * (ref.out_mag + ref.out.abs()) + 1e-30).all()
    assert ((dqkv.cpu().double() - ref.dqkv).abs() <= SLACK * (ref.dmag + U * ref.dqkv.abs()) + 2.0 ** -16 * ref.dqkv.abs().max()).all()
    assert ((dt.cpu().double() - ref.dtable).abs() <= 2.0 ** -16 * ref.dtable_mag).all()
    assert ((dt.cpu().double() - ref.dtable).norm() / ref.dtable.norm()) < 1e-5


def test_graph_replays_equal_eager():
    pl = plan((14, 14), 1, True)
    qkv, table = make(3, 197, 4, 4, 64, pl.num_buckets)
    x, t = qkv.to(DEV), table.to(DEV)
    g = torch.randn(3, 197, 256, device=DEV).to(BF)
    lens = torch.tensor([197, 100, 3], dtype=torch.int32, device=DEV)

    def step():
        out, lse = ops.attention_rel_bias_train(x, 4, t, pl, lengths=lens)
        return (out,) + ops.attention_rel_bias_backward(x, out, g, lse, 4, t, pl, lengths=lens)

    step()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(3):
        x.copy_(torch.randn_like(x))
        t.copy_(torch.randn_like(t))
        lens.copy_(torch.tensor([197 - k, 50 * k, 197], dtype=torch.int32, device=DEV))
        graph.replay()
        torch.cuda.synchronize()
        for a, e in zip(captured, step()):
            assert torch.equal(a, e)


def test_two_streams_at_once():
    pl = plan((14, 14), 1, False)
    qkv, table = make(8, 197, 4, 4, 64, pl.num_buckets)
    t = table.to(DEV)
    xs = [qkv.to(DEV), qkv.to(DEV).flip(0).contiguous()]
    g = torch.randn(8, 197, 256, device=DEV).to(BF)

    def step(x):
        out, lse = ops.attention_rel_bias_train(x, 4, t, pl)
        return (out,) + ops.attention_rel_bias_backward(x, out, g, lse, 4, t, pl)

    ref = [step(x) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in xs]
    got = []
    for x, s in zip(xs, streams):
        with torch.cuda.stream(s):
            got.append(step(x))
    torch.cuda.synchronize()
    for a, r in zip(got, ref):
        assert all(torch.equal(p, q) for p, q in zip(a, r))


def test_projection_norm_attention_run():
    """The path they are made for: linear -> qk_norm_rope -> attention_rel_bias -> linear, forward and every gradient
    through the package's own backward calls, against 64-bit autograd of the whole run."""
    b, h, dh, d = 2, 4, 64, 256
    pl = plan((6, 6), 1, False)
    n = pl.seq
    x = synth.normal((b, n, d), 1, "x").to(BF)
    wqkv, wo = (synth.normal(s, 1, k, std=d ** -0.5).to(BF) for s, k in (((3 * d, d), "wqkv"), ((d, d), "wo")))
    qw, kw = (1 + synth.normal((dh,), 1, k, std=0.2) for k in ("qw", "kw"))
    table = synth.normal((pl.num_buckets, h), 1, "t", std=0.5)
    gy = synth.normal((b, n, d), 1, "gy").to(BF)
    rope = ops.rope_table((6, 6), dh, device="cpu")
    pos = torch.arange(-1, n - 1, dtype=torch.int32)

    dev = [v.to(DEV) for v in (x, wqkv, wo, qw, kw, table, gy, rope, pos)]
    X, WQKV, WO, QW, KW, T, GY, ROPE, POS = dev
    qkv = ops.linear(X, WQKV)
    normed = ops.qk_norm_rope(qkv, h, QW, KW, rope=ROPE, positions=POS)
    att, saved = ops.attention_rel_bias_train(normed, h, T, pl)
    y = ops.linear(att, WO)
    d_att = ops.linear_dgrad(GY, WO.t().contiguous())
    d_normed, d_table = ops.attention_rel_bias_backward(normed, att, d_att, saved, h, T, pl)
    d_qkv, dqw, dkw, _, _ = ops.qk_norm_rope_backward(qkv, d_normed, h, QW, KW, rope=ROPE, positions=POS)
    dx = ops.linear_dgrad(d_qkv, WQKV.t().contiguous())

    leaves = [v.double().requires_grad_() for v in (x, wqkv, wo, qw, kw, table)]
    rx, rw, ro, rqw, rkw, rt = leaves
    e = (rx @ rw.t()).unflatten(-1, (3, h, dh))
    z = torch.cat([torch.ones(1, dh // 2, dtype=torch.complex128), torch.view_as_complex(rope.double())]).unsqueeze(-2)

    def norm(t, w):
        t = t * torch.rsqrt((t * t).mean(-1, keepdim=True) + 1e-6) * w
        v = torch.complex(t[..., :dh // 2], t[..., dh // 2:]) * z
        return torch.cat([v.real, v.imag], -1).transpose(1, 2)

    q, k, v = norm(e[:, :, 0], rqw), norm(e[:, :, 1], rkw), e[:, :, 2].transpose(1, 2)
    s = q @ k.transpose(-1, -2) * dh ** -0.5 + rt[pl.index()].permute(2, 0, 1)
    ry = (torch.softmax(s, -1) @ v).transpose(1, 2).flatten(2) @ ro.t()
    grads = torch.autograd.grad(ry, leaves, gy.double())
    # a chain of four to eight bf16 roundings (2^-8 at most, 2^-9.8 rms each): 3 % of the norm is more than twice their sum
    rel = lambda a, r: ((a.cpu().double() - r).norm() / r.norm()).item()  # noqa: E731
    for got, want in ((y, ry.detach()), (dx, grads[0]), (dqw, grads[3]), (dkw, grads[4]), (d_table, grads[5])):
        assert rel(got, want) < 3e-2, rel(got, want)


def test_refusals_on_device():
    from vit_amd._lib import VitError
    pl = plan((4, 4), 0, False)
    qkv, table = make(2, 16, 2, 2, 32, pl.num_buckets)
    x, t = qkv.to(DEV), table.to(DEV)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    for args, kw in (((x, 3, t, pl), {}), ((x[:, :15], 2, t, pl), {}), ((x, 2, t[:-1], pl), {}), ((x, 2, t.cpu(), pl), {}),
                     ((x, 2, t, pl), dict(lengths=lens.long())), ((x, 2, t, pl), dict(lengths=lens[:1])),
                     ((x, 2, t, pl), dict(lengths=lens.cpu())), ((x[0], 2, t, pl), {}), ((x[:0], 2, t, pl), {})):
        with pytest.raises(ValueError):
            ops.attention_rel_bias(*args, **kw)
    with pytest.raises(TypeError):
        ops.attention_rel_bias(x.half(), 2, t, pl)
    with pytest.raises(TypeError):
        ops.attention_rel_bias_train(x.float(), 2, t, pl)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(VitError):
            ops.attention_rel_bias(x, 2, t, pl, scale=scale)
    out, lse = ops.attention_rel_bias_train(x, 2, t, pl)
    with pytest.raises(ValueError):
        ops.attention_rel_bias_backward(x, out, out, lse[:1], 2, t, pl)
    with pytest.raises(ValueError):
        ops.attention_rel_bias_backward(x, out, out[:1], lse, 2, t, pl)
    big = RelPosBuckets((128, 128), device=DEV)
    xb = torch.zeros(1, 128 * 128, 3 * 16, dtype=BF, device=DEV)
    with pytest.raises(VitError, match="bias entries"):
        ops.attention_rel_bias(xb, 1, torch.zeros(big.num_buckets, 1, device=DEV), big)
