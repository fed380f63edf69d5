"""CPU: bucket plans, rotary tables and the refusals of the head norm / relative position bias entry points (no kernel runs)."""
import ctypes
import math

import pytest
import torch

from vit_amd import _lib, ops
from vit_amd.rel_pos import RelPosBuckets


def test_grid_index_by_hand():
    p = RelPosBuckets((2, 3), prefix=1, device="cpu")
    assert (p.seq, p.offsets, p.num_buckets) == (7, 15, 18)
    idx = p.index()
    assert idx[0, 0] == 17 and (idx[0, 1:] == 15).all() and (idx[1:, 0] == 16).all()
    for i in range(6):
        for j in range(6):
            dy, dx = i // 3 - j // 3, i % 3 - j % 3
            assert idx[1 + i, 1 + j] == (dy + 1) * 5 + dx + 2
    # one offset, one bucket: the same for every pair that has it
    assert idx[1, 1] == idx[6, 6] and len(set(idx[1:, 1:].flatten().tolist())) == 15


def test_map_and_inverse():
    m = [i % 4 for i in range(15)]
    p = RelPosBuckets((2, 3), bucket_of=m, num_buckets=5, device="cpu")
    assert p.bucket_start.tolist() == [0, 4, 8, 12, 15, 15]
    for b in range(5):
        at = p.by_bucket[p.bucket_start[b]:p.bucket_start[b + 1]].tolist()
        assert at == [i for i in range(15) if m[i] == b]


def test_log_buckets():
    b = RelPosBuckets.log_buckets(200, 32, 128)
    assert len(b) == 399 and b[199] == 0 and min(b) == 0 and max(b) == 31
    for d in range(8):  # exact buckets, both directions
        assert b[199 + d] == d and b[199 - d] == (16 + d if d else 0)
    for d in range(8, 200):
        want = min(8 + math.floor(math.log(d / 8) / math.log(16) * 8 + 1e-9), 15)
        assert b[199 + d] == want and b[199 - d] == 16 + want
    assert b[199 + 16] == 10 and b[199 + 128] == 15 and b[199 + 199] == 15
    one = RelPosBuckets.log_buckets(50, 8, 20, bidirectional=False)
    assert all(v == 0 for v in one[:50]) and max(one) == 7 and one[49 + 3] == 3


@pytest.mark.parametrize("kw,err", [
    (dict(grid=(0, 4)), ValueError), (dict(grid=(200, 200)), ValueError), (dict(grid=(2, 2), prefix=33), ValueError),
    (dict(grid=(2, 2), prefix=-1), ValueError), (dict(grid=(2, 2), num_buckets=8), ValueError),
    (dict(grid=(2, 2), bucket_of=[0] * 8), ValueError), (dict(grid=(2, 2), bucket_of=[0] * 8 + [-1]), ValueError),
    (dict(grid=(2, 2), bucket_of=[0] * 8 + [3], num_buckets=3), ValueError), (dict(grid=(2, 2), bucket_of=[0.0] * 9), TypeError)])
def test_plan_refusals(kw, err):
    with pytest.raises(err):
        RelPosBuckets(device="cpu", **kw)


def test_rope_table():
    t = ops.rope_table((1, 5), 8, device="cpu").double()
    for p in range(5):
        for i in range(4):
            a = p * 10000.0 ** (-i / 4)
            assert abs(t[p, i, 0] - math.cos(a)) < 1e-7 and abs(t[p, i, 1] - math.sin(a)) < 1e-7
    g = ops.rope_table((3, 4), 8, device="cpu").double()
    assert g.shape == (12, 4, 2)
    a = 2 * 100.0 ** -0.5  # row 2, second row frequency; column 3, first column frequency
    assert abs(g[2 * 4 + 3, 1, 0] - math.cos(a)) < 1e-7 and abs(g[2 * 4 + 3, 2, 1] - math.sin(3.0)) < 1e-7
    with pytest.raises(ValueError):
        ops.rope_table((2, 2), 6, device="cpu")


def test_wrappers_have_no_cpu_path():
    x = torch.zeros(1, 4, 3 * 32, dtype=torch.bfloat16)
    w = torch.ones(32)
    p = RelPosBuckets((2, 2), device="cpu")
    t = torch.zeros(9, 1)
    for call in (lambda: ops.qk_norm_rope(x, 1, w, w), lambda: ops.qk_norm_rope_backward(x, x, 1, w, w),
                 lambda: ops.attention_rel_bias(x, 1, t, p), lambda: ops.attention_rel_bias_train(x, 1, t, p),
                 lambda: ops.attention_rel_bias_backward(x, x[..., :32], x[..., :32], t, 1, t, p)):
        with pytest.raises(ValueError, match="GPU"):
            call()


FAKE = 1 << 20  # an aligned address that no refused call reads


def qk_cfg(**kw):
    d = dict(batch=1, seq=4, heads=2, kv_heads=1, head_dim=32, norm=0, rot_dim=32, interleaved=0, rope_len=4, positions_per_sample=0,
             dtype=1, eps=1e-6)
    d.update(kw)
    return _lib.vit_qk_norm_config(**d)


@pytest.mark.parametrize("kw", [dict(batch=0), dict(seq=-1), dict(heads=3, kv_heads=2), dict(head_dim=24), dict(head_dim=144),
                                dict(rot_dim=48), dict(rot_dim=8), dict(norm=2), dict(dtype=2), dict(eps=0.0), dict(eps=math.inf),
                                dict(rope_len=0), dict(batch=1 << 20, seq=1 << 12)])
def test_qk_norm_c_refusals(kw):
    lib = _lib.load()
    c = qk_cfg(**kw)
    assert lib.vit_qk_norm_rope_fwd(c, FAKE, FAKE, FAKE, None, None, FAKE, None, 2 * FAKE, None) == -1
    assert lib.vit_qk_norm_rope_bwd(c, FAKE, 2 * FAKE, FAKE, FAKE, FAKE, None, 3 * FAKE, FAKE, FAKE, None, None, FAKE, 1 << 30, None) == -1
    assert lib.vit_last_error()


def test_qk_norm_c_refusals_of_pointers():
    lib = _lib.load()
    c = qk_cfg()
    for a in ([None, FAKE, FAKE, None, None, FAKE, None, 2 * FAKE], [FAKE, FAKE, None, None, None, FAKE, None, 2 * FAKE],
              [FAKE, FAKE, FAKE, FAKE, None, FAKE, None, 2 * FAKE], [FAKE, FAKE, FAKE, None, None, None, None, 2 * FAKE],
              [FAKE + 2, FAKE, FAKE, None, None, FAKE, None, 2 * FAKE], [FAKE, FAKE, FAKE, None, None, FAKE, None, FAKE + 64]):
        assert lib.vit_qk_norm_rope_fwd(c, *a, None) == -1
    assert lib.vit_qk_norm_rope_fwd(None, FAKE, FAKE, FAKE, None, None, FAKE, None, FAKE, None) == -1
    # dqkv inside qkv, or beside d_out without being it
    for d in (FAKE, FAKE + 64, 2 * FAKE + 64):
        assert lib.vit_qk_norm_rope_bwd(c, FAKE, 2 * FAKE, FAKE, FAKE, FAKE, None, d, FAKE, FAKE, None, None, FAKE, 1 << 30, None) == -1


def rel_pos(**kw):
    d = dict(prefix=0, grid_h=4, grid_w=4, num_buckets=49, bucket_of=None, by_bucket=None, bucket_start=None)
    d.update(kw)
    return _lib.vit_rel_pos(**d)


REL_BAD = [(dict(prefix=-1), {}), (dict(prefix=33), {}), (dict(grid_h=0), {}), (dict(grid_h=200, grid_w=200), {}), (dict(num_buckets=48), {}),
           (dict(prefix=1), {}), (dict(num_buckets=0, bucket_of=FAKE), {}), ({}, dict(batch=0)), ({}, dict(heads=3, kv_heads=2)),
           ({}, dict(head_dim=40)), ({}, dict(head_dim=144)), ({}, dict(scale=0.0)), ({}, dict(scale=math.nan)), ({}, dict(scale=math.inf)),
           ({}, dict(batch=1 << 21)), ({}, dict(qkv=None)), ({}, dict(qkv=FAKE + 8)), ({}, dict(out=None)), ({}, dict(table=None)),
           (dict(grid_h=128, grid_w=128, num_buckets=255 * 255), {})]


@pytest.mark.parametrize("pos,kw", REL_BAD)
def test_attention_rel_c_refusals(pos, kw):
    lib = _lib.load()
    d = dict(qkv=FAKE, table=FAKE, out=FAKE, batch=1, heads=2, kv_heads=2, head_dim=32, scale=0.2)
    d.update(kw)
    tail = [d[k] for k in ("batch", "heads", "kv_heads", "head_dim", "scale")]
    p = rel_pos(**pos)
    assert lib.vit_attention_rel_fwd(p, d["qkv"], d["table"], None, d["out"], None, *tail, 1, None) == -1
    assert lib.vit_last_error()
    if pos.get("grid_h") != 128:  # (the backward first needs the device's size for its plan)
        assert lib.vit_attention_rel_bwd(p, d["qkv"], d["table"], None, d["out"], FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, *tail, None) == -1


def test_attention_rel_c_more_refusals():
    lib = _lib.load()
    assert lib.vit_attention_rel_fwd(rel_pos(), FAKE, FAKE, None, FAKE, FAKE, 1, 2, 2, 32, 0.2, 0, None) == -1  # lse in fp32 mode
    assert lib.vit_attention_rel_fwd(rel_pos(), FAKE, FAKE, None, FAKE, None, 1, 2, 2, 32, 0.2, 7, None) == -1
    assert lib.vit_attention_rel_fwd(None, FAKE, FAKE, None, FAKE, None, 1, 2, 2, 32, 0.2, 1, None) == -1
    m = rel_pos(bucket_of=FAKE, num_buckets=3)  # the gradient of a mapped table without the map's inverse
    assert lib.vit_attention_rel_bwd(m, FAKE, FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, FAKE, 1 << 40, 1, 2, 2, 32, 0.2, None) == -1
    assert lib.vit_attention_rel_bwd_workspace_bytes(None, 1, 1, 32) == 0
    assert ctypes.sizeof(_lib.vit_rel_pos) == 40 and ctypes.sizeof(_lib.vit_qk_norm_config) == 48
