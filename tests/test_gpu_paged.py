"""The paged key/value cache: append with rotation, attention of single tokens
over shared prefixes, attention of prompts, each against a 64-bit oracle that
works sequence by sequence; bounds as derived in ``paged_helpers``."""
import math
import sys
import threading

import pytest
import torch

from helpers import cbq, need_cuda
from paged_helpers import Setup, check_attention

pytestmark = pytest.mark.gpu
L = cbq._lib
DT = {"bf16": torch.bfloat16, "f32": torch.float32}


def run(s, op, dev, scale=None, **kw):
    k, v = s.pools(dev)
    c = cbq.PagedKVCache(k, v)
    b = s.batch(cbq, dev, decode=op == "decode", **kw)
    f = c.attend_decode if op == "decode" else c.attend_extend
    return f(b, s.q.to(dev), scale=scale)


def verify(s, op, dev, scale=None, **kw):
    got = run(s, op, dev, scale, **kw)
    check_attention(got, *s.attention(s.d ** -0.5 if scale is None else scale, op == "extend"))
    return got


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (6, 2), (5, 1), (16, 1), (40, 1), (64, 1)])
def test_decode_heads(dt, d, heads, kv_heads):
    dev = need_cuda()
    verify(Setup([1, 16, 17, 0, 33, 300], heads=heads, kv_heads=kv_heads, d=d, dtype=DT[dt]), "decode", dev)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["hnd", "nhd", "joint"])
def test_decode_pages_and_layouts(dt, page, layout):
    dev = need_cuda()
    verify(Setup([5, 255, 256, 257, 0, 1030], d=128, page=page, dtype=DT[dt], layout=layout, slack=2), "decode", dev)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("kv", [[1], [63], [64], [65], [4097], [0], [0, 0, 0]])
def test_decode_single_lengths(dt, kv):
    dev = need_cuda()
    got = verify(Setup(kv, heads=8, kv_heads=2, d=128, dtype=DT[dt]), "decode", dev)
    if not any(kv):
        assert not got.any()


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("groups", [[(9, 500)], [(4, 33), (5, 700)], [(1, 1), (3, 0), (5, 129)]],
                         ids=["one", "two", "three"])
def test_decode_shared_prefix(dt, d, groups):
    dev = need_cuda()
    kv = [0, 1, 40, 0, 17, 300, 64, 5, 128]
    verify(Setup(kv, groups=groups, heads=8, kv_heads=2, d=d, dtype=DT[dt]), "decode", dev)


@pytest.mark.parametrize("n", [1, 31, 33, 150])
def test_decode_prefix_of_many_sequences(n):
    dev = need_cuda()
    verify(Setup([(7 * i) % 50 for i in range(n)], groups=[(n, 1000)], heads=8, kv_heads=2, d=128), "decode", dev)


def test_decode_more_sequences_than_threads():
    """The line of tiles is planned in blocks of owners."""
    dev = need_cuda()
    verify(Setup([(i * 13) % 37 for i in range(700)], heads=2, kv_heads=1, d=64), "decode", dev)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("heads,kv_heads", [(2, 2), (8, 2), (7, 1), (12, 4)])
def test_extend_ragged(dt, d, heads, kv_heads):
    dev = need_cuda()
    verify(Setup([5, 0, 140, 64, 31, 1], new=[5, 0, 30, 64, 1, 1], heads=heads, kv_heads=kv_heads, d=d, dtype=DT[dt]),
           "extend", dev)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("groups", [[(4, 100)], [(1, 17), (3, 300)]], ids=["one", "two"])
def test_extend_behind_prefix(dt, d, groups):
    dev = need_cuda()
    verify(Setup([20, 130, 3, 64], new=[20, 70, 0, 2], groups=groups, heads=8, kv_heads=2, d=d, dtype=DT[dt], page=32),
           "extend", dev)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("new,kv", [(1, 1), (1, 3000), (7, 2000), (127, 127), (128, 128), (129, 129), (257, 700),
                                    (600, 600)])
def test_extend_one_sequence(dt, new, kv):
    dev = need_cuda()
    verify(Setup([kv], new=[new], heads=8, kv_heads=2, d=128, dtype=DT[dt], page=64), "extend", dev)


@pytest.mark.parametrize("page", [16, 128, 256])
@pytest.mark.parametrize("layout", ["nhd", "joint"])
def test_extend_pages_and_layouts(page, layout):
    dev = need_cuda()
    verify(Setup([400, 333], new=[150, 333], groups=[(2, 77)], heads=4, kv_heads=2, d=128, page=page, layout=layout),
           "extend", dev)


@pytest.mark.parametrize("op", ["decode", "extend"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_tokens_without_rows_see_the_prefix_only(op, dt):
    """More new tokens than rows: the first ones see nothing of their own, and without a prefix give zeros."""
    dev = need_cuda()
    if op == "decode":
        s = Setup([0, 3], heads=4, kv_heads=2, dtype=DT[dt])
    else:
        s = Setup([2, 0, 40], new=[5, 4, 40], heads=4, kv_heads=2, dtype=DT[dt])
    got = verify(s, op, dev)
    assert not got[0].any()


def test_scores_of_one_sign_and_large_scores():
    """Softmax over scores far from zero: only differences count."""
    dev = need_cuda()
    s = Setup([300, 80], heads=4, kv_heads=2, d=128)
    s.q *= 30
    verify(s, "decode", dev)
    s.k[..., 0] = torch.where(s.k[..., 0].isnan(), s.k[..., 0], torch.full_like(s.k[..., 0], -50.0))
    verify(s, "decode", dev)


@pytest.mark.parametrize("scale", [0.0, -0.1, 1.0])
@pytest.mark.parametrize("op", ["decode", "extend"])
def test_scales(op, scale):
    dev = need_cuda()
    new = None if op == "decode" else [40, 3]
    verify(Setup([90, 33], new=new, heads=4, kv_heads=2, d=64), op, dev, scale=scale)


@pytest.mark.parametrize("op", ["decode", "extend"])
def test_infinite_rows_outside_the_lengths(op):
    dev = need_cuda()
    new = None if op == "decode" else [40, 3]
    for stale in (math.inf, -math.inf, torch.finfo(torch.bfloat16).min):
        verify(Setup([90, 33], new=new, groups=[(2, 21)], heads=4, kv_heads=2, d=64, stale=stale), op, dev)


@pytest.mark.parametrize("op", ["decode", "extend"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_same_bits_every_time_and_on_another_stream(op, dt):
    dev = need_cuda()
    n = 40
    kv = [(91 * i) % 400 for i in range(n)]
    new = None if op == "decode" else [min(k, (7 * i) % 60) for i, k in enumerate(kv)]
    s = Setup(kv, new=new, groups=[(15, 210), (25, 33)], heads=8, kv_heads=2, d=128, dtype=DT[dt])
    k, v = s.pools(dev)
    c, b, q = cbq.PagedKVCache(k, v), s.batch(cbq, dev, decode=op == "decode"), s.q.to(dev)
    f = c.attend_decode if op == "decode" else c.attend_extend
    first = f(b, q)
    side = torch.cuda.Stream(dev)
    side.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(side):
        others = [f(b, q) for _ in range(5)]
    torch.cuda.current_stream(dev).wait_stream(side)
    for o in others:
        assert torch.equal(o, first)


def test_graph_follows_the_lengths():
    """A captured decode step reads tables and lengths on the device."""
    dev = need_cuda()
    s = Setup([200, 100, 50], groups=[(3, 64)], heads=8, kv_heads=2, d=128, stale=0.0)
    k, v = s.pools(dev)
    c, b, q = cbq.PagedKVCache(k, v), s.batch(cbq, dev, decode=True), s.q.to(dev)
    out = torch.empty_like(q)
    c.attend_decode(b, q, out=out)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c.attend_decode(b, q, out=out)
    for kv in ([200, 100, 50], [1, 0, 37], [180, 99, 2]):
        s.kv = kv
        b.kv_lens.copy_(torch.tensor(kv, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        check_attention(out, *s.attention(s.d ** -0.5, False))


def test_query_slices_of_one_projection():
    dev = need_cuda()
    s = Setup([70, 33, 9], heads=4, kv_heads=2, d=64)
    k, v = s.pools(dev)
    qkv = torch.randn(3, 4 + 2 * 2, 64, device=dev).to(torch.bfloat16)
    qkv[:, :4] = s.q.to(dev)
    got = cbq.PagedKVCache(k, v).attend_decode(s.batch(cbq, dev, decode=True), qkv[:, :4])
    check_attention(got, *s.attention(s.d ** -0.5, False))


@pytest.mark.parametrize("op", ["decode", "extend"])
@pytest.mark.parametrize("bad", [-1, 1 << 20])
def test_pages_outside_the_pool_read_as_zeros(op, bad):
    dev = need_cuda()
    s = Setup([40, 33], new=None if op == "decode" else [3, 2], heads=4, kv_heads=2, d=64, stale=0.0, spare=1)
    # the oracle's page of zeros: a spare one
    used = set(s.table[s.table >= 0].tolist())
    spare = next(i for i in range(s.pages) if i not in used)
    s.table[0, 1] = spare
    ref = s.attention(s.d ** -0.5, op == "extend")
    s.table[0, 1] = bad
    status = cbq.PagedBatch.new_status(dev)
    got = run(s, op, dev, status=status)
    check_attention(got, *ref)
    assert int(status[0]) & L.FLAG_CORRUPT
    with pytest.raises(L.CbqError):
        cbq.paged.check_status(status)


def test_lengths_above_the_table_are_cut():
    dev = need_cuda()
    s = Setup([48, 33], heads=4, kv_heads=2, d=64)
    ref = s.attention(s.d ** -0.5, False)
    status = cbq.PagedBatch.new_status(dev)
    b = s.batch(cbq, dev, decode=True, status=status)
    b.kv_lens[0] = 1000
    k, v = s.pools(dev)
    check_attention(cbq.PagedKVCache(k, v).attend_decode(b, s.q.to(dev)), *ref)
    assert int(status[0]) & L.FLAG_CORRUPT
    status = cbq.PagedBatch.new_status(dev)
    run(s, "decode", dev, status=status)
    assert int(status[0]) == 0
    cbq.paged.check_status(status)


def test_sequences_that_share_pages():
    """Two sequences may name the same pages (a forked conversation)."""
    dev = need_cuda()
    s = Setup([100, 90], heads=4, kv_heads=2, d=64)
    s.table[1] = s.table[0]
    verify(s, "decode", dev)


def test_offsets_past_32_bits():
    """A pool of more than 2^31 elements: rows at its end."""
    dev = need_cuda()
    page, d, hkv = 256, 128, 8
    pages = (1 << 31) // (page * d * hkv) + 40
    k = torch.empty(pages, hkv, page, d, dtype=torch.bfloat16, device=dev)
    v = torch.empty_like(k)
    s = Setup([700, 513], heads=8, kv_heads=hkv, d=d, page=page)
    far = pages - s.pages
    k[far:] = s.k.to(dev)
    v[far:] = s.v.to(dev)
    ref = s.attention(s.d ** -0.5, False)
    s.table = torch.where(s.table >= 0, s.table + far, s.table)
    got = cbq.PagedKVCache(k, v).attend_decode(s.batch(cbq, dev, decode=True), s.q.to(dev))
    check_attention(got, *ref)


def test_empty_calls():
    dev = need_cuda()
    s = Setup([3, 4], new=[0, 0], heads=4, kv_heads=2, d=64)
    assert run(s, "extend", dev).shape == (0, 4, 64)
    e = torch.empty(0, 1, dtype=torch.int32, device=dev)
    b = cbq.PagedBatch(e, torch.empty(0, dtype=torch.int32, device=dev))
    k, v = s.pools(dev)
    assert cbq.PagedKVCache(k, v).attend_decode(b, s.q.to(dev)).shape == (0, 4, 64)


# ------------------------------------------------------------------- append
def tables(d, n):
    qd = __import__("importlib").import_module("codebook-quantization_b200.qwen3_decode")
    return qd.rope_tables(d, n, 1e6, "cpu")


def append_oracle(s, q, k, v, cos, sin, eps, qw, kw):
    kp, vp, out, scale = s.k.double(), s.v.double(), torch.zeros(s.tokens, s.heads, s.d, dtype=torch.float64), None
    h, t = s.d // 2, 0

    def turn(x, w, p):
        x = x.double()
        if eps >= 0:
            x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
            x = x if w is None else x * w.double()
        c, z = cos[p].double(), sin[p].double()
        return torch.cat((x[..., :h] * c[:h] - x[..., h:] * z[:h], x[..., h:] * c[h:] + x[..., :h] * z[h:]), -1)

    for i in range(s.n):
        for a in range(s.new[i]):
            r = s.kv[i] - s.new[i] + a
            if r >= 0:
                p = r + (s.plens[s.group_of[i]] if s.group_of[i] >= 0 else 0)
                page, line = s.table[i, r // s.page], r % s.page
                out[t] = turn(q[t], qw, p)
                kp[page, :, line] = turn(k[t], kw, p)
                vp[page, :, line] = v[t].double()
            t += 1
    return out, kp, vp


def same(got, ref):
    """One rounding of an fp32 result: half an ulp of the type, and the fp32
    arithmetic of a norm and a rotation (a few 2^-24 of the values' size; the
    size of a rotated pair is bounded by the row's largest element times 2)."""
    g = got.double().cpu()
    assert torch.equal(g.isnan(), ref.isnan())
    u = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -24
    size = ref.nan_to_num(0.0).abs().amax(-1, keepdim=True) * 2
    tol = u * ref.abs() + 16 * 2.0 ** -24 * size
    assert bool(((g - ref).abs() <= tol).logical_or(ref.isnan()).all())


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("case", ["one", "decode", "prompts", "prefix"])
@pytest.mark.parametrize("norm", ["weights", "unit", "none"])
def test_append(dt, d, case, norm):
    dev = need_cuda()
    kw = dict(d=d, dtype=DT[dt], heads=6, kv_heads=2)
    s = {"one": lambda: Setup([33], **kw),
         "decode": lambda: Setup([1, 0, 16, 17, 300], page=32, layout="nhd", **kw),
         "prompts": lambda: Setup([40, 5, 90, 64], new=[40, 0, 3, 17], page=16, layout="joint", **kw),
         "prefix": lambda: Setup([40, 5, 90, 64], new=[7, 5, 1, 64], groups=[(1, 9), (3, 100)], page=64, **kw)}[case]()
    qkv = torch.randn(s.tokens, s.heads + 2 * s.kv_heads, d).to(DT[dt])
    q, k, v = qkv.split((s.heads, s.kv_heads, s.kv_heads), 1)
    cos, sin = tables(d, 500)
    qw, kw_ = (torch.rand(d) + 0.5, torch.rand(d) + 0.5) if norm == "weights" else (None, None)
    eps = -1.0 if norm == "none" else 1e-6
    kp, vp = s.pools(dev)
    status = cbq.PagedBatch.new_status(dev)
    on = qkv.to(dev)
    b = s.batch(cbq, dev, decode=case in ("one", "decode"), status=status)
    got = cbq.PagedKVCache(kp, vp).append_rope(
        b, on[:, :s.heads], on[:, s.heads:s.heads + s.kv_heads], on[:, s.heads + s.kv_heads:], cos.to(dev),
        sin.to(dev), eps=eps, q_weight=None if qw is None else qw.to(dev),
        k_weight=None if kw_ is None else kw_.to(dev))
    ref, rk, rv = append_oracle(s, q, k, v, cos, sin, eps, qw, kw_)
    same(got, ref)
    same(kp, rk)
    assert torch.equal(vp.cpu().nan_to_num(7.0), rv.to(DT[dt]).nan_to_num(7.0))
    assert int(status[0]) == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_append_many_tokens(dt):
    """The shape that thousands of tokens take, with more heads than one pass holds."""
    dev = need_cuda()
    s = Setup([1500, 40, 900], new=[1400, 0, 800], d=64, dtype=DT[dt], heads=30, kv_heads=15, page=64, stale=0.0)
    qkv = torch.randn(s.tokens, 60, 64).to(DT[dt])
    cos, sin = tables(64, 1500)
    kp, vp = s.pools(dev)
    on = qkv.to(dev)
    got = cbq.PagedKVCache(kp, vp).append_rope(s.batch(cbq, dev), on[:, :30], on[:, 30:45], on[:, 45:], cos.to(dev),
                                               sin.to(dev))
    ref, rk, rv = append_oracle(s, qkv[:, :30], qkv[:, 30:45], qkv[:, 45:], cos, sin, 1e-6, None, None)
    same(got, ref)
    same(kp, rk)
    assert torch.equal(vp.cpu(), rv.to(DT[dt]))


def test_append_outside_the_tables_writes_nothing():
    dev = need_cuda()
    s = Setup([33, 16, 20, 8], heads=4, kv_heads=2, d=64, stale=0.0)
    s.table[0, 2] = s.pages                            # no such page
    cos, sin = tables(64, 18)                          # no position 19 (sequence 2)
    qkv = torch.randn(4, 8, 64, device=dev).to(torch.bfloat16)
    kp, vp = s.pools(dev)
    k0, v0 = kp.clone(), vp.clone()
    status = cbq.PagedBatch.new_status(dev)
    b = s.batch(cbq, dev, decode=True, status=status)
    b.kv_lens[1] = 500                                 # beyond the table's row
    got = cbq.PagedKVCache(kp, vp).append_rope(b, qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cos.to(dev), sin.to(dev))
    assert not got[:3].any() and got[3].any()
    page = int(s.table[3, 0])
    assert not torch.equal(kp[page], k0[page])
    kp[page], vp[page] = k0[page], v0[page]
    assert torch.equal(kp, k0) and torch.equal(vp, v0)
    assert int(status[0]) & L.FLAG_CORRUPT and int(status[2]) == 3


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("pad", [(0, 5), (3, 0), (2, 2100)], ids=str)
def test_append_skips_tokens_of_no_sequence(dt, pad):
    """Tokens before the first sequence's or behind the last one's: nothing
    written (the table's unused entries name another sequence's page), zeros back."""
    dev = need_cuda()
    s = Setup([20, 30, 12], new=[7, 1, 12], heads=4, kv_heads=2, d=64, dtype=DT[dt], slack=200, stale=0.0)
    s.table = torch.where(s.table < 0, s.table[0, 0], s.table)
    before, behind = pad
    n = s.tokens + before + behind
    qkv = torch.randn(n, 8, 64).to(DT[dt])
    mine = qkv[before:before + s.tokens]
    cos, sin = tables(64, 3000)
    kp, vp = s.pools(dev)
    status = cbq.PagedBatch.new_status(dev)
    b = s.batch(cbq, dev, status=status)
    b.cu_tokens.add_(before)
    on = qkv.to(dev)
    got = cbq.PagedKVCache(kp, vp).append_rope(b, on[:, :4], on[:, 4:6], on[:, 6:], cos.to(dev), sin.to(dev))
    ref, rk, rv = append_oracle(s, mine[:, :4], mine[:, 4:6], mine[:, 6:], cos, sin, 1e-6, None, None)
    same(got[before:before + s.tokens], ref)
    same(kp, rk)
    assert torch.equal(vp.cpu(), rv.to(DT[dt]))
    assert not got[:before].any() and not got[before + s.tokens:].any()
    assert int(status[0]) == 0


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("pad", [(0, 5), (3, 0), (2, 300)], ids=str)
@pytest.mark.parametrize("kv,new", [([20, 30, 12], [7, 1, 12]), ([700, 50], [600, 50]), ([2000], [100]), ([8, 8], [0, 0])],
                         ids=["few", "many", "long", "none"])
def test_extend_gives_zeros_for_tokens_of_no_sequence(dt, kv, new, pad):
    """Row and tile kernel, results written by the units and by the join."""
    dev = need_cuda()
    s = Setup(kv, new=new, heads=8, kv_heads=2, d=64, dtype=DT[dt], page=64)
    before, behind = pad
    n = s.tokens + before + behind
    k, v = s.pools(dev)
    b = s.batch(cbq, dev)
    b.cu_tokens.add_(before)
    q = torch.randn(n, 8, 64, device=dev).to(DT[dt])
    q[before:before + s.tokens] = s.q.to(dev)
    out = torch.full_like(q, float("nan"))
    cbq.PagedKVCache(k, v).attend_extend(b, q, out=out)
    assert not out[:before].any() and not out[before + s.tokens:].any()
    if s.tokens:
        check_attention(out[before:before + s.tokens], *s.attention(64 ** -0.5, True))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_captured_step_with_fewer_tokens_than_captured(dt):
    """Append and extend in one graph; the token counts change between replays."""
    dev = need_cuda()
    n = 24
    s = Setup([40, 24, 9], new=[10, 8, 6], heads=4, kv_heads=2, d=64, dtype=DT[dt], stale=0.0, slack=2)
    s.table = torch.where(s.table < 0, s.table[0, 0], s.table)
    cos, sin = (t.to(dev) for t in tables(64, 200))
    kp, vp = s.pools(dev)
    b, c = s.batch(cbq, dev), cbq.PagedKVCache(kp, vp)
    qkv = torch.randn(n, 8, 64, device=dev).to(DT[dt])
    out = torch.empty(n, 4, 64, dtype=DT[dt], device=dev)

    def step():
        q = c.append_rope(b, qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cos, sin)
        c.attend_extend(b, q, out=out)
        return q

    k0, v0 = kp.clone(), vp.clone()
    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        rotated = step()
    for new in ([10, 8, 6], [1, 1, 1], [3, 0, 0], [0, 0, 0], [10, 8, 6]):
        kp.copy_(k0)
        vp.copy_(v0)
        s.new, s.tokens = new, sum(new)
        b.cu_tokens.copy_(torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        on = qkv[:s.tokens].cpu()
        s.k, s.v = k0.cpu(), v0.cpu()
        ref, rk, rv = append_oracle(s, on[:, :4], on[:, 4:6], on[:, 6:], cos.cpu(), sin.cpu(), 1e-6, None, None)
        same(rotated[:s.tokens], ref)
        same(kp, rk)
        assert torch.equal(vp.cpu(), rv.to(DT[dt]))
        assert not rotated[s.tokens:].any() and not out[s.tokens:].any()
        if s.tokens:
            s.k, s.v, s.q = kp.cpu(), vp.cpu(), rotated[:s.tokens].cpu()
            check_attention(out[:s.tokens], *s.attention(64 ** -0.5, True))


def test_threads_that_share_a_stream():
    """A call is up to three launches over the stream's scratch; those of another
    thread's call must not come between them."""
    dev = need_cuda()
    cases = [(Setup([40, 0, 300, 17], groups=[(4, 500)], heads=8, kv_heads=2, d=128, seed=1), "decode"),
             (Setup([(9 * i) % 90 for i in range(30)], groups=[(10, 90), (20, 700)], heads=8, kv_heads=2, d=64, seed=2),
              "decode"),
             (Setup([700, 90], new=[60, 30], heads=8, kv_heads=2, d=128, seed=3), "extend"),
             (Setup([25, 600], groups=[(2, 77)], heads=8, kv_heads=2, d=64, dtype=torch.float32, seed=4), "decode")]
    calls = []
    for s, op in cases:
        k, v = s.pools(dev)
        c, b, q = cbq.PagedKVCache(k, v), s.batch(cbq, dev, decode=op == "decode"), s.q.to(dev)
        f = c.attend_decode if op == "decode" else c.attend_extend
        calls.append((f, b, q, f(b, q)))
    torch.cuda.synchronize()
    wrong, interval = [], sys.getswitchinterval()
    start = threading.Barrier(len(calls))

    def work(i):
        f, b, q, want = calls[i]
        start.wait()
        outs = [f(b, q) for _ in range(300)]
        wrong.append(sum(not torch.equal(o, want) for o in outs))

    sys.setswitchinterval(1e-6)
    try:
        threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    finally:
        sys.setswitchinterval(interval)
    assert wrong == [0] * len(calls)


@pytest.mark.parametrize("d", [64, 128])
def test_counters_are_zero_after_every_call(d):
    """What lets calls of any shape share a workspace: its first 16 KB count arrivals."""
    dev = need_cuda()
    ws = torch.zeros(64 << 20, dtype=torch.uint8, device=dev)
    for kv, new, heads in (([700, 90], [600, 90], 8), ([3000], [1], 8), ([64] * 20, [64] * 20, 4), ([900] * 3, None, 4)):
        s = Setup(kv, new=new, heads=heads, kv_heads=2, d=d, page=64)
        k, v = s.pools(dev)
        c, b = cbq.PagedKVCache(k, v), s.batch(cbq, dev, decode=new is None)
        f = c.attend_decode if new is None else c.attend_extend
        check_attention(f(b, s.q.to(dev), workspace=ws), *s.attention(d ** -0.5, new is not None))
        assert not ws[:16384].any()


@pytest.mark.parametrize("op", ["decode", "extend"])
def test_one_batch_over_pools_of_different_layouts(op):
    """Padded pages go to the row kernel, whole ones to the tile kernel: other workspaces."""
    dev = need_cuda()
    s = Setup([300, 200, 500], new=None if op == "decode" else [300, 200, 100], groups=[(3, 90)], heads=32, kv_heads=4,
              d=128)
    b, q = s.batch(cbq, dev, decode=op == "decode"), s.q.to(dev)
    shape, each = s.k.shape, s.k[0].numel()
    padded = []
    for x in (s.k, s.v):
        t = torch.empty(shape[0], each + 8, dtype=x.dtype, device=dev)[:, :each].unflatten(1, shape[1:])
        t.copy_(x)
        padded.append(t)
    ref = s.attention(s.d ** -0.5, op == "extend")
    for k, v in (padded, s.pools(dev), padded):
        c = cbq.PagedKVCache(k, v)
        f = c.attend_decode if op == "decode" else c.attend_extend
        n = c.workspace_bytes(b, s.tokens, 32, op == "extend")
        check_attention(f(b, q, workspace=torch.zeros(n, dtype=torch.uint8, device=dev)), *ref)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("op", ["decode", "extend"])
@pytest.mark.parametrize("what", ["inf value", "-inf value", "largest value", "lowest value", "-inf key", "lowest key",
                                  "largest query"])
def test_infinities_and_largest_values_inside_the_lengths(what, op, d, dt):
    """A visible value of inf gives inf where its weight is not 0; a key of -inf
    or of the type's lowest value takes its row out; a prefix and own rows."""
    dev = need_cuda()
    new = None if op == "decode" else [40, 2, 17]
    s = Setup([90, 100, 67], new=new, groups=[(3, 50)], heads=4, kv_heads=2, d=d, dtype=DT[dt])
    slack = s.attention(d ** -0.5, op == "extend")[2]
    top = torch.finfo(DT[dt]).max
    number = {"inf": math.inf, "-inf": -math.inf, "largest": top, "lowest": -top}[what.split()[0]]
    pages = ((s.table[0, 0], 5), (s.table[1, 3], 2), (s.ptable[0, 1], 9), (s.table[2, 0], 3))
    if what.endswith("query"):
        # one query's largest element against keys of 0 but for a small one: scores stay finite
        s.k[..., 7] = torch.where(s.k[..., 7].isnan(), s.k[..., 7], torch.zeros_like(s.k[..., 7]))
        s.k[pages[0][0], :, pages[0][1], 7] = 2.0 ** -124
        s.q[:, :, 7] = number
    for page, line in pages:
        if what.endswith("value"):
            s.v[page, :, line, 7] = number
        elif what.endswith("key"):
            s.k[page, :, line, 7] = number
            s.q[:, :, 7] = 0.25
    ref, spread, changed = s.attention(d ** -0.5, op == "extend")
    # what bounds the scores' errors: a key that is taken out does not count, one element of the others moved
    slack = changed if not what.endswith("key") else 2 * slack
    got = run(s, op, dev)
    finite = ref.isfinite()
    assert torch.equal(got.double().cpu()[~finite], ref[~finite])
    if what.endswith("inf value"):
        assert not finite.all()
    u = 2.0 ** -8 if dt == "bf16" else 2.0 ** -23
    tol = u * ref.abs() + ((2.0 ** -8 if dt == "bf16" else 0.0) + slack) * spread + 1e-30
    assert bool(((got.double().cpu() - ref).abs()[finite] <= tol[finite]).all())


@pytest.mark.parametrize("op", ["decode", "extend"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_tables_without_columns(op, dt):
    """No own rows at all, or no prefix: an empty table, whose address may be null."""
    dev = need_cuda()
    new = None if op == "decode" else [40, 2]
    s = Setup([0, 0], new=new, groups=[(1, 30), (1, 70)], heads=4, kv_heads=2, d=64, dtype=DT[dt])
    s.table = s.table[:, :0]
    verify(s, op, dev)
    s = Setup([50, 9], new=new, groups=[(1, 0), (1, 0)], heads=4, kv_heads=2, d=64, dtype=DT[dt])
    s.ptable = s.ptable[:, :0]
    verify(s, op, dev)
    s = Setup([0, 0], new=new, heads=4, kv_heads=2, d=64, dtype=DT[dt])
    s.table = s.table[:, :0]
    assert not verify(s, op, dev).any()
    qkv = torch.randn(s.tokens, 8, 64, device=dev).to(DT[dt])
    cos, sin = tables(64, 8)
    kp, vp = s.pools(dev)
    before = kp.clone()
    got = cbq.PagedKVCache(kp, vp).append_rope(s.batch(cbq, dev, decode=op == "decode"), qkv[:, :4], qkv[:, 4:6],
                                               qkv[:, 6:], cos.to(dev), sin.to(dev))
    assert not got.any() and torch.equal(kp.nan_to_num(7.0), before.nan_to_num(7.0))


@pytest.mark.parametrize("op", ["decode", "extend"])
@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("rows", [48, 0])
def test_prefixes_above_their_table_are_cut_and_reported(rows, op, dt):
    dev = need_cuda()
    s = Setup([48, 33, 60], new=None if op == "decode" else [40, 33, 2], groups=[(1, 16), (2, rows)], heads=4, kv_heads=2,
              d=64, dtype=DT[dt])
    if rows == 0:
        s.plens[0], s.groups = 0, [(1, 0), (2, 0)]
        s.ptable = s.ptable[:, :0]                     # a table that names nothing
    ref = s.attention(s.d ** -0.5, op == "extend")
    status = cbq.PagedBatch.new_status(dev)
    b = s.batch(cbq, dev, decode=op == "decode", status=status)
    k, v = s.pools(dev)
    c, q = cbq.PagedKVCache(k, v), s.q.to(dev)
    f = c.attend_decode if op == "decode" else c.attend_extend
    check_attention(f(b, q), *ref)
    assert int(status[0]) == 0
    b.prefix_lens[1] = 1000
    check_attention(f(b, q), *ref)
    assert int(status[0]) == L.FLAG_CORRUPT and int(status[1]) == 1


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("tokens", [148, 149, 741, 1037, 1185, 1481, 2221])
def test_append_around_the_waves(dt, tokens):
    """Both shapes of the kernel, on either side of what the GPU holds at once."""
    dev = need_cuda()
    s = Setup([tokens + 5, 3], new=[tokens - 2, 2], d=64, dtype=DT[dt], heads=3, kv_heads=1, page=64, stale=0.0)
    qkv = torch.randn(tokens, 5, 64).to(DT[dt])
    cos, sin = tables(64, tokens + 5)
    kp, vp = s.pools(dev)
    on = qkv.to(dev)
    got = cbq.PagedKVCache(kp, vp).append_rope(s.batch(cbq, dev), on[:, :3], on[:, 3:4], on[:, 4:], cos.to(dev),
                                               sin.to(dev))
    ref, rk, rv = append_oracle(s, qkv[:, :3], qkv[:, 3:4], qkv[:, 4:], cos, sin, 1e-6, None, None)
    same(got, ref)
    same(kp, rk)
    assert torch.equal(vp.cpu(), rv.to(DT[dt]))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("seqs", [1, 5, 20])
@pytest.mark.parametrize("new", [2, 4, 6])
def test_extend_a_few_tokens_of_each_sequence(d, seqs, new):
    """8 to 24 query rows a kv head, few units and many: either kernel."""
    dev = need_cuda()
    verify(Setup([200 + 7 * i for i in range(seqs)], new=[new] * seqs, heads=16, kv_heads=4, d=d), "extend", dev)


def test_a_prompt_chunk_among_single_tokens():
    """Continuous batching: one kernel for the batch, by its mean."""
    dev = need_cuda()
    for chunk, singles in ((300, 40), (900, 20)):
        kv = [chunk + 50] + [(37 * i) % 300 + 1 for i in range(singles)]
        verify(Setup(kv, new=[chunk] + [1] * singles, groups=[(singles + 1, 40)], heads=8, kv_heads=2, d=128, page=32),
               "extend", dev)


@pytest.mark.parametrize("dt", ["bf16", "f32"])
def test_extend_and_append_past_32_bits(dt):
    """Rows at the end of a pool of more than 2^31 elements, by both kernels."""
    dev = need_cuda()
    page, d, hkv = 256, 128, 8
    pages = (1 << 31) // (page * d * hkv) + 40
    k = torch.empty(pages, hkv, page, d, dtype=DT[dt], device=dev)
    v = torch.empty_like(k)
    for new in ([300, 213], [3, 1]):
        s = Setup([700, 513], new=new, groups=[(2, 300)], heads=16, kv_heads=hkv, d=d, page=page, dtype=DT[dt], stale=0.0)
        far = pages - s.pages
        k[far:] = s.k.to(dev)
        v[far:] = s.v.to(dev)
        s.table = torch.where(s.table >= 0, s.table + far, s.table)
        s.ptable = torch.where(s.ptable < 1 << 20, s.ptable + far, s.ptable)
        b, c = s.batch(cbq, dev), cbq.PagedKVCache(k, v)
        near = (s.table - far, s.ptable - far)
        s.table, s.ptable = (torch.where(t < 0, -1, t) for t in near)
        check_attention(c.attend_extend(b, s.q.to(dev)), *s.attention(d ** -0.5, True))
        qkv = torch.randn(s.tokens, 32, d).to(DT[dt])
        cos, sin = tables(d, 1100)
        on = qkv.to(dev)
        got = c.append_rope(b, on[:, :16], on[:, 16:24], on[:, 24:], cos.to(dev), sin.to(dev))
        ref, rk, rv = append_oracle(s, qkv[:, :16], qkv[:, 16:24], qkv[:, 24:], cos, sin, 1e-6, None, None)
        same(got, ref)
        same(k[far:], rk)
        assert torch.equal(v[far:].cpu(), rv.to(DT[dt]))


@pytest.mark.parametrize("dt", ["bf16", "f32"])
@pytest.mark.parametrize("new", [1, 30])
@pytest.mark.parametrize("inside", [(1, 2), (0, 2), (3, 2), (2, 0)], ids=str)
def test_sequences_in_no_group_have_no_prefix(inside, new, dt):
    """Groups that begin behind the first sequence or end before the last one."""
    dev = need_cuda()
    first, n = inside
    s = Setup([40, 90, 31, 64, 300], new=[new] * 5, groups=[(first, 0), (n, 70), (5 - first - n, 0)], heads=4, kv_heads=2,
              d=64, dtype=DT[dt], stale=0.0)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    shared = dict(group_starts=i32([first, first + n]), prefix_lens=i32([70]), prefix_table=s.ptable[1:2].to(dev))
    cu = i32([new * i for i in range(6)])
    k, v = s.pools(dev)
    c, b = cbq.PagedKVCache(k, v), cbq.PagedBatch(s.table.to(dev), i32(s.kv), cu_tokens=cu, **shared)
    check_attention(c.attend_extend(b, s.q.to(dev)), *s.attention(64 ** -0.5, True))
    if new == 1:
        check_attention(c.attend_decode(b, s.q.to(dev)), *s.attention(64 ** -0.5, False))
    qkv = torch.randn(s.tokens, 8, 64).to(DT[dt])
    cos, sin = tables(64, 400)
    on = qkv.to(dev)
    got = c.append_rope(b, on[:, :4], on[:, 4:6], on[:, 6:], cos.to(dev), sin.to(dev))
    ref, rk, rv = append_oracle(s, qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], cos, sin, 1e-6, None, None)
    same(got, ref)
    same(k, rk)
    b.check()
