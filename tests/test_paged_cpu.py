"""What the paged-cache operators refuse, on the host, before any CUDA call."""
import contextlib
import ctypes as ct
import struct

import pytest
import torch

from helpers import cbq

L = cbq._lib
lib = L.lib


def cache(**kw):
    f = dict(k=4096, v=8192, pages=4, kv_heads=2, page_size=16, head_dim=64, page_stride=2048, head_stride=1024,
             row_stride=64, dtype=L.CBQ_BF16)
    f.update(kw)
    return ct.create_string_buffer(struct.pack("<10q", *f.values()), 80)


def batch(**kw):
    f = dict(seqs=2, cu=0, lens=64, table=64, width=3, stride=3, max_kv=48, groups=0, gs=0, plens=0, ptable=0, pwidth=0,
             pstride=0, max_prefix=0, status=0)
    f.update(kw)
    return ct.create_string_buffer(struct.pack("<15q", *f.values()), 120)


def attend(c, b, tokens=2, q=256, qs=256, heads=4, out=512, ws=0, nws=0, name="cbq_paged_attn_decode"):
    return getattr(lib(), name)(c, b, tokens, q, qs, heads, 0.125, out, ws, nws, None)


def append(c, b, tokens=2, q=256, qs=256, k=256, ks=128, v=256, vs=128, heads=4, cos=256, sin=256, n=10, out=512):
    return lib().cbq_paged_append_rope(c, b, tokens, q, qs, k, ks, v, vs, heads, 1e-6, None, None, cos, sin, n, out, None)


ARG, NO = L.CBQ_ERR_ARG, L.CBQ_ERR_UNSUPPORTED


@pytest.mark.parametrize("bad,rc", [
    (dict(dtype=2), ARG), (dict(pages=-1), ARG), (dict(kv_heads=0), ARG), (dict(kv_heads=3), ARG),
    (dict(head_dim=96), NO), (dict(page_size=8), NO), (dict(page_size=48), NO), (dict(page_size=512), NO),
    (dict(k=0), ARG), (dict(v=0), ARG), (dict(k=4100), ARG), (dict(row_stride=32), ARG), (dict(row_stride=68), ARG),
    (dict(page_stride=2052), ARG), (dict(head_stride=-64), ARG)], ids=str)
def test_cache_refusals(bad, rc):
    assert attend(cache(**bad), batch()) == rc
    assert attend(cache(**bad), batch(), name="cbq_paged_attn_extend") == rc
    assert append(cache(**bad), batch()) == rc


@pytest.mark.parametrize("bad,rc", [
    (dict(seqs=-1), ARG), (dict(lens=0), ARG), (dict(table=0), ARG), (dict(stride=2), ARG), (dict(width=-1), ARG),
    (dict(max_kv=-1), ARG), (dict(groups=3), ARG), (dict(groups=1), ARG), (dict(groups=-1), ARG),
    (dict(groups=1, gs=64, plens=64, ptable=64, pwidth=2, pstride=1), ARG), (dict(seqs=70000), NO),
    (dict(seqs=3), ARG), (dict(width=1 << 28, stride=1 << 28), NO)], ids=str)
def test_batch_refusals(bad, rc):
    assert attend(cache(), batch(**bad)) == rc
    assert append(cache(), batch(**bad)) == rc


def test_null_descriptors():
    assert attend(None, batch()) == ARG and attend(cache(), None) == ARG
    assert append(None, batch()) == ARG and append(cache(), None) == ARG
    assert lib().cbq_paged_attn_workspace_bytes(None, None, 1, 1, 0) == -1


def test_append_argument_refusals():
    c, b = cache(), batch()
    for bad in (dict(q=0), dict(k=0), dict(v=0), dict(cos=0), dict(sin=0), dict(out=0), dict(q=264), dict(out=520),
                dict(qs=128), dict(ks=64), dict(vs=132), dict(qs=260), dict(n=-1), dict(heads=3), dict(heads=0),
                dict(tokens=-1), dict(tokens=1)):
        assert append(c, b, **bad) == ARG, bad
    assert append(c, b, heads=2 * 65, qs=2 * 65 * 64) == NO
    assert append(cache(), batch(seqs=0, lens=0, table=0), tokens=0) == L.CBQ_OK


def test_nothing_to_do_is_ok():
    assert attend(cache(), batch(seqs=0), tokens=0) == L.CBQ_OK
    assert attend(cache(), batch(cu=64), tokens=0, name="cbq_paged_attn_extend") == L.CBQ_OK
    assert attend(cache(), batch(seqs=0, cu=64), tokens=3, name="cbq_paged_attn_extend") == ARG


def test_python_refusals():
    k = torch.zeros(4, 2, 16, 64)
    with pytest.raises(RuntimeError):
        cbq.PagedKVCache(k, k)                         # no CPU fallback
    t, n = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    cbq.PagedBatch(t, n)
    for a, kw in (((t.long(), n), {}), ((t, n.long()), {}), ((t[0], n), {}), ((t[:1], n), {}),
                  ((t, n), dict(cu_tokens=n)), ((t, n), dict(prefix_lens=n)),
                  ((t, n), dict(prefix_lens=n, group_starts=n, prefix_table=t)),
                  ((t, n), dict(status=n)), ((t.T.contiguous().T, n), {})):
        with pytest.raises(ValueError):
            cbq.PagedBatch(*a, **kw)


class Stub:
    """A cache whose tensors are on the CPU and whose library calls are
    recorded instead of made: what reaches the library, without a GPU."""

    def __init__(self, monkeypatch, shape=(4, 2, 16, 64), strides=None):
        self.calls, self.device = [], -1               # a CPU tensor's device number
        monkeypatch.setattr(cbq.paged, "_run", lambda name, *a: self.calls.append((name, self.device)))
        monkeypatch.setattr(cbq.paged, "_current", lambda: self.device, raising=False)
        monkeypatch.setattr(cbq.paged, "_stream", lambda i: 0)
        k = torch.zeros(shape) if strides is None else torch.empty_strided(shape, strides)
        monkeypatch.setattr(cbq.paged.torch.Tensor, "is_cuda", True, raising=False)
        self.cache = cbq.PagedKVCache(k, k.clone() if strides is None else torch.empty_strided(shape, strides))
        self.ws = torch.zeros(1 << 20, dtype=torch.uint8)

    def attend(self, b, **kw):
        return self.cache.attend_decode(b, torch.zeros(2, 4, 64), **{"workspace": self.ws, **kw})

    def append(self, b):
        k = torch.zeros(2, 2, 64)
        t = torch.zeros(8, 64)
        return self.cache.append_rope(b, torch.zeros(2, 4, 64), k, k, t, t)


def tables(device="cpu"):
    return torch.zeros(2, 3, dtype=torch.int32, device=device), torch.zeros(2, dtype=torch.int32, device=device)


def test_a_batch_on_another_device_is_refused(monkeypatch):
    s = Stub(monkeypatch)
    far = cbq.PagedBatch(*tables("meta"))
    for call in (s.attend, s.append, lambda b: s.cache.workspace_bytes(b, 2, 4, False),
                 lambda b: s.cache.attend_extend(b, torch.zeros(2, 4, 64), workspace=s.ws)):
        with pytest.raises(ValueError):
            call(far)
    assert not s.calls
    s.attend(cbq.PagedBatch(*tables()))
    s.append(cbq.PagedBatch(*tables()))
    assert [c for c, _ in s.calls] == ["cbq_paged_attn_decode", "cbq_paged_append_rope"]


@pytest.mark.parametrize("ws", [torch.empty(1 << 16, dtype=torch.uint8, device="meta"), torch.zeros(1 << 16),
                                torch.zeros(1 << 17, dtype=torch.uint8)[::2]], ids=["device", "dtype", "strided"])
def test_a_workspace_of_another_kind_is_refused(monkeypatch, ws):
    s = Stub(monkeypatch)
    with pytest.raises(ValueError):
        s.attend(cbq.PagedBatch(*tables()), workspace=ws)
    assert not s.calls


def strides_of(b):
    f = struct.unpack("<15q", b._desc.raw)
    return f[5], f[12]                                 # table_stride, prefix_stride


def test_tables_whose_rows_overlap_are_refused():
    """An expanded row was read with a stride of its width, past its storage."""
    n, gs, pl = torch.zeros(4, dtype=torch.int32), torch.tensor([0, 2, 4], dtype=torch.int32), torch.zeros(
        2, dtype=torch.int32)
    row = torch.zeros(1, 3, dtype=torch.int32)
    for table in (row.expand(4, -1), torch.zeros(12, dtype=torch.int32).unfold(0, 6, 2)):
        with pytest.raises(ValueError):
            cbq.PagedBatch(table, n)
        with pytest.raises(ValueError):
            cbq.PagedBatch(torch.zeros(4, 3, dtype=torch.int32), n, group_starts=gs, prefix_lens=pl,
                           prefix_table=table[:2])
    assert strides_of(cbq.PagedBatch(row.expand(4, -1).contiguous(), n)) == (3, 0)
    wide = torch.zeros(4, 9, dtype=torch.int32)
    one = cbq.PagedBatch(wide[:, :3], n, group_starts=gs, prefix_lens=pl, prefix_table=wide[:2, 4:8])
    assert strides_of(one) == (9, 9)
    assert strides_of(cbq.PagedBatch(row.expand(1, -1), n[:1])) == (3, 0)
    assert strides_of(cbq.PagedBatch(torch.zeros(4, 0, dtype=torch.int32), n)) == (1, 0)


def test_calls_run_on_the_device_of_the_cache(monkeypatch):
    """The library launches on the current device, which may be another one."""
    s = Stub(monkeypatch)
    entered = []

    @contextlib.contextmanager
    def device(index):
        entered.append(index)
        was, s.device = s.device, index
        yield
        s.device = was

    monkeypatch.setattr(torch.cuda, "device", device)
    s.device = 3
    s.attend(cbq.PagedBatch(*tables()))
    s.append(cbq.PagedBatch(*tables()))
    assert [d for _, d in s.calls] == [-1, -1] and entered == [-1, -1] and s.device == 3
    s.device = -1
    s.attend(cbq.PagedBatch(*tables()))
    assert len(entered) == 2


@pytest.mark.parametrize("flags,rc", [(0, None), (L.FLAG_CORRUPT, L.CBQ_ERR_CORRUPT),
                                      (L.FLAG_TIMEOUT, L.CBQ_ERR_TIMEOUT),
                                      (L.FLAG_TIMEOUT | L.FLAG_CORRUPT, L.CBQ_ERR_TIMEOUT)], ids=str)
def test_status_tells_what_was_recorded(flags, rc):
    b = cbq.PagedBatch(*tables())                      # a status of its own
    assert struct.unpack("<15q", b._desc.raw)[14] == b.status.data_ptr() and b.status.tolist() == [0, -1, 0, 0]
    b.status[0] = flags
    for check in (b.check, lambda: cbq.paged.check_status(b.status)):
        if rc is None:
            check()
        else:
            with pytest.raises(L.CbqError) as e:
                check()
            assert e.value.status == rc


def test_workspace_sizes_are_kept_by_layout(monkeypatch):
    """The kernel, and so the size, depends on the strides too."""
    shape, asked = (4, 2, 16, 64), []
    monkeypatch.setattr(L, "query", lambda name, cache, *a: asked.append(cache) or len(asked))
    flat, padded = (Stub(monkeypatch, shape, (n, 1024, 64, 1)).cache for n in (2048, 2056))
    b = cbq.PagedBatch(*tables())
    got = [c.workspace_bytes(b, 2, 4, True) for c in (padded, flat, padded, flat)]
    assert got == [1, 2, 1, 2] and asked == [padded._addr, flat._addr]


def test_held_tensors_cannot_be_replaced(monkeypatch):
    """A replaced tensor was freed while the kernels went on reading its address."""
    c, (t, n) = Stub(monkeypatch).cache, tables()
    b = cbq.PagedBatch(t, n)
    for o, name in ((b, "kv_lens"), (b, "page_table"), (b, "cu_tokens"), (b, "status"), (c, "k_pages"), (c, "v_pages")):
        with pytest.raises(AttributeError):
            setattr(o, name, tables()[1])
    b.kv_lens += 1
    b.kv_lens[0] = 5
    assert n.tolist() == [5, 1] and b.kv_lens is n
