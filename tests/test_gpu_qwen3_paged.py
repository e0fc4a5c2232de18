"""The paged path of the whole model: prompts in one pass, a shared prefix kept
once, a ragged batch decoded together, against the one-token-a-step decoder
run on every sequence by itself (fp32 activations: identical greedy tokens)."""
import importlib

import pytest
import torch

from helpers import cbq, need_cuda

pytestmark = pytest.mark.gpu
q3 = cbq.qwen3
qd = importlib.import_module("codebook-quantization_b200.qwen3_decode")
qp = importlib.import_module("codebook-quantization_b200.qwen3_paged")

TINY = q3.Qwen3Config("tiny", 2, 256, 512, 4, 2, 64, 1000, 1e6, False)


def alone(W, ids, n):
    dec = qd.Qwen3Decoder(W, batch=1, max_len=128, act_dtype=torch.float32)
    return dec.generate(ids[None], n).cpu()[0]


@pytest.mark.parametrize("huffman", [False, True], ids=["fixed", "huffman"])
@pytest.mark.parametrize("plen", [0, 1, 37])
@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_ragged_batch_matches_each_sequence_alone(huffman, plen, graph):
    dev = need_cuda()
    W = q3.CompressedQwen3Weights(TINY, dev, huffman=huffman, seed=5)
    g = torch.Generator().manual_seed(11)
    lens = [1, 5, 16, 33]
    prompts = [torch.randint(0, TINY.vocab, (n,), generator=g) for n in lens]
    prefix = torch.randint(0, TINY.vocab, (plen,), generator=g) if plen else None
    m = qp.PagedQwen3(W, pages=40, page_size=16, max_len=128, act_dtype=torch.float32)
    got = m.generate(prompts, 12, prefix=prefix, graph=graph).cpu()
    assert len(m.free) == 40
    for i, p in enumerate(prompts):
        want = alone(W, p if prefix is None else torch.cat((prefix, p)), 12)
        assert torch.equal(got[i], want), i


def test_bf16_runs_and_repeats():
    dev = need_cuda()
    W = q3.CompressedQwen3Weights(TINY, dev, seed=5)
    m = qp.PagedQwen3(W, pages=40, page_size=32, max_len=256)
    prompts = [torch.arange(40), torch.arange(3)]
    a = m.generate(prompts, 8, prefix=torch.arange(50))
    b = m.generate(prompts, 8, prefix=torch.arange(50))
    assert a.shape == (2, 8) and torch.equal(a, b)


def test_refusals():
    dev = need_cuda()
    W = q3.CompressedQwen3Weights(TINY, dev, seed=5)
    m = qp.PagedQwen3(W, pages=4, page_size=16, max_len=64, act_dtype=torch.float32)
    with pytest.raises(ValueError):
        m.generate([torch.arange(60)], 10)
    with pytest.raises(ValueError):
        m.generate([torch.arange(0)], 3)
    with pytest.raises(RuntimeError):
        m.generate([torch.arange(30), torch.arange(30)], 20)
    assert len(m.free) == 4


@pytest.mark.parametrize("graph", [False, True], ids=["eager", "graph"])
def test_an_error_that_a_kernel_reports_is_raised(graph):
    """A table entry outside the pool (nothing is read or written there)."""
    dev = need_cuda()
    m = qp.PagedQwen3(q3.CompressedQwen3Weights(TINY, dev, seed=5), pages=4, page_size=16, max_len=64)
    prompts = [torch.arange(5), torch.arange(9)]
    m.generate(prompts, 4, graph=graph)
    table = m._table
    m._table = lambda rows: table(rows) + 4
    with pytest.raises(cbq._lib.CbqError) as e:
        m.generate(prompts, 4, graph=graph)
    assert e.value.status == cbq._lib.CBQ_ERR_CORRUPT and len(m.free) == 4


def test_bf16_hidden_states_follow_fp32():
    """The same prompts and one decode step in both types: about 20 roundings of
    2^-9 a layer on the way, two layers, each of them random."""
    dev = need_cuda()
    W = q3.CompressedQwen3Weights(TINY, dev, seed=5)
    g = torch.Generator().manual_seed(3)
    lens, hidden = [40, 3, 100], {}
    ids = torch.randint(0, TINY.vocab, (sum(lens),), generator=g).to(dev)
    nxt = torch.randint(0, TINY.vocab, (3,), generator=g).to(dev)
    for dt in (torch.float32, torch.bfloat16):
        m = qp.PagedQwen3(W, pages=16, page_size=16, max_len=128, act_dtype=dt)
        table, kv = m._table([m._take(n + 1) for n in lens]), m._ints(lens)
        b = cbq.PagedBatch(table, kv, cu_tokens=m._ints([0, 40, 43, 143]))
        first = m.forward(ids, b, decode=False).double()
        kv.add_(1)
        b = cbq.PagedBatch(table, kv)
        hidden[dt] = first, m.forward(nxt, b, decode=True).double()
        b.check()
    for want, got in zip(*hidden.values()):
        assert float((got - want).norm() / want.norm()) < (2 * 20) ** 0.5 * 2.0 ** -8
