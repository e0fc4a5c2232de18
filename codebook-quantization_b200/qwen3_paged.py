"""Greedy decoding of a compressed Qwen3-architecture model over a paged cache.

Where :class:`qwen3_decode.Qwen3Decoder` steps a batch of equally long
sequences one token at a time, ``PagedQwen3`` takes prompts of any length in
one pass (``cbq_paged_attn_extend``; the linears run on the tensor-core GEMM
from three tokens on), keeps a common beginning of all prompts once
(``prefix=``), and decodes the ragged batch with ``cbq_paged_attn_decode``,
one captured CUDA graph for every step.

One GPU.  The layer's math is the decoder's (RMSNorm, q/k RMSNorm and rotary
embedding, grouped-query attention, SiLU-gated MLP, greedy argmax with the
first index on ties); q and k are rounded to the activation type once, after
the rotation.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import torch

from . import _lib
from .gpu_accelerated_functions import device_stream
from .paged import PagedBatch, PagedKVCache, check_status
from .qwen3 import CompressedQwen3Weights
from .qwen3_decode import rope_tables

__all__ = ["PagedQwen3"]


class PagedQwen3:
    """``pages`` pages of ``page_size`` rows per layer; ``max_len`` bounds a sequence, its prefix included."""

    def __init__(self, weights: CompressedQwen3Weights, pages: int, page_size: int = 16, max_len: int = 4096,
                 act_dtype=torch.bfloat16):
        if weights.world != 1:
            raise ValueError("PagedQwen3 runs on one GPU (use Qwen3Decoder for tensor parallelism)")
        self.w, self.cfg, self.dev, self.dt = weights, weights.cfg, weights.device, act_dtype
        c = self.cfg
        self.page_size, self.max_len = page_size, max_len
        self.cos, self.sin = rope_tables(c.head_dim, max_len, c.rope_theta, self.dev)
        self.code = _lib.CBQ_BF16 if act_dtype == torch.bfloat16 else _lib.CBQ_F32
        shape = (pages, c.kv_heads, page_size, c.head_dim)
        self.caches = [PagedKVCache(*(torch.zeros(shape, dtype=act_dtype, device=self.dev) for _ in range(2)))
                       for _ in range(c.layers)]
        self.free = list(range(pages - 1, -1, -1))
        L = weights.layers
        self.emb, self.lm_head = L["model.embed_tokens.weight"], L["lm_head.weight"]
        self.layers = [tuple(L[f"model.layers.{i}.{n}.weight"] for n in (
            "self_attn.q_proj", "self_attn.k_proj", "self_attn.v_proj", "self_attn.o_proj", "mlp.gate_proj",
            "mlp.up_proj", "mlp.down_proj")) for i in range(c.layers)]

    # ------------------------------------------------------------- page tables
    def _take(self, rows: int) -> List[int]:
        n = -(-rows // self.page_size)
        if n > len(self.free):
            raise RuntimeError(f"{n} pages wanted, {len(self.free)} free")
        return [self.free.pop() for _ in range(n)]

    def _give(self, pages: Sequence[int]) -> None:
        self.free.extend(pages)

    def _table(self, rows: Sequence[Sequence[int]]) -> torch.Tensor:
        t = torch.zeros(len(rows), max([1] + [len(r) for r in rows]), dtype=torch.int32)
        for i, r in enumerate(rows):
            t[i, :len(r)] = torch.tensor(r, dtype=torch.int32)
        return t.to(self.dev)

    def _ints(self, values: Sequence[int]) -> torch.Tensor:
        return torch.tensor(list(values), dtype=torch.int32, device=self.dev)

    # ----------------------------------------------------------------- forward
    def _norm(self, x: torch.Tensor, add: Optional[torch.Tensor] = None) -> torch.Tensor:
        """RMSNorm of x, after x += add in place."""
        h = torch.empty_like(x)
        _lib.call("cbq_rmsnorm", x.data_ptr(), None if add is None else add.data_ptr(), self.code, x.shape[0],
                  x.shape[1], None, float(self.cfg.rms_eps), h.data_ptr(), device_stream(self.dev))
        return h

    def forward(self, ids: torch.Tensor, batch: PagedBatch, decode: bool) -> torch.Tensor:
        """The final hidden states [tokens, hidden] (normalised) of the new
        tokens ``ids``, whose keys and values are left in the cache."""
        c, n = self.cfg, ids.shape[0]
        x = self.emb(ids, out_dtype=self.dt)
        h = self._norm(x)
        for cache, (q_p, k_p, v_p, o_p, g_p, u_p, d_p) in zip(self.caches, self.layers):
            q, k, v = (p(h).view(n, -1, c.head_dim) for p in (q_p, k_p, v_p))
            q = cache.append_rope(batch, q, k, v, self.cos, self.sin, eps=float(c.rms_eps))
            a = (cache.attend_decode if decode else cache.attend_extend)(batch, q)
            h = self._norm(x, add=o_p(a.view(n, -1)))
            g, u = g_p(h), u_p(h)
            _lib.call("cbq_silu_mul", g.data_ptr(), u.data_ptr(), self.code, g.numel(), g.data_ptr(),
                      device_stream(self.dev))
            h = self._norm(x, add=d_p(g))
        return h

    def _pick(self, h: torch.Tensor, out: torch.Tensor) -> None:
        logits = self.lm_head(h)
        code = _lib.CBQ_BF16 if logits.dtype == torch.bfloat16 else _lib.CBQ_F32
        _lib.call("cbq_greedy_pick", logits.data_ptr(), code, logits.shape[0], logits.shape[1], logits.shape[1], 0, 1,
                  None, None, None, out.data_ptr(), None, device_stream(self.dev))

    # ---------------------------------------------------------------- generate
    def generate(self, prompts: Sequence[torch.Tensor], n_new: int, prefix: Optional[torch.Tensor] = None,
                 graph: bool = True) -> torch.Tensor:
        """Greedy tokens [len(prompts), n_new] after each prompt (1-D token
        ids, one token at least); ``prefix``: token ids that stand before all
        of them, computed and kept once.  Raises if a kernel reported an error."""
        lens = [int(p.numel()) for p in prompts]
        plen = 0 if prefix is None else int(prefix.numel())
        if not lens or min(lens) < 1 or n_new < 1:
            raise ValueError("prompts of one token at least and one new token at least")
        if plen + max(lens) + n_new > self.max_len:
            raise ValueError("sequence longer than max_len")
        held: List[List[int]] = []
        status = PagedBatch.new_status(self.dev)
        try:
            shared = {}
            if plen:
                held.append(self._take(plen))
                b = PagedBatch(self._table(held[:1]), self._ints([plen]), cu_tokens=self._ints([0, plen]), max_kv_len=plen,
                               status=status)
                self.forward(prefix.to(self.dev).long(), b, decode=False)
                shared = dict(group_starts=self._ints([0, len(lens)]), prefix_lens=self._ints([plen]),
                              prefix_table=self._table(held[:1]), max_prefix_len=plen)
            for n in lens:
                held.append(self._take(n + n_new))
            own = held[-len(lens):]
            table, kv = self._table(own), self._ints(lens)
            cu = self._ints([0] + torch.tensor(lens).cumsum(0).tolist())
            # the prompts in one pass, then one token of each at a time
            b = PagedBatch(table, kv, cu_tokens=cu, max_kv_len=max(lens), status=status, **shared)
            h = self.forward(torch.cat([p.reshape(-1) for p in prompts]).to(self.dev).long(), b, decode=False)
            nxt = torch.zeros(len(lens), dtype=torch.int64, device=self.dev)
            self._pick(h.index_select(0, cu[1:].long() - 1), nxt)
            out = torch.empty(len(lens), n_new, dtype=torch.int64, device=self.dev)
            b = PagedBatch(table, kv, max_kv_len=max(lens) + n_new, status=status, **shared)

            def step():
                kv.add_(1)
                self._pick(self.forward(nxt, b, decode=True), nxt)

            g = None
            for t in range(n_new):
                out[:, t].copy_(nxt)
                if t + 1 == n_new:
                    break
                if g is not None:
                    g.replay()
                elif graph and t:                      # the first step ran eagerly and warmed everything up
                    torch.cuda.synchronize(self.dev)
                    g = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(g):
                        step()
                    g.replay()
                else:
                    step()
            torch.cuda.synchronize(self.dev)
            check_status(status)
            return out
        finally:
            for pages in held:
                self._give(pages)
