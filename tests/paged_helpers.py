"""Inputs and 64-bit oracle of the paged-cache tests (no test functions here).

Everything is made on the CPU in float64 from a seed and rounded to the cache's
dtype; the oracle works on those rounded values sequence by sequence from the
definitions.
"""
import torch


class Setup:
    """A ragged batch over a shuffled page pool.

    ``kv``: own rows per sequence (new tokens included), ``new``: new tokens per
    sequence (None: one each), ``groups``: list of (sequences, prefix length).
    Rows no sequence owns hold ``stale`` (NaN by default)."""

    def __init__(self, kv, new=None, groups=(), heads=4, kv_heads=2, d=64, page=16, dtype=torch.bfloat16, seed=0,
                 layout="hnd", stale=float("nan"), spare=3, slack=0):
        g = torch.Generator().manual_seed(seed)
        self.kv, self.new = list(kv), ([1] * len(kv) if new is None else list(new))
        self.groups, self.heads, self.kv_heads, self.d, self.page, self.dtype = groups, heads, kv_heads, d, page, dtype
        self.n, self.tokens = len(self.kv), sum(self.new)
        self.G = heads // kv_heads
        own = [-(-k // page) for k in self.kv]
        pre = [-(-p // page) for _, p in groups]
        self.pages = sum(own) + sum(pre) + spare
        perm = torch.randperm(self.pages, generator=g).tolist()
        width, pwidth = max(own + [1]) + slack, max(pre + [1]) + slack
        # unused table entries name no page at all
        self.table = torch.full((self.n, width), -1, dtype=torch.int32)
        self.ptable = torch.full((max(len(pre), 1), pwidth), 1 << 30, dtype=torch.int32)
        at = 0
        for i, c in enumerate(own):
            self.table[i, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
            at += c
        for i, c in enumerate(pre):
            self.ptable[i, :c] = torch.tensor(perm[at:at + c], dtype=torch.int32)
            at += c
        self.plens = [p for _, p in groups]
        self.starts = [0]
        for c, _ in groups:
            self.starts.append(self.starts[-1] + c)
        self.group_of = [next((j for j in range(len(groups)) if self.starts[j] <= i < self.starts[j + 1]), -1)
                         for i in range(self.n)]
        rnd = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64).to(dtype)  # noqa: E731
        self.k = torch.full((self.pages, kv_heads, page, d), stale, dtype=dtype)
        self.v = self.k.clone()
        for tab, lens in ((self.table, self.kv), (self.ptable, self.plens)):
            for i, n in enumerate(lens):
                for j in range(-(-n // page)):
                    m = min(page, n - j * page)
                    self.k[tab[i, j], :, :m] = rnd(kv_heads, m, d)
                    self.v[tab[i, j], :, :m] = rnd(kv_heads, m, d)
        self.q = rnd(self.tokens, heads, d)
        self.layout = layout

    def pools(self, dev):
        """The pools on the device: contiguous, rows before heads, or k and v as halves of one pool."""
        if self.layout == "nhd":
            return tuple(x.transpose(1, 2).contiguous().to(dev).transpose(1, 2) for x in (self.k, self.v))
        if self.layout == "joint":
            both = torch.stack((self.k, self.v), 1).to(dev)
            return both[:, 0], both[:, 1]
        return self.k.to(dev), self.v.to(dev)

    def batch(self, cbq, dev, decode=False, **kw):
        i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
        cu = None if decode else i32([0] + torch.tensor(self.new).cumsum(0).tolist())
        shared = dict(group_starts=i32(self.starts), prefix_lens=i32(self.plens),
                      prefix_table=self.ptable.to(dev)) if self.groups else {}
        return cbq.PagedBatch(self.table.to(dev), i32(self.kv), cu_tokens=cu, **shared, **kw)

    def rows(self, i, pool):
        """Prefix rows then own rows of sequence i: [n, kv_heads, d] float64."""
        out = []
        g = self.group_of[i]
        for tab, r, n in ([(self.ptable, g, self.plens[g])] if g >= 0 else []) + [(self.table, i, self.kv[i])]:
            for j in range(-(-n // self.page)):
                out.append(pool[tab[r, j], :, :min(self.page, n - j * self.page)].transpose(0, 1).double())
        return torch.cat(out) if out else torch.zeros(0, self.kv_heads, self.d, dtype=torch.float64)

    def attention(self, scale, causal):
        """(out, spread, slack): the result, sum_j p_j |v_j|, and a bound of
        the relative error that fp32 scores cause in a row's weights."""
        q = self.q.double()
        out, spread = torch.zeros_like(q), torch.zeros_like(q)
        slack = torch.zeros(self.tokens, self.heads, 1, dtype=torch.float64)
        t = 0
        for i in range(self.n):
            k, v = self.rows(i, self.k), self.rows(i, self.v)
            for a in range(self.new[i]):
                n = k.shape[0] - (self.new[i] - 1 - a if causal else 0)
                n = max(n, k.shape[0] - self.kv[i])            # own rows that are not there hide nothing of the prefix
                if n:
                    kk = k[:n].repeat_interleave(self.G, 1)    # [n, heads, d]
                    vv = v[:n].repeat_interleave(self.G, 1)
                    x = torch.einsum("hd,nhd->hn", q[t], kk) * scale
                    p = torch.softmax(x, -1)
                    out[t] = torch.einsum("hn,nhd->hd", p, vv)
                    spread[t] = torch.einsum("hn,nhd->hd", p, vv.abs())
                    mag = torch.einsum("hd,nhd->hn", q[t].abs(), kk.abs()).amax(-1) * abs(scale)
                    slack[t, :, 0] = 2 * (self.d + 4) * 2.0 ** -24 * mag + n * 2.0 ** -23
                t += 1
        return out, spread, slack


def check_attention(got, ref, spread, slack):
    """Element by element: the output's rounding, the rounding of the softmax
    weights to bf16 (bf16 only; at most 2^-8 of each weight, in numerator and
    sum at most once) and fp32 arithmetic; and the relative L2 distance that
    independent roundings of that size give (bf16: 2^-8, fp32: 1e-5)."""
    bf = got.dtype == torch.bfloat16
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    u = 2.0 ** -8 if bf else 2.0 ** -23
    tol = u * ref.abs() + ((2.0 ** -8 if bf else 0.0) + slack) * spread + 1e-30
    bad = (got - ref).abs() > tol
    assert not bad.any(), (int(bad.sum()), float(((got - ref).abs() / tol).max()))
    rel = float((got - ref).norm() / ref.norm().clamp(min=1e-30))
    assert rel <= (2.0 ** -8 if bf else 1e-5), rel
