"""The paged-cache operators as workloads: what is measured, their plain forms and their 64-bit values.

Three operators over one cache of pages ``[pages, kv_heads, page_size, head_dim]``:

* ``append``: per-head RMSNorm and rotary embedding of the new tokens' queries and keys, keys and values
  written to the rows of their sequences' pages;
* ``decode``: one query token per sequence over its own pages, and before them the pages of a prefix that
  the sequences of a group share;
* ``extend``: the new tokens of each sequence (a prompt, or a piece of one) over the shared prefix and
  the sequence's own rows, causally.

``run`` computes them in elementary torch operations (32 bits, rounded once at the end) while ``own`` is
false, and through the package's public entry points while it is true.
"""
import importlib
import math
import random

import torch

own = False

EPS = 1e-6
THETA = 1e6


# --------------------------------------------------------------------------- cases
def _case(name, op, **kw):
    c = dict(op=op, dtype="bf16", heads=32, kv_heads=8, head_dim=128, page=16, seqs=1, new=1, kv_lo=1, kv_hi=1,
             groups=0, prefix=0, spread=1)
    c.update(kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the append of one decode step, one sequence in flight: a call that is all latency
        _case("append, 1 token", "append", kv_lo=4003, kv_hi=4003),
        # fp32 activations, small heads, a ragged batch of prompt pieces with an odd token count
        _case("append, f32 ragged 777", "append", dtype="f32", heads=16, head_dim=64, page=64, seqs=9, new=777,
              kv_lo=40, kv_hi=900),
        # whole prompts arriving together behind a shared prefix
        _case("append, prompts 16384", "append", heads=32, seqs=24, new=16384, kv_lo=100, kv_hi=1500, groups=1,
              prefix=512),
        # one user talking to a model with 16 query heads: latency of a decode step
        _case("decode, 1 x 1000", "decode", heads=16, kv_lo=1000, kv_hi=1000),
        # an ordinary serving batch, lengths from nothing to 8192, no shared prefix: bandwidth
        _case("decode, 64 ragged 8192", "decode", seqs=64, kv_lo=0, kv_hi=8192),
        # fp32 cache, 3 query heads to a kv head, two prefixes, some sequences with no row of their own
        _case("decode, f32 two prefixes", "decode", dtype="f32", heads=12, kv_heads=4, head_dim=64, page=32, seqs=21,
              kv_lo=0, kv_hi=700, groups=2, prefix=1500),
        # a system prompt shared by a middling batch
        _case("decode, 32 on 8192", "decode", seqs=32, kv_lo=1, kv_hi=512, groups=1, prefix=8192, page=64),
        # many samples of one long document: the prefix dominates the arithmetic, the own rows the bytes
        _case("decode, 256 on 32768", "decode", seqs=256, kv_lo=64, kv_hi=1024, groups=1, prefix=32768),
        # a few drafted tokens checked against a long conversation
        _case("extend, 6 after 20000", "extend", heads=32, new=6, kv_lo=20006, kv_hi=20006),
        # users' questions behind a shared prefix, odd lengths
        _case("extend, ragged on 1031", "extend", heads=16, seqs=11, new=3333, kv_lo=50, kv_hi=700, groups=1,
              prefix=1031, page=32),
        # fp32, 64-wide heads
        _case("extend, f32 500", "extend", dtype="f32", heads=8, kv_heads=2, head_dim=64, seqs=2, new=500, kv_lo=100,
              kv_hi=500, page=128),
        # one long prompt from its first token
        _case("extend, prompt 8192", "extend", new=8192, kv_lo=8192, kv_hi=8192, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "extend"])
    kv_heads = rng.choice([1, 2, 4, 8])
    g = rng.choice([1, 2, 3, 4, 5, 7, 8])
    f32 = rng.random() < 0.25
    d = rng.choice([64, 128, 128])
    groups = rng.choice([0, 0, 1, 2, 3])
    c = dict(dtype="f32" if f32 else "bf16", heads=g * kv_heads, kv_heads=kv_heads, head_dim=d,
             page=rng.choice([16, 32, 64, 128, 256]), spread=rng.randrange(1, 1 << 20))
    if op == "append":
        new = _log(rng, 1, 12000)
        seqs = min(new, _log(rng, 1, 64))
        c.update(seqs=seqs, new=new, kv_lo=1, kv_hi=max(2, 3 * new // seqs), groups=min(groups, seqs),
                 prefix=_log(rng, 1, 4000))
    elif op == "decode":
        seqs = _log(rng, 1, 200)
        top = max(2, min(16000, 200000 // seqs))
        groups = min(groups, seqs)
        c.update(seqs=seqs, new=seqs, kv_lo=rng.choice([0, 1]), kv_hi=_log(rng, 2, top), groups=groups,
                 prefix=_log(rng, 1, 16000))
    else:
        seqs = _log(rng, 1, 12)
        new = max(seqs, _log(rng, 2, 2000 if f32 else 5000))
        c.update(seqs=seqs, new=new, kv_lo=1, kv_hi=_log(rng, max(2, new // seqs), 2 * new + 4000 // seqs),
                 groups=min(groups, seqs), prefix=_log(rng, 1, 4000))
        # the scores of the padded plain form stay below those of the largest listed case
        while c["heads"] * c["seqs"] * c["new"] * (c["kv_hi"] + c["new"] + c["prefix"]) > 2 * 32 * 8192 * 8192:
            c.update(new=max(c["seqs"], c["new"] * 3 // 4), kv_hi=max(2, c["kv_hi"] * 3 // 4),
                     prefix=max(1, c["prefix"] * 3 // 4))
    return _case(None, op, **c)


def _shape(case):
    """Lengths of a case, made from its values alone: (new tokens, own rows after them) of each sequence, the
    sequences of each group and the prefixes' lengths."""
    rng = random.Random(case["spread"] * 7919 + case["seqs"])
    n, op = case["seqs"], case["op"]
    lo, hi = case["kv_lo"], case["kv_hi"]
    kv = [lo + int((hi - lo) * rng.random() ** 1.5) for _ in range(n)]
    kv[0] = hi
    if n > 2:
        kv[-1] = lo
    if op == "decode":
        new = [1] * n
    else:
        cut = sorted(rng.randrange(case["new"] + 1) for _ in range(n - 1))
        new = [b - a for a, b in zip([0] + cut, cut + [case["new"]])]
        kv = [max(a, b) for a, b in zip(kv, new)]
    p = case["groups"]
    starts, plens = [], []
    if p:
        cut = sorted(rng.sample(range(1, n), p - 1)) if p > 1 else []
        starts = [0] + cut + [n]
        plens = [case["prefix"]] + [max(1, int(case["prefix"] * rng.uniform(0.3, 1.0))) for _ in range(p - 1)]
    return new, kv, starts, plens


# --------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    new, kv, starts, plens = _shape(case)
    gen = torch.Generator(dev).manual_seed(seed)
    dt = torch.bfloat16 if case["dtype"] == "bf16" else torch.float32
    hq, hkv, d, ps, n = case["heads"], case["kv_heads"], case["head_dim"], case["page"], case["seqs"]
    width = max(1, -(-max(kv) // ps))
    pwidth = max([1] + [-(-p // ps) for p in plens])
    own_pages, pre_pages = [-(-k // ps) for k in kv], [-(-p // ps) for p in plens]
    pages = sum(own_pages) + sum(pre_pages) + 3
    perm = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)

    def table(counts, wide, first):
        """Rows of distinct pages, unused entries 0."""
        c = torch.tensor(counts, device=dev)
        base = first + c.cumsum(0) - c
        j = torch.arange(wide, device=dev)[None]
        return torch.where(j < c[:, None], perm[(base[:, None] + j).clamp(max=pages - 1)], 0).to(torch.int32)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32).to(dt)

    s = {"case": case, "op": case["op"], "scale": d ** -0.5, "dtype": dt,
         "k_pages": normal(pages, hkv, ps, d), "v_pages": normal(pages, hkv, ps, d),
         "page_table": table(own_pages, width, 0),
         "kv_lens": torch.tensor(kv, dtype=torch.int32, device=dev),
         "cu_tokens": None, "group_starts": None, "prefix_lens": None, "prefix_table": None,
         "max_kv": max(kv), "max_prefix": max([0] + plens), "max_new": max(new),
         "max_group": max([b - a for a, b in zip(starts, starts[1:])] + [0])}
    total = sum(new)
    if case["op"] != "decode":
        s["cu_tokens"] = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=dev)
    if plens:
        s["group_starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
        s["prefix_lens"] = torch.tensor(plens, dtype=torch.int32, device=dev)
        s["prefix_table"] = table(pre_pages, pwidth, sum(own_pages))
    if case["op"] == "append":
        # the projections of the new tokens as one matrix product leaves them: q, k and v side by side
        qkv = normal(total, hq + 2 * hkv, d)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        s["q_weight"] = torch.rand(d, generator=gen, device=dev) + 0.5
        s["k_weight"] = torch.rand(d, generator=gen, device=dev) + 0.5
        length = s["max_kv"] + s["max_prefix"]
        inv = THETA ** (-torch.arange(0, d, 2, device=dev, dtype=torch.float64) / d)
        f = torch.outer(torch.arange(length, device=dev, dtype=torch.float64), inv).repeat(1, 2)
        s["cos"], s["sin"] = f.cos().float(), f.sin().float()
    else:
        s["q"] = normal(total, hq, d)
    if own:
        # what a serving program keeps from step to step: the cache and the batch that describes its tensors
        cbq = importlib.import_module("codebook-quantization_b200")
        s["cache"] = cbq.PagedKVCache(s["k_pages"], s["v_pages"])
        s["batch"] = cbq.PagedBatch(s["page_table"], s["kv_lens"], cu_tokens=s["cu_tokens"],
                                    group_starts=s["group_starts"], prefix_lens=s["prefix_lens"],
                                    prefix_table=s["prefix_table"], max_kv_len=s["max_kv"],
                                    max_prefix_len=s["max_prefix"])
    return s


def run(state):
    if own:
        c, b = state["cache"], state["batch"]
        if state["op"] == "append":
            q = c.append_rope(b, state["q"], state["k"], state["v"], state["cos"], state["sin"], eps=EPS,
                              q_weight=state["q_weight"], k_weight=state["k_weight"])
            return {"q": q, "k_pages": state["k_pages"], "v_pages": state["v_pages"]}
        if state["op"] == "decode":
            return {"out": c.attend_decode(b, state["q"], scale=state["scale"])}
        return {"out": c.attend_extend(b, state["q"], scale=state["scale"])}
    if state["op"] == "append":
        return _plain_append(state)
    return _plain_decode(state) if state["op"] == "decode" else _plain_extend(state)


# --------------------------------------------------------------------------- plain forms
def _tokens(s):
    """Sequence and own row of every new token."""
    cu, total = s["cu_tokens"], s["q"].shape[0]
    t = torch.arange(total, device=cu.device, dtype=torch.int32)
    seq = torch.searchsorted(cu, t, right=True) - 1
    return seq, (s["kv_lens"][seq] - cu[seq + 1] + t).long()


def _prefix_of(s):
    """Prefix length of every sequence, and its group."""
    n = s["kv_lens"].shape[0]
    if s["group_starts"] is None:
        return None, None
    i = torch.arange(n, device=s["kv_lens"].device, dtype=torch.int32)
    g = torch.searchsorted(s["group_starts"], i, right=True) - 1
    return g, s["prefix_lens"][g].long()


def _rows(s, page_table, index):
    """Keys and values (32 bits) at own rows ``index`` [n, l] of tables [n, w]: [n, l, kv_heads, head_dim]."""
    ps = s["k_pages"].shape[2]
    page = page_table.long().gather(1, (index // ps).clamp(max=page_table.shape[1] - 1))
    line = index % ps
    return s["k_pages"][page, :, line].float(), s["v_pages"][page, :, line].float()


def _plain_append(s):
    seq, row = _tokens(s)
    pos = row if s["group_starts"] is None else row + _prefix_of(s)[1][seq]
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]

    def rotate(x, w):
        x = x.float()
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w
        a, b = x.chunk(2, -1)
        return x * cos + torch.cat((-b, a), -1) * sin

    ps = s["k_pages"].shape[2]
    page, line = s["page_table"].long()[seq, row // ps], row % ps
    s["k_pages"][page, :, line] = rotate(s["k"], s["k_weight"]).to(s["dtype"])
    s["v_pages"][page, :, line] = s["v"]
    return {"q": rotate(s["q"], s["q_weight"]).to(s["dtype"]), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _plain_decode(s):
    n, hq, d = s["q"].shape
    hkv = s["k_pages"].shape[1]
    q = s["q"].float().view(n, hkv, hq // hkv, d) * s["scale"]
    j = torch.arange(max(1, s["max_kv"]), device=q.device)
    k, v = _rows(s, s["page_table"], j[None].expand(n, -1))
    x = torch.einsum("bhgd,blhd->bhgl", q, k)
    x = x.masked_fill(~(j[None] < s["kv_lens"][:, None])[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    group, plen = _prefix_of(s)
    if group is not None:
        p, lp = s["prefix_table"].shape[0], max(1, s["max_prefix"])
        slot = torch.arange(n, device=q.device) - s["group_starts"].long()[group]
        qg = q.new_zeros(p, s["max_group"], hkv, hq // hkv, d)
        qg[group, slot] = q
        jp = torch.arange(lp, device=q.device)
        kp, vp = _rows(s, s["prefix_table"], jp[None].expand(p, -1))
        y = torch.einsum("pbhgd,plhd->pbhgl", qg, kp)
        y = y.masked_fill(~(jp[None] < s["prefix_lens"][:, None])[:, None, None, None], -math.inf)
        m = torch.maximum(m, y.amax(-1, keepdim=True)[group, slot])
    m = m.masked_fill(m == -math.inf, 0.0)
    e = torch.exp(x - m)
    total, acc = e.sum(-1, keepdim=True), torch.einsum("bhgl,blhd->bhgd", e, v)
    if group is not None:
        mg = q.new_zeros(p, s["max_group"], hkv, hq // hkv, 1)
        mg[group, slot] = m
        e = torch.exp(y - mg)
        total = total + e.sum(-1, keepdim=True)[group, slot]
        acc = acc + torch.einsum("pbhgl,plhd->pbhgd", e, vp)[group, slot]
    out = acc / total.masked_fill(total == 0, 1.0)
    return {"out": out.view(n, hq, d).to(s["dtype"])}


def _plain_extend(s):
    total, hq, d = s["q"].shape
    n, hkv = s["kv_lens"].shape[0], s["k_pages"].shape[1]
    seq, row = _tokens(s)
    at = torch.arange(total, device=seq.device) - s["cu_tokens"].long()[seq]
    q = s["q"].new_zeros(n, s["max_new"], hq, d, dtype=torch.float32)
    q[seq, at] = s["q"].float() * s["scale"]
    last = torch.full((n, s["max_new"]), -1, device=q.device)
    last[seq, at] = row
    j = torch.arange(s["max_kv"], device=q.device)
    k, v = _rows(s, s["page_table"], j[None].expand(n, -1))
    seen = j[None, None] <= last[..., None]
    group, plen = _prefix_of(s)
    if group is not None:
        jp = torch.arange(max(1, s["max_prefix"]), device=q.device)
        kp, vp = _rows(s, s["prefix_table"], jp[None].expand(s["prefix_table"].shape[0], -1))
        k, v = torch.cat((kp[group], k), 1), torch.cat((vp[group], v), 1)
        seen = torch.cat(((jp[None] < plen[:, None])[:, None].expand(-1, s["max_new"], -1), seen), -1)
    q = q.view(n, s["max_new"], hkv, hq // hkv, d)
    x = torch.einsum("bthgd,blhd->bhgtl", q, k)
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    m = x.amax(-1, keepdim=True)
    e = x.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = e.sum(-1, keepdim=True)
    e = e.div_(total.masked_fill(total == 0, 1.0))
    out = torch.einsum("bhgtl,blhd->bthgd", e, v).reshape(n, s["max_new"], hq, d)
    return {"out": out[seq, at].to(s["dtype"])}


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """Each sequence by itself, from the definition, in 64 bits."""
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    new, kv, starts, plens = _shape(case)
    hq, hkv, d, ps = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    group = [next(g for g in range(len(plens)) if starts[g] <= i < starts[g + 1]) if plens else -1
             for i in range(len(kv))]
    dev = s["q"].device
    q = s["q"].double()
    if case["op"] == "append":
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        half = d // 2
        out = torch.empty_like(q)

        def turn(x, w, c, t):
            x = x.double()
            x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / d + EPS) * w.double()
            lo, hi = x[..., :half], x[..., half:]
            return torch.cat((lo * c[..., :half] - hi * t[..., :half], hi * c[..., half:] + lo * t[..., half:]), -1)

        first = 0
        for i, (t, n) in enumerate(zip(new, kv)):
            if t:
                rows = torch.arange(n - t, n, device=dev)
                pos = rows + (plens[group[i]] if plens else 0)
                c, z = s["cos"][pos].double()[:, None], s["sin"][pos].double()[:, None]
                part = slice(first, first + t)
                out[part] = turn(s["q"][part], s["q_weight"], c, z)
                page = s["page_table"][i].long()[rows // ps]
                kp[page, :, rows % ps] = turn(s["k"][part], s["k_weight"], c, z)
                vp[page, :, rows % ps] = s["v"][part].double()
            first += t
        return {"q": out, "k_pages": kp, "v_pages": vp}

    def rows_of(table, n):
        pages = table[: -(-n // ps)].long() if n else table[:0].long()
        take = lambda pool: pool[pages].transpose(1, 2).reshape(-1, hkv, d)[:n].double()  # noqa: E731
        return take(s["k_pages"]), take(s["v_pages"])

    shared = [rows_of(s["prefix_table"][g], p) for g, p in enumerate(plens)]
    out = torch.zeros_like(q)
    first = 0
    for i, (t, n) in enumerate(zip(new, kv)):
        k, v = rows_of(s["page_table"][i], n)
        if plens:
            k, v = torch.cat((shared[group[i]][0], k)), torch.cat((shared[group[i]][1], v))
        if t and k.shape[0]:
            sees = k.shape[0] - t + torch.arange(t, device=dev) if case["op"] == "extend" else \
                torch.full((t,), k.shape[0] - 1, device=dev)
            hide = torch.arange(k.shape[0], device=dev)[None] > sees[:, None]
            for h in range(hkv):
                part = q[first:first + t, h * (hq // hkv):(h + 1) * (hq // hkv)]
                x = torch.matmul(part.transpose(0, 1), k[:, h].T) / math.sqrt(d)
                p = torch.softmax(x.masked_fill_(hide[None], -math.inf), -1)
                out[first:first + t, h * (hq // hkv):(h + 1) * (hq // hkv)] = torch.matmul(p, v[:, h]).transpose(0, 1)
                del x, p
        first += t
    return {"out": out}


# --------------------------------------------------------------------------- least work
def work(case):
    new, kv, starts, plens = _shape(case)
    e = 2 if case["dtype"] == "bf16" else 4
    hq, hkv, d = case["heads"], case["kv_heads"], case["head_dim"]
    total = sum(new)
    if case["op"] == "append":
        # q, k, v read and written once, a row of each table for every token
        return {"bytes": 2 * total * (hq + 2 * hkv) * d * e + total * 2 * d * 4, "flops": 10 * total * (hq + hkv) * d}
    before = [0] * len(kv)
    for g, p in enumerate(plens):
        before[starts[g]:starts[g + 1]] = [p] * (starts[g + 1] - starts[g])
    # a decode row sees all its keys, the i-th new token of an extension all but the later ones
    seen = sum(t * (p + n) - (t * (t - 1) // 2 if case["op"] == "extend" else 0)
               for t, n, p in zip(new, kv, before))
    rows = sum(n for t, n in zip(new, kv) if t) + sum(plens)
    return {"bytes": 2 * rows * hkv * d * e + 2 * total * hq * d * e, "flops": 4 * seen * hq * d}
