"""Operators of speculative decoding on the exact integer engine, and their plain forms.

A serving step drafts a tree of tokens, runs all of its nodes through the model at once, keeps the
path that the target model itself would have produced, and tidies the cache:

  tree_attention   attention of the tree's rows over a paged K/V cache (K int16 with a shift per
                   row, V int32): the cached positions of the sequence, then the row's own
                   ancestors in the tree, by a bit mask
  tree_verify      the target's token of every row from given random numbers (or its argmax), and
                   the path of drafted tokens that agree with it
  kv_compact       the cache rows of the accepted path moved next to the sequence's older rows, in
                   every layer
  kv_copy_pages    pages copied to other pages, whole or their first rows: a forked sequence's last
                   page, a page that two sequences shared

All arithmetic is integer arithmetic of the exact program, so both forms give the same bits:
  score   s = shr((q . k) * INV, 32 - qs - ks),  INV = round(2^16 / sqrt(hd))
  e       table exp at (max s - s) with linear interpolation, Q24; 0 from 40.0 on
  p       (e << 20) // sum(e)
  output  shr(sum(p * v), 20)
  shr     round half up: (a + (1 << (n - 1))) >> n for n > 0, a << -n otherwise
The plain form keeps whole numbers in 64 bits (scores reach 2^50) and multiplies matrices in 64-bit
floats where every partial sum stays below 2^53, which is exact.
"""
import math

import numpy as np
import torch

own = False

ONE = 1 << 16
EXP_LEN = 256 * 40 + 2


# ------------------------------------------------------------------------------------------ cases
def _attn(name, H, KV, hd, B, ctx, nodes, page):
    return dict(name=name, op="tree_attention", H=H, KV=KV, hd=hd, B=B, ctx=ctx, nodes=nodes, page=page)


def _verify(name, V, B, nodes, greedy):
    return dict(name=name, op="tree_verify", V=V, B=B, nodes=nodes, greedy=greedy)


def _compact(name, L, KV, hd, B, ctx, nodes, acc, page):
    return dict(name=name, op="kv_compact", L=L, KV=KV, hd=hd, B=B, ctx=ctx, nodes=nodes, acc=acc, page=page)


def _copy(name, L, KV, hd, n, page, rows):
    return dict(name=name, op="kv_copy_pages", L=L, KV=KV, hd=hd, n=n, page=page, rows=rows)


def listed():
    return [
        # the first token of an empty sequence, the 0.5B model's heads: nothing but latency
        _attn("attention: first token, 14 heads of 64", 14, 2, 64, 1, 0, 1, 64),
        # plain decoding of a batch: one token of each of 32 sequences (7B heads)
        _attn("attention: 32 sequences, one token each", 28, 4, 128, 32, 1000, 1, 64),
        # one user's tree behind a 512-token prompt; the cache is one slot of consecutive positions
        _attn("attention: one tree of 26 after 513 tokens", 28, 4, 128, 1, 513, 26, 1024),
        # a serving batch: ragged trees over ragged contexts
        _attn("attention: 8 trees of up to 63, 4097 tokens", 28, 4, 128, 8, 4097, 63, 128),
        # a long document and a wide tree (14B heads)
        _attn("attention: one tree of 61 after 32768 tokens", 40, 8, 128, 1, 32768, 61, 256),
        # greedy decoding without a draft: one row
        _verify("verify: one greedy row", 151936, 1, 1, True),
        # one user's tree, sampled
        _verify("verify: one tree of 26", 152064, 1, 26, False),
        # a serving batch of ragged trees, sampled
        _verify("verify: 8 trees of up to 63", 152064, 8, 63, False),
        # the accepted path of one small tree, 0.5B cache
        _compact("compact: one path, 24 layers", 24, 2, 64, 1, 100, 8, 4, 64),
        # the accepted paths of a serving batch, 7B cache
        _compact("compact: 8 paths, 28 layers", 28, 4, 128, 8, 1000, 63, 9, 64),
        # a forked sequence's half-filled last page, 0.5B cache
        _copy("copy: half a page, 24 layers", 24, 2, 64, 1, 64, 33),
        # a batch of pages, 7B cache
        _copy("copy: 96 pages, 28 layers", 28, 4, 128, 96, 64, 64),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["tree_attention", "tree_attention", "tree_verify", "kv_compact", "kv_copy_pages"])
    # heads and head widths of the configurations: 0.5B, 7B, 14B, the mixture model, and its tests' 16 and 32
    H, KV, hd = rng.choice([(14, 2, 64), (28, 4, 128), (40, 8, 128), (16, 16, 128), (4, 2, 16), (6, 2, 32)])
    page = rng.choice([16, 32, 48, 64, 100, 128, 256])
    if op == "tree_attention":
        ctx, nodes, B = _log_int(rng, 1, 32768) - 1, _log_int(rng, 1, 64), _log_int(rng, 1, 32)
        while B * (ctx + nodes) * nodes * H > 61 * 40 * 32768 or B * (ctx + nodes) * KV * hd > 32 * 32768 * 128:
            B, ctx = max(1, B // 2), (ctx if B > 1 else ctx // 2)
        return dict(op=op, H=H, KV=KV, hd=hd, B=B, ctx=ctx, nodes=nodes, page=page)
    if op == "tree_verify":
        V, nodes, B = _log_int(rng, 500, 152064), _log_int(rng, 1, 64), _log_int(rng, 1, 8)
        return dict(op=op, V=V, B=B, nodes=nodes, greedy=rng.random() < 0.3)
    L = _log_int(rng, 1, 28)
    if op == "kv_compact":
        nodes = _log_int(rng, 2, 63)
        return dict(op=op, L=L, KV=KV, hd=hd, B=_log_int(rng, 1, 8), ctx=_log_int(rng, 1, 1001) - 1, nodes=nodes,
                    acc=_log_int(rng, 2, max(2, nodes // 3)), page=page)
    rows = rng.randint(1, page)
    return dict(op=op, L=L, KV=KV, hd=hd, n=_log_int(rng, 1, max(1, 96 * 64 // page // max(1, KV // 4))), page=page,
                rows=rows)


def _lens(case):
    """Context length and node count of every sequence: ragged, but settled by the case alone."""
    B, ctx, nodes = case["B"], case["ctx"], case["nodes"]
    return ([ctx - (b * 389) % (ctx // 2 + 1) for b in range(B)], [nodes - (b * 11) % (nodes // 2 + 1) for b in range(B)])


def _accepted(case):
    """Rows of every sequence's accepted path (the root among them)."""
    _, nodes = _lens(case)
    return [min(n, max(1, case["acc"] - (3 * b) % case["acc"])) for b, n in enumerate(nodes)]


# ------------------------------------------------------------------------------------------ inputs
def _exp_table():
    return [round(math.exp(-i / 256) * (1 << 24)) for i in range(EXP_LEN)]


def _quant(x):
    """Rows of Q16 whole numbers as int16 with a shift per row, as the engine stores them."""
    m = x.abs().amax(-1, keepdim=True)
    s = (torch.floor(torch.log2(m.clamp(min=1).double())).long() + 1 - 15).clamp(min=0)
    half = torch.where(s > 0, torch.ones_like(s) << (s - 1).clamp(min=0), torch.zeros_like(s))
    return ((x + half) >> s).clamp(-32767, 32767).to(torch.int16), s.squeeze(-1)


def _pages(need, page, g):
    """A page table for sequences of `need` positions each: page ids in a random order, and the pool's size."""
    counts = [-(-n // page) for n in need]
    pool = sum(counts) + 2                                    # two pages that nobody holds
    ids = torch.randperm(pool, generator=g)[:sum(counts)].tolist()
    table = torch.full((len(need), max(max(counts), 1)), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = torch.tensor(ids[at:at + c], dtype=torch.int32)
        at += c
    return table, pool


def _fill(case, layers, pool, g):
    """A cache whose every row, stale ones among them, holds values of the size that a model leaves there."""
    shape = (layers, pool, case["KV"], case["page"])
    hd, dev = case["hd"], "cuda"
    k = torch.empty(*shape, hd, dtype=torch.int16, device=dev)
    ks = torch.empty(*shape, dtype=torch.int8, device=dev)
    v = torch.empty(*shape, hd, dtype=torch.int32, device=dev)
    for i in range(layers):
        x = torch.randn(*shape[1:], hd, generator=g, device=dev) * (1.5 * ONE)
        x[..., :2] *= 6.0                                     # a few channels are far larger than the others
        kq, s = _quant(x.long())
        k[i], ks[i] = kq, s.to(torch.int8)
        v[i] = (torch.randn(*shape[1:], hd, generator=g, device=dev) * (0.8 * ONE)).int()
    return k, ks, v


def _trees(nodes, cg):
    """Parents (node 0 is the root, -1) of trees that widen towards the root, as drafts do."""
    out = []
    for n in nodes:
        r = torch.rand(max(n, 1), generator=cg).tolist()
        out.append([-1] + [max(0, i - 1 - int(r[i] * min(i, 6))) for i in range(1, n)])
    return out


def prepare(case, seed):
    cg = torch.Generator().manual_seed((seed * 2 + 1) % (1 << 62))
    g = torch.Generator(device="cuda").manual_seed((seed * 2 + 2) % (1 << 62))
    st = dict(case)
    if own:
        import exact_llm_b200.ops  # noqa: F401  (registers torch.ops.exact.*)
    st["exp_t"] = torch.tensor(_exp_table(), dtype=torch.int32).cuda()
    if case["op"] == "kv_copy_pages":
        n, page = case["n"], case["page"]
        pool = 2 * n + 2
        st["k"], st["ks"], st["v"] = _fill(case, case["L"], pool, g)
        ids = torch.randperm(pool, generator=cg)
        st["src"], st["dst"] = ids[:n].int().cuda(), ids[n:2 * n].int().cuda()
        rows = [max(1, case["rows"] - (7 * i) % case["rows"]) if case["rows"] < page else page for i in range(n)]
        st["rows"] = torch.tensor(rows, dtype=torch.int32).cuda()
        return st
    ctx, nodes = _lens(case) if "ctx" in case else (None, _lens(dict(case, ctx=0))[1])
    starts = [0]
    for n in nodes:
        starts.append(starts[-1] + n)
    R = starts[-1]
    parents = _trees(nodes, cg)
    st["row_start"] = torch.tensor(starts, dtype=torch.int32).cuda()
    if case["op"] == "tree_verify":
        V = case["V"]
        lg = torch.empty(R, V, dtype=torch.int64, device="cuda")
        best = torch.randint(0, V, (R,), generator=g, device="cuda")
        for r in range(R):                                    # a bell of logits and one likely token a row
            lg[r] = (torch.randn(V, generator=g, device="cuda") * (2.5 * ONE)).long()
            lg[r, best[r]] += int((math.log(V) + 5.0) * ONE)
        st["logits"] = lg
        par = torch.tensor([p for t in parents for p in t], dtype=torch.int32)
        gpar = torch.tensor([starts[b] + max(p, 0) for b, t in enumerate(parents) for p in t])
        drafted = torch.rand(R, generator=cg) < 0.75          # the draft often names the target's likely token
        toks = torch.where(drafted.cuda(), best[gpar.cuda()], torch.randint(0, V, (R,), generator=g, device="cuda"))
        st["tokens"], st["parent"] = toks.int(), par.cuda()
        depth = []
        for t in parents:
            d = []
            for p in t:
                d.append(0 if p < 0 else d[p] + 1)
            depth += d
        u = torch.randint(0, 1 << 20, (case["B"], max(nodes)), generator=cg)       # one number per output position
        seq = [b for b, t in enumerate(parents) for _ in t]
        u20 = u[torch.tensor(seq), torch.tensor(depth)].int()
        st["u20"] = (torch.full_like(u20, -1) if case["greedy"] else u20).cuda()
        st["tnum"] = round(ONE / 0.8)
        st["max_len"] = max(nodes)                            # no path is longer
        return st
    st["ctx_len"] = torch.tensor(ctx, dtype=torch.int32).cuda()
    table, pool = _pages([c + n for c, n in zip(ctx, nodes)], case["page"], cg)
    st["table"] = table.cuda()
    if case["op"] == "kv_compact":
        st["k"], st["ks"], st["v"] = _fill(case, case["L"], pool, g)
        acc = _accepted(case)
        width = max(acc)
        path = torch.full((case["B"], width), -1, dtype=torch.int32)
        for b, (a, n) in enumerate(zip(acc, nodes)):          # a row stays, or comes from behind the kept rows
            far = (torch.randperm(n - a, generator=cg)[:a - 1] + a).sort().values.tolist() if n > a else []
            path[b, :a] = torch.tensor([*range(a - len(far)), *far], dtype=torch.int32)
        st["path"], st["n_acc"] = path.cuda(), torch.tensor(acc, dtype=torch.int32).cuda()
        return st
    k, ks, v = _fill(case, 1, pool, g)
    st["k"], st["ks"], st["v"] = k[0], ks[0], v[0]
    q, s = _quant((torch.randn(R, case["H"], case["hd"], generator=g, device="cuda") * (2.0 * ONE)).long())
    st["q"], st["qs"] = q, s.int()
    words = -(-max(nodes) // 64)
    mask = []
    for t in parents:                                         # a node sees itself and its ancestors
        m = []
        for i, p in enumerate(t):
            m.append((m[p] if p >= 0 else 0) | (1 << i))
        mask += m
    flat = [[(x >> (64 * w)) & (2**64 - 1) for w in range(words)] for x in mask]
    st["mask"] = torch.from_numpy(np.array(flat, dtype=np.uint64).view(np.int64)).cuda()
    st["nodes_of"], st["ctx_of"] = nodes, ctx
    return st


# ------------------------------------------------------------------------------------------ plain forms
def _shr(a, n):
    right = (a + torch.where(n > 0, torch.ones_like(n) << (n - 1).clamp(min=0), torch.zeros_like(n))) >> n.clamp(min=0)
    return torch.where(n > 0, right, a << (-n).clamp(min=0))


def _exp(table, d):
    i = (d >> 8).clamp(max=EXP_LEN - 2)
    a, b = table[i], table[i + 1]
    e = a - (((a - b) * (d & 255) + 128) >> 8)
    return torch.where(d < (40 << 16), e, torch.zeros_like(e))


def _rows_of(st, b):
    """K, its shifts and V of sequence b: (S, KV, hd), (S, KV), (S, KV, hd)."""
    S = st["ctx_of"][b] + st["nodes_of"][b]
    pos = torch.arange(S, device="cuda")
    pg, off = st["table"][b].long()[pos // st["page"]], pos % st["page"]
    return st["k"][pg, :, off], st["ks"][pg, :, off], st["v"][pg, :, off]


def _plain_attention(st):
    H, KV, hd = st["H"], st["KV"], st["hd"]
    rep = H // KV
    inv = round(ONE / math.sqrt(hd))
    table = st["exp_t"].long()
    out = torch.empty(st["q"].shape, dtype=torch.int64, device="cuda")
    r0 = 0
    for b, (T, ctx) in enumerate(zip(st["nodes_of"], st["ctx_of"])):
        kb, sb, vb = _rows_of(st, b)
        S = ctx + T
        q = st["q"][r0:r0 + T].view(T, KV, rep, hd).permute(1, 0, 2, 3).reshape(KV, T * rep, hd)
        qs = st["qs"][r0:r0 + T].view(T, KV, rep).permute(1, 0, 2).reshape(KV, T * rep, 1).long()
        node = torch.arange(T, device="cuda")
        see = torch.ones(T, S, dtype=torch.bool, device="cuda")
        see[:, ctx:] = (st["mask"][r0:r0 + T][:, node // 64] >> (node % 64)) & 1 == 1
        see = see.repeat_interleave(rep, 0)
        acc = (q.double() @ kb.permute(1, 2, 0).double()).long()                 # below 2^38
        s = _shr(acc * inv, 32 - qs - sb.permute(1, 0).long()[:, None, :])
        low = torch.iinfo(torch.int64).min // 4
        d = torch.where(see, s, low).amax(-1, keepdim=True) - s
        e = torch.where(see, _exp(table, torch.where(see, d, 0)), 0)
        p = (e << 20) // e.sum(-1, keepdim=True).clamp(min=1)
        vv = vb.permute(1, 0, 2).long()                                          # two halves: sums below 2^37
        o = ((p.double() @ (vv >> 16).double()).long() << 16) + (p.double() @ (vv & 0xFFFF).double()).long()
        o = (o + (1 << 19)) >> 20
        out[r0:r0 + T] = o.view(KV, T, rep, hd).permute(1, 0, 2, 3).reshape(T, H, hd)
        r0 += T
    return out


def _plain_verify(st):
    lg, V = st["logits"], st["V"]
    R = lg.shape[0]
    table = st["exp_t"].long()
    y = (lg * st["tnum"] + (1 << 15)) >> 16
    top = y.amax(1, keepdim=True)
    if st["greedy"]:
        at = torch.arange(V, device="cuda").expand(R, V)
        sampled = torch.where(lg == lg.amax(1, keepdim=True), at, V).amin(1)
    else:
        e = _exp(table, top - y)
        p = (e << 20) // e.sum(1, keepdim=True)
        cum = p.cumsum(1)
        target = (st["u20"].long()[:, None] * cum[:, -1:]) >> 20
        sampled = (cum <= target).sum(1)
    row = torch.arange(R, device="cuda")
    first = st["row_start"].long()
    seq = torch.searchsorted(first, row, right=True) - 1
    par = st["parent"].long()
    gpar = first[seq] + par.clamp(min=0)
    ok = (par >= 0) & (st["tokens"].long() == sampled[gpar])
    nxt = torch.full((R,), R, dtype=torch.int64, device="cuda")
    nxt = nxt.scatter_reduce(0, torch.where(ok, gpar, row), torch.where(ok, row, R), "amin")
    cur, alive = first[:-1], torch.ones(len(first) - 1, dtype=torch.bool, device="cuda")
    path, toks = [], []
    for _ in range(st["max_len"]):
        path.append(torch.where(alive, cur - first[:-1], -1))
        toks.append(torch.where(alive, sampled[cur], -1))
        step = nxt[cur]
        alive = alive & (step < R)
        cur = torch.where(alive, step, cur)
    path = torch.stack(path, 1)
    return [sampled.int(), (path >= 0).sum(1).int(), path.int(), torch.stack(toks, 1).int()]


def _plain_compact(st):
    page, path, n = st["page"], st["path"].long(), st["n_acc"].long()
    B, width = path.shape
    j = torch.arange(width, device="cuda").expand(B, width)
    keep = j < n[:, None]
    seq = torch.arange(B, device="cuda")[:, None].expand(B, width)[keep]
    src, dst = (st["ctx_len"].long()[:, None] + path)[keep], (st["ctx_len"].long()[:, None] + j)[keep]
    t = st["table"].long()
    ps, os, pd, od = t[seq, src // page], src % page, t[seq, dst // page], dst % page
    for name in ("k", "ks", "v"):
        x = st[name]
        x[:, pd, :, od] = x[:, ps, :, os]
    return [(st["ctx_len"] + st["n_acc"]).int(), st["k"], st["ks"], st["v"]]


def _plain_copy(st):
    src, dst = st["src"].long(), st["dst"].long()
    first = torch.arange(st["page"], device="cuda")[None, :] < st["rows"][:, None]          # (n, page)
    for name in ("k", "ks", "v"):
        x = st[name]
        m = first[None, :, None, :] if x.dim() == 4 else first[None, :, None, :, None]
        x[:, dst] = torch.where(m, x[:, src], x[:, dst])
    return [st["k"], st["ks"], st["v"]]


def run(state):
    st = state
    op = st["op"]
    if not own:
        return {"tree_attention": _plain_attention, "tree_verify": _plain_verify, "kv_compact": _plain_compact,
                "kv_copy_pages": _plain_copy}[op](st)
    ex = torch.ops.exact
    if op == "tree_attention":
        return ex.tree_attention(st["q"], st["qs"], st["k"], st["ks"], st["v"], st["table"], st["ctx_len"],
                                 st["row_start"], st["mask"], st["exp_t"])
    if op == "tree_verify":
        return list(ex.tree_verify(st["logits"], st["u20"], st["tokens"], st["parent"], st["row_start"], st["exp_t"],
                                   st["tnum"], st["max_len"]))
    if op == "kv_compact":
        return [ex.kv_compact_(st["k"], st["ks"], st["v"], st["table"], st["ctx_len"], st["path"], st["n_acc"]),
                st["k"], st["ks"], st["v"]]
    ex.kv_copy_pages_(st["k"], st["ks"], st["v"], st["src"], st["dst"], st["rows"])
    return [st["k"], st["ks"], st["v"]]


def work(case):
    """What one pass cannot do without: every input it uses read once, every output written once."""
    op = case["op"]
    if op == "tree_verify":
        R = sum(_lens(dict(case, ctx=0))[1])
        return {"bytes": R * (case["V"] * 8 + 4 * 4), "flops": R * case["V"]}
    row = case["KV"] * (case["hd"] * 6 + 1)                   # K, its shift and V of one position, one layer
    if op == "kv_copy_pages":
        n, page, rows = case["n"], case["page"], case["rows"]
        total = sum(max(1, rows - (7 * i) % rows) if rows < page else page for i in range(n))
        return {"bytes": 2 * case["L"] * row * total, "flops": 0}
    ctx, nodes = _lens(case)
    if op == "kv_compact":
        moved = sum(min(a - 1, n - a) for a, n in zip(_accepted(case), nodes))
        return {"bytes": 2 * case["L"] * row * moved + 4 * sum(_accepted(case)), "flops": 0}
    R, HD = sum(nodes), case["H"] * case["hd"]
    return {"bytes": sum(c + n for c, n in zip(ctx, nodes)) * row + R * (HD * (2 + 8) + case["H"] * 4 + 8),
            "flops": 4 * HD * sum(n * (c + 1) for c, n in zip(ctx, nodes))}


# ------------------------------------------------------------------------------------------ from the definition
def exact(case, seed):
    """The outputs from the definitions, row by row in 64-bit whole numbers on the host."""
    if case["op"] == "tree_attention" and case["H"] * sum(n * (c + n) for c, n in zip(*_lens(case))) > 6_000_000:
        return None                                           # minutes on one core
    st = {k: (x.cpu().numpy() if torch.is_tensor(x) else x) for k, x in prepare(case, seed).items()}
    T = np.array(_exp_table(), np.int64)

    def weights(s):
        d = s.max() - s
        i = np.minimum(d // 256, EXP_LEN - 2)
        drop = (T[i] - T[i + 1]) * (d % 256)
        e = np.where(d >= 40 * ONE, 0, T[i] - (drop + 128) // 256)
        return e * (1 << 20) // int(e.sum())

    op = case["op"]
    if op == "tree_attention":
        H, KV, page = case["H"], case["KV"], case["page"]
        inv = int(round(ONE / math.sqrt(case["hd"])))
        out = np.zeros(st["q"].shape, np.int64)
        r = 0
        for b, (n, c) in enumerate(zip(st["nodes_of"], st["ctx_of"])):
            for i in range(n):
                vis = list(range(c)) + [c + j for j in range(n) if (int(st["mask"][r, j // 64]) >> (j % 64)) & 1]
                pos = np.array(vis, np.int64)
                pg, off = st["table"][b][pos // page], pos % page
                for h in range(H):
                    kv = h // (H // KV)
                    kk, vv = st["k"][pg, kv, off].astype(np.int64), st["v"][pg, kv, off].astype(np.int64)
                    sh = 32 - int(st["qs"][r, h]) - st["ks"][pg, kv, off].astype(np.int64)
                    # whole numbers in floats: every product and partial sum is below 2^53
                    raw = (kk.astype(np.float64) @ st["q"][r, h].astype(np.float64)).astype(np.int64) * inv
                    p = weights((raw + (1 << (sh - 1))) >> sh)
                    hi, lo = vv >> 16, vv & 65535
                    o = (p.astype(np.float64) @ hi.astype(np.float64)).astype(np.int64) * ONE + \
                        (p.astype(np.float64) @ lo.astype(np.float64)).astype(np.int64)
                    out[r, h] = (o + (1 << 19)) >> 20
                r += 1
        return torch.from_numpy(out)
    if op == "tree_verify":
        R, first = len(st["tokens"]), st["row_start"]
        sampled = np.zeros(R, np.int32)
        for r in range(R):
            lg = st["logits"][r]
            if st["u20"][r] < 0:
                sampled[r] = np.argmax(lg)
            else:
                cum = np.cumsum(weights((lg * st["tnum"] + (1 << 15)) >> 16))
                sampled[r] = np.searchsorted(cum, int(st["u20"][r]) * int(cum[-1]) // (1 << 20), side="right")
        path = np.full((case["B"], st["max_len"]), -1, np.int32)
        toks, n = path.copy(), np.zeros(case["B"], np.int32)
        for b in range(case["B"]):
            cur = 0
            while cur is not None:
                t = sampled[first[b] + cur]
                path[b, n[b]], toks[b, n[b]] = cur, t
                n[b] += 1
                kids = [i for i in range(first[b + 1] - first[b])
                        if st["parent"][first[b] + i] == cur and st["tokens"][first[b] + i] == t]
                cur = kids[0] if kids else None
        return [torch.from_numpy(x) for x in (sampled, n, path, toks)]
    page, new = case["page"], {x: st[x].copy() for x in ("k", "ks", "v")}
    if op == "kv_compact":
        for b in range(case["B"]):
            for j in range(int(st["n_acc"][b])):
                s, d = int(st["ctx_len"][b] + st["path"][b, j]), int(st["ctx_len"][b]) + j
                for x in new:
                    new[x][:, st["table"][b, d // page], :, d % page] = st[x][:, st["table"][b, s // page], :, s % page]
        return [torch.from_numpy((st["ctx_len"] + st["n_acc"]).astype(np.int32))] + [torch.from_numpy(new[x]) for x in new]
    for s, d, r in zip(st["src"], st["dst"], st["rows"]):
        for x in new:
            new[x][:, d, :, :r] = st[x][:, s, :, :r]
    return [torch.from_numpy(new[x]) for x in new]
