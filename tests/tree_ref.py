"""Plain implementations of the tree-decoding operators in 64-bit whole numbers (numpy), row by row
from their definitions, and the inputs of their tests.  Integer results: the tolerance is zero."""
import numpy as np

from oracle import exact_oracle as eo

INV = {16: 16384, 32: 11585, 64: 8192, 128: 5793}      # round(2^16 / sqrt(hd))


def attention(q, qs, k, ks, v, table, ctx, row_start, mask):
    """k (P, KV, page, hd), ks (P, KV, page), v (P, KV, page, hd) ... -> int64 (R, H, hd)."""
    R, H, hd = q.shape
    KV, page = k.shape[1], k.shape[2]
    out = np.zeros((R, H, hd), np.int64)
    for b in range(len(ctx)):
        T, c = int(row_start[b + 1] - row_start[b]), int(ctx[b])
        pos = np.arange(c + T)
        pg, off = table[b][pos // page], pos % page
        kb, sb, vb = (x[pg, :, off].astype(np.int64) for x in (k, ks, v))       # (S, KV, ...)
        for i in range(T):
            r = int(row_start[b]) + i
            see = np.concatenate([np.ones(c, bool),
                                  [(int(mask[r, j // 64]) >> (j % 64)) & 1 == 1 for j in range(T)]]).astype(bool)
            if not see.any():
                continue
            for h in range(H):
                g = h // (H // KV)
                acc = kb[see, g] @ q[r, h].astype(np.int64)
                s = eo.shr(acc * INV[hd], 32 - int(qs[r, h]) - sb[see, g])
                p = eo.isoftmax(s[None], np.ones((1, len(s)), bool))[0]
                out[r, h] = eo.shr((p[:, None] * vb[see, g]).sum(0), 20)
    return out


def verify(logits, u20, tokens, parent, row_start, tnum, max_len):
    R, V = logits.shape
    T = eo.EXP_T
    sampled = np.zeros(R, np.int32)
    for r in range(R):
        if u20[r] < 0:
            sampled[r] = int(np.argmax(logits[r]))
            continue
        y = eo.shr(logits[r] * np.int64(tnum), 16)
        d = y.max() - y
        i = np.minimum(d >> 8, len(T) - 2)
        e = np.where(d < (40 << 16), T[i] - eo.shr((T[i] - T[i + 1]) * (d & 255), 8), 0)
        cum = np.cumsum((e << 20) // e.sum())
        sampled[r] = np.searchsorted(cum, (int(u20[r]) * int(cum[-1])) >> 20, side="right")
    B = len(row_start) - 1
    n = np.zeros(B, np.int32)
    path = np.full((B, max_len), -1, np.int32)
    out = path.copy()
    for b in range(B):
        a, z = int(row_start[b]), int(row_start[b + 1])
        cur = 0 if z > a else None
        while cur is not None and n[b] < max_len:
            t = sampled[a + cur]
            path[b, n[b]], out[b, n[b]] = cur, t
            n[b] += 1
            kids = [i for i in range(z - a) if parent[a + i] == cur and tokens[a + i] == t]
            cur = kids[0] if kids else None
    return sampled, n, path, out


def compact(cache, table, ctx, path, n):
    """cache: arrays (L, P, KV, page[, hd]); returns them moved, and the new lengths."""
    page = cache[0].shape[3]
    new = [x.copy() for x in cache]
    for b in range(len(ctx)):
        for j in range(int(n[b])):
            s, d = int(ctx[b] + path[b, j]), int(ctx[b]) + j
            for x, y in zip(cache, new):
                y[:, table[b, d // page], :, d % page] = x[:, table[b, s // page], :, s % page]
    return new, (ctx + n).astype(np.int32)


def masks(parent, row_start, words):
    out = np.zeros((len(parent), words), np.uint64)
    for b in range(len(row_start) - 1):
        a, z = int(row_start[b]), int(row_start[b + 1])
        for i in range(z - a):
            j = i
            while j >= 0:
                out[a + i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
                j = int(parent[a + j])
    return out.view(np.int64)


def parents(rng, nodes):
    return np.concatenate([np.array([-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, n)], np.int32)[:n]
                           for n in nodes] + [np.zeros(0, np.int32)])


def paged(rng, need, page, spare=2):
    """table (B, pages) for sequences of `need` positions, in a random page order, and the pool size."""
    counts = [-(-x // page) for x in need]
    pool = sum(counts) + spare
    ids = rng.permutation(pool)
    table = np.full((len(need), max(counts + [1])), -1, np.int32)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = ids[at:at + c]
        at += c
    return table, pool


def cache(rng, shape, hd, kscale=1.5, vscale=0.8, shifts=None):
    """K rows quantised as the engine stores them, their shifts, V rows."""
    x = (rng.standard_normal((*shape, hd)) * kscale * eo.ONE).astype(np.int64)
    kq, s = eo.qrow(x.reshape(-1, hd))
    k, ks = kq.reshape(*shape, hd).astype(np.int16), s.reshape(shape).astype(np.int8)
    if shifts is not None:
        ks = rng.integers(shifts[0], shifts[1] + 1, shape).astype(np.int8)
    v = (rng.standard_normal((*shape, hd)) * vscale * eo.ONE).astype(np.int64)
    return k, ks, np.clip(v, -2**31, 2**31 - 1).astype(np.int32)


def problem(seed, H, KV, hd, page, ctx, nodes, qscale=2.0, kscale=1.5, vscale=0.8, qshifts=None, kshifts=None,
            words=None):
    """All arguments of tree_attention as numpy arrays."""
    rng = np.random.default_rng(seed)
    row_start = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    R = int(row_start[-1])
    table, pool = paged(rng, [c + n for c, n in zip(ctx, nodes)], page)
    k, ks, v = cache(rng, (pool, KV, page), hd, kscale, vscale, kshifts)
    x = (rng.standard_normal((R * H, hd)) * qscale * eo.ONE).astype(np.int64)
    q, s = eo.qrow(x)
    q, qs = q.reshape(R, H, hd).astype(np.int16), s.reshape(R, H).astype(np.int32)
    if qshifts is not None:
        qs = rng.integers(qshifts[0], qshifts[1] + 1, (R, H)).astype(np.int32)
    parent = parents(rng, nodes)
    words = words or max(1, -(-max(nodes, default=1) // 64))
    return dict(q=q, qs=qs, k=k, ks=ks, v=v, table=table, ctx=np.array(ctx, np.int32), row_start=row_start,
                mask=masks(parent, row_start, words))
