"""Operators of drafted trees (tree attention, verification, cache compaction, page copies) against
plain 64-bit implementations (tests/tree_ref.py), bit for bit, and their refusals."""
import ctypes

import numpy as np
import pytest

from oracle import exact_oracle as eo
from tests import tree_ref as ref


def _ops():
    import exact_llm_b200.ops as ops
    return ops


def _dev(torch, x):
    return torch.from_numpy(np.ascontiguousarray(x)).cuda()


@pytest.fixture(scope="module")
def gpu(cuda_ok):
    import torch
    _ops()
    return torch


@pytest.fixture(scope="module")
def exp_t(gpu):
    return gpu.from_numpy(eo.EXP_T.astype(np.int32)).cuda()


ORDER = ("q", "qs", "k", "ks", "v", "table", "ctx", "row_start", "mask")


def _attend(torch, exp_t, p, status=None, wide=False, **replace):
    a = {n: _dev(torch, p[n]) for n in ORDER}
    if wide:                                                # unused columns: room for 2^20 positions
        page = p["k"].shape[2]
        more = -(-(1 << 20) // page) - p["table"].shape[1]
        a["table"] = torch.nn.functional.pad(a["table"], (0, more), value=-1).contiguous()
    a.update(replace)
    return torch.ops.exact.tree_attention(*[a[n] for n in ORDER], exp_t, status)


# ------------------------------------------------------------------------------------------ host side
def test_tree_masks():
    torch = pytest.importorskip("torch")
    ops = _ops()
    rng = np.random.default_rng(3)
    nodes = [1, 0, 7, 64, 65, 130]
    start = np.concatenate([[0], np.cumsum(nodes)])
    parent = ref.parents(rng, nodes)
    assert np.array_equal(ops.tree_masks(parent.tolist(), start.tolist()).numpy(), ref.masks(parent, start, 3))
    assert ops.tree_masks(torch.tensor([-1, 0]), [0, 2], words=2).shape == (2, 2)
    for bad in (([-1, 1], [0, 2]), ([-1, -2], [0, 2]), ([-1, 0], [0, 1]), ([-1, 0], [1, 2]), ([-1, 0], [0, 2, 1, 2])):
        with pytest.raises(ValueError):
            ops.tree_masks(*bad)
    with pytest.raises(ValueError):
        ops.tree_masks(parent.tolist(), start.tolist(), words=2)


def test_refusals_without_gpu():
    """Every host check of the C entries answers with an error before anything is launched."""
    from exact_llm_b200._lib import KvView, lib

    def view(**kw):
        d = dict(k=4096, ks=4096, v=4096, layers=1, pages=4, KV=2, page=16, hd=64, k_layer=0, k_page=2048, k_head=1024,
                 k_pos=64, s_layer=0, s_page=32, s_head=16, s_pos=1, v_layer=0, v_page=2048, v_head=1024, v_pos=64)
        d.update(kw)
        return ctypes.byref(KvView(**d))

    P = 4096                                               # an aligned address that is never read

    def attn(kv, q=P, qs=P, R=1, H=4, table=P, B=1, mp=2, ctx=P, rs=P, mask=P, w=1, e=P, out=P, ws=P, nb=1 << 40):
        return lib.exb_tree_attention(kv, q, qs, R, H, table, B, mp, ctx, rs, mask, w, e, out, ws, nb, None, None)

    def refused(rc, text):
        msg = lib.exb_last_error().decode()
        assert rc == 1 and text in msg, (rc, msg)

    refused(attn(view(hd=48)), "hd must be")
    refused(attn(view(k=4104)), "16-byte aligned")
    refused(attn(view(k_pos=68)), "multiples of 8")
    refused(attn(view(v_head=1026)), "multiples of 4")
    refused(attn(view(page=0)), "positive")
    refused(attn(view(k=None)), "null cache")
    refused(attn(view(), H=5), "multiple of KV")
    refused(attn(view(), q=None), "null argument")
    refused(attn(view(), out=4100), "aligned")
    refused(attn(view(), w=0), "mask_words")
    refused(attn(view(), w=65), "mask_words")
    refused(attn(view(page=1 << 20), mp=1 << 12), "2^30")
    refused(attn(view(), nb=0), "workspace")
    refused(attn(view(), R=-1), "negative")
    assert attn(view(), R=0) == 0
    ver = lambda lg=P, ld=100, R=1, V=100, tnum=1 << 16, B=1, ml=4, e=P, n=P: lib.exb_tree_verify(  # noqa: E731
        lg, ld, R, V, P, tnum, P, P, P, B, ml, e, P, n, P, P, None)
    refused(ver(ld=99), "row stride")
    refused(ver(tnum=0), "temperature")
    refused(ver(tnum=(1 << 32) + 1), "temperature")
    refused(ver(V=0, ld=0), "V, max_len")
    refused(ver(ml=0), "V, max_len")
    refused(ver(lg=None), "null argument")
    refused(ver(n=None), "null argument")
    comp = lambda kv, B=1, mp=2, path=P, ld=4: lib.exb_kv_compact(kv, P, B, mp, P, path, ld, P, P, None, None)  # noqa: E731
    refused(comp(view(hd=8)), "hd must be")
    refused(comp(view(), B=-1), "B >= 0")
    refused(comp(view(), ld=0), "ld_path")
    refused(comp(view(), path=None), "null argument")
    refused(comp(view(layers=40000)), "65535")
    copy = lambda kv, n=1, src=P: lib.exb_kv_copy_pages(kv, src, P, P, n, None, None)  # noqa: E731
    refused(copy(view(v=4100)), "16-byte aligned")
    refused(copy(view(), n=65536), "count")
    refused(copy(view(), src=None), "null argument")
    assert copy(view(), n=0) == 0


def test_shapes_without_gpu():
    """The fake implementations give the outputs' shapes and refuse what the kernels refuse."""
    torch = pytest.importorskip("torch")
    _ops()
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        i32, i16 = torch.int32, torch.int16
        q, qs = torch.empty(3, 4, 64, dtype=i16), torch.empty(3, 4, dtype=i32)
        k, ks, v = torch.empty(5, 2, 16, 64, dtype=i16), torch.empty(5, 2, 16, dtype=torch.int8), torch.empty(5, 2, 16, 64, dtype=i32)
        t, c, rs = torch.empty(2, 3, dtype=i32), torch.empty(2, dtype=i32), torch.empty(3, dtype=i32)
        m, e = torch.empty(3, 1, dtype=torch.int64), torch.empty(10242, dtype=i32)
        o = torch.ops.exact.tree_attention(q, qs, k, ks, v, t, c, rs, m, e)
        assert o.shape == (3, 4, 64) and o.dtype == torch.int64
        with pytest.raises(ValueError):
            torch.ops.exact.tree_attention(q[:, :3], qs[:, :3], k, ks, v, t, c, rs, m, e)
        with pytest.raises(TypeError):
            torch.ops.exact.tree_attention(q, qs.long(), k, ks, v, t, c, rs, m, e)
        lg = torch.empty(3, 50, dtype=torch.int64)
        s, n, p, x = torch.ops.exact.tree_verify(lg, c.new_empty(3), c.new_empty(3), c.new_empty(3), rs, e, 1 << 16, 7)
        assert (s.shape, n.shape, p.shape, x.shape) == ((3,), (2,), (2, 7), (2, 7))
        new = torch.ops.exact.kv_compact_(k[None], ks[None], v[None], t, c, t, c)
        assert new.shape == (2,) and new.dtype == i32
        assert torch.ops.exact.kv_copy_pages_(k[None], ks[None], v[None], c, c, c) is None


# ------------------------------------------------------------------------------------------ attention
ATTENTION = {
    "one token of an empty sequence": dict(H=4, KV=2, hd=16, page=16, ctx=[0], nodes=[1]),
    "width 32, pages of one position": dict(H=6, KV=2, hd=32, page=1, ctx=[5], nodes=[3]),
    "width 64, odd pages": dict(H=14, KV=2, hd=64, page=100, ctx=[99, 100, 101], nodes=[1, 2, 5]),
    "single tokens of many sequences": dict(H=28, KV=4, hd=128, page=48, ctx=[0, 1, 15, 16, 47, 48, 200, 331, 7],
                                            nodes=[1] * 9),
    "page end inside the tree": dict(H=28, KV=4, hd=128, page=64, ctx=[61], nodes=[26]),
    "an empty sequence in between": dict(H=5, KV=1, hd=128, page=32, ctx=[10, 40, 0], nodes=[4, 0, 9]),
    "one head a group": dict(H=16, KV=16, hd=128, page=256, ctx=[130, 3], nodes=[17, 33]),
    "eight heads a group": dict(H=16, KV=2, hd=64, page=16, ctx=[200], nodes=[31]),
    "65 nodes, two words": dict(H=4, KV=2, hd=32, page=64, ctx=[33], nodes=[65]),
    "130 nodes, three words": dict(H=10, KV=2, hd=128, page=128, ctx=[70, 0], nodes=[130, 2]),
    "long context": dict(H=10, KV=2, hd=128, page=256, ctx=[5003], nodes=[3]),
    "long context, single token": dict(H=4, KV=2, hd=64, page=128, ctx=[20011], nodes=[1]),
    "long context, width 16": dict(H=4, KV=2, hd=16, page=128, ctx=[3333], nodes=[20]),
    "wide tree, long context": dict(H=7, KV=1, hd=128, page=64, ctx=[2500], nodes=[61]),
    "large values": dict(H=7, KV=1, hd=128, page=64, ctx=[200], nodes=[20], vscale=2.0**14),
    "sharp scores": dict(H=6, KV=2, hd=128, page=64, ctx=[300], nodes=[12], qscale=20.0, kscale=20.0),
    "flat scores": dict(H=6, KV=2, hd=128, page=64, ctx=[300], nodes=[12], qscale=0.01, kscale=0.01),
    "shifts past 32 bits": dict(H=6, KV=2, hd=128, page=64, ctx=[300], nodes=[12], qshifts=(6, 9), kshifts=(6, 10)),
    "left shifts": dict(H=6, KV=2, hd=64, page=64, ctx=[150], nodes=[9], qshifts=(18, 22), kshifts=(12, 22)),
    "mixed shifts": dict(H=14, KV=2, hd=64, page=32, ctx=[700], nodes=[40], qshifts=(0, 22), kshifts=(0, 22)),
    "mixed shifts, wide tree": dict(H=14, KV=2, hd=128, page=32, ctx=[400], nodes=[63], qshifts=(0, 14), kshifts=(0, 14)),
}


# A table with room for a long cache takes the kernels for long caches, whatever the lengths in it are.
WIDE = pytest.mark.parametrize("wide", [False, True], ids=["", "long table"])


@pytest.mark.gpu
@WIDE
@pytest.mark.parametrize("name", list(ATTENTION))
def test_attention(gpu, exp_t, name, wide):
    p = ref.problem(len(name), **ATTENTION[name])
    status = gpu.zeros(1, dtype=gpu.int32, device="cuda")
    got = _attend(gpu, exp_t, p, status, wide).cpu().numpy()
    assert np.array_equal(got, ref.attention(**p))
    assert int(status) == 0


@pytest.mark.gpu
@WIDE
@pytest.mark.parametrize("hd", [16, 32, 64, 128])
@pytest.mark.parametrize("nodes", [1, 3, 40])
def test_attention_extreme_values(gpu, exp_t, hd, nodes, wide):
    """Every factor at the end of its type: sums and digits at their largest."""
    for seed, (qv, kv, vv) in enumerate([(32767, 32767, 2**31 - 1), (-32768, 32767, -2**31), (-32768, -32768, -1),
                                         (255, -256, 2**23), (-1, 1, -2**23 - 1)]):
        p = ref.problem(seed, H=4, KV=2, hd=hd, page=64, ctx=[150], nodes=[nodes])
        p["q"][:] = qv
        p["k"][:] = kv
        p["k"][..., ::3] = -1 - kv                          # scores that differ from row to row
        p["k"][:, :, ::2] = kv
        p["v"][:] = vv
        p["v"][:, :, 1::3] = -1 - vv
        p["qs"][:], p["ks"][:] = 0, 0
        assert np.array_equal(_attend(gpu, exp_t, p, None, wide).cpu().numpy(), ref.attention(**p)), seed


@pytest.mark.gpu
@WIDE
@pytest.mark.parametrize("seed", range(12))
def test_attention_random(gpu, exp_t, seed, wide):
    rng = np.random.default_rng(1000 + seed)
    KV, rep, hd = int(rng.integers(1, 5)), int(rng.integers(1, 9)), int(rng.choice([16, 32, 64, 128]))
    B = int(rng.integers(1, 6))
    ctx = [int(x) for x in np.exp(rng.uniform(0, 7, B)).astype(int) - 1]
    nodes = [int(x) for x in np.exp(rng.uniform(0, 4.3, B)).astype(int)]
    p = ref.problem(seed, H=KV * rep, KV=KV, hd=hd, page=int(rng.choice([1, 7, 16, 64, 100])), ctx=ctx, nodes=nodes)
    assert np.array_equal(_attend(gpu, exp_t, p, None, wide).cpu().numpy(), ref.attention(**p))


@pytest.mark.gpu
@WIDE
@pytest.mark.parametrize("seed", range(4))
def test_attention_many_short_sequences(gpu, exp_t, seed, wide):
    """More sequences than SMs, of a few hundred positions at most and trees of all sizes: every CTA goes through
    several short pieces of work."""
    rng = np.random.default_rng(50 + seed)
    B = 250
    nodes = rng.integers(1, [5, 30, 40, 64][seed], B)
    ctx = rng.integers(0, [100, 300, 200, 100][seed], B)
    p = ref.problem(seed, H=8, KV=2, hd=[64, 32, 128, 16][seed], page=16, ctx=[int(x) for x in ctx], nodes=[int(x) for x in nodes])
    want = ref.attention(**p)
    for _ in range(3):
        assert np.array_equal(_attend(gpu, exp_t, p, None, wide).cpu().numpy(), want)


@pytest.mark.gpu
@WIDE
def test_attention_masks(gpu, exp_t, wide):
    """Rows that see nothing give zeros; bits past the tree count for nothing; any set of nodes will do."""
    p = ref.problem(5, H=6, KV=2, hd=64, page=16, ctx=[0, 20], nodes=[9, 70], words=3)
    rng = np.random.default_rng(0)
    p["mask"] = rng.integers(-2**63, 2**63, p["mask"].shape, dtype=np.int64)
    p["mask"][2] = 0                                        # no context, no node
    p["mask"][5] = np.int64(-1) << np.int64(9)              # only bits past the tree
    p["mask"][12] = 0                                       # the context alone
    got = _attend(gpu, exp_t, p, None, wide).cpu().numpy()
    assert np.array_equal(got, ref.attention(**p))
    assert not got[2].any() and not got[5].any() and got[12].any()


@pytest.mark.gpu
@WIDE
def test_attention_ignores_stale_rows(gpu, exp_t, wide):
    """Positions past the tree, other pages and hidden nodes hold anything: no bit changes."""
    p = ref.problem(6, H=14, KV=2, hd=64, page=32, ctx=[50, 200], nodes=[5, 40])
    want = ref.attention(**p)
    used = np.zeros(p["ks"].shape, bool)
    for b in range(2):
        pos = np.arange(p["ctx"][b] + [5, 40][b])
        used[p["table"][b][pos // 32], :, pos % 32] = True
    for n, x in (("k", -32768), ("ks", 127), ("v", -2**31)):
        p[n][~used] = x
    assert np.array_equal(_attend(gpu, exp_t, p, None, wide).cpu().numpy(), want)


@pytest.mark.gpu
@WIDE
def test_attention_strides(gpu, exp_t, wide):
    """A layer of a slot cache, head-last storage, padded rows: the same bits, and the rows of other layers unread."""
    torch = gpu
    p = ref.problem(7, H=10, KV=2, hd=64, page=48, ctx=[100, 30], nodes=[7, 20])
    want = ref.attention(**p)
    for how in ("layer", "positions first", "padded", "keys padded", "values padded"):
        new = {}
        for n in ("k", "ks", "v"):
            x = _dev(torch, p[n])
            if how == "layer":
                new[n] = torch.stack([x.roll(1, 0), x, x.roll(2, 0)])[1]
            elif how == "positions first":
                new[n] = x.transpose(1, 2).contiguous().transpose(1, 2)
            elif n in {"padded": "kv", "keys padded": "k", "values padded": "v"}[how]:
                pad = torch.full((*x.shape[:-1], x.shape[-1] + 8), -7, dtype=x.dtype, device="cuda")
                pad[..., :x.shape[-1]] = x
                new[n] = pad[..., :x.shape[-1]]
        assert np.array_equal(_attend(torch, exp_t, p, None, wide, **new).cpu().numpy(), want), how


def _far(torch, x, pages):
    """The array with its pages (axis `pages`) more than 2^29 elements apart: offsets past 32 bits."""
    stride, at = [0] * x.ndim, 1
    for i in [i for i in reversed(range(x.ndim)) if i != pages]:
        stride[i], at = at, at * x.shape[i]
    stride[pages] = (1 << 29) + 64
    assert at <= stride[pages] and x.shape[pages] * stride[pages] > 1 << 31
    far = torch.empty_strided(x.shape, stride, dtype=_dev(torch, x[:0]).dtype, device="cuda")
    return far.copy_(_dev(torch, x))


@pytest.mark.gpu
@WIDE
def test_attention_far_pages(gpu, exp_t, wide):
    p = ref.problem(11, H=6, KV=2, hd=64, page=16, ctx=[50, 3], nodes=[7, 20])
    far = {n: _far(gpu, p[n], 0) for n in ("k", "v")}
    assert np.array_equal(_attend(gpu, exp_t, p, None, wide, **far).cpu().numpy(), ref.attention(**p))


@pytest.mark.gpu
@WIDE
def test_attention_out_of_range(gpu, exp_t, wide):
    """A page id or a position that does not exist is left out and reported, never read."""
    torch = gpu
    p = ref.problem(8, H=4, KV=2, hd=32, page=16, ctx=[40], nodes=[6])
    for bad in (-1, len(p["k"]), 2**31 - 1):
        x = dict(p, table=p["table"].copy())
        x["table"][0, 1] = bad                              # positions 16..31 are gone
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = _attend(torch, exp_t, x, status, wide).cpu().numpy()
        assert int(status) == 8
        keep = np.r_[0:16, 32:46]
        y = dict(p, table=np.array([[0, 1]], np.int32), ctx=np.array([24], np.int32))
        for n in ("k", "ks", "v"):                          # the rest, laid out anew
            rows = p[n][p["table"][0][keep // 16], :, keep % 16]
            rows = np.concatenate([rows, rows[:2]])
            y[n] = np.ascontiguousarray(rows.reshape(2, 16, *rows.shape[1:]).swapaxes(1, 2))
        assert np.array_equal(got, ref.attention(**y))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    _attend(torch, exp_t, dict(p, ctx=np.array([43], np.int32)), status, wide)  # a node past the table's end
    assert int(status) == 8
    for rs in ([0, 7], [-1, 6], [4, 2]):
        status.zero_()
        got = _attend(torch, exp_t, dict(p, row_start=np.array(rs, np.int32)), status, wide)
        assert int(status) == 8 and not got.any()
    got = _attend(torch, exp_t, dict(p, row_start=np.array([2, 5], np.int32)), None, wide)   # rows that no sequence owns
    assert not got[:2].any() and not got[5:].any() and got[2:5].any()


@pytest.mark.gpu
def test_attention_stream_and_graph(gpu, exp_t):
    """On a side stream, and captured in a graph that is replayed on other contexts."""
    torch = gpu
    p = ref.problem(9, H=14, KV=2, hd=64, page=32, ctx=[100, 7], nodes=[5, 18])
    want = ref.attention(**p)
    a = {n: _dev(torch, p[n]) for n in ORDER}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.ops.exact.tree_attention(*[a[n] for n in ORDER], exp_t)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            again = torch.ops.exact.tree_attention(*[a[n] for n in ORDER], exp_t)
    side.synchronize()
    assert np.array_equal(got.cpu().numpy(), want)
    for ctx in ([100, 7], [33, 0]):
        a["ctx"].copy_(torch.tensor(ctx, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(again.cpu().numpy(), ref.attention(**dict(p, ctx=np.array(ctx, np.int32))))


@pytest.mark.gpu
def test_attention_refusals(gpu, exp_t):
    p = ref.problem(10, H=4, KV=2, hd=16, page=16, ctx=[4], nodes=[3])
    from exact_llm_b200 import ExbError
    t = {n: _dev(gpu, p[n]) for n in ORDER}
    bad = [(dict(q=t["q"].int()), ValueError), (dict(qs=t["qs"].long()), TypeError), (dict(qs=t["qs"][:2]), ValueError),
           (dict(k=t["k"].int()), TypeError), (dict(v=t["v"][..., :8]), ValueError), (dict(table=t["table"][0]), ValueError),
           (dict(mask=t["mask"][:2]), ValueError), (dict(row_start=t["row_start"][:1]), ValueError),
           (dict(ctx=t["ctx"].cpu()), Exception), (dict(q=t["q"][:, :3].contiguous(), qs=t["qs"][:, :3].contiguous()), ValueError),
           (dict(k=gpu.zeros(t["k"].numel() + 4, dtype=gpu.int16, device="cuda")[4:].view(t["k"].shape)), ExbError)]
    for change, error in bad:
        with pytest.raises(error):
            _attend(gpu, exp_t, p, **change)
    assert _attend(gpu, exp_t, p, q=t["q"][:0], qs=t["qs"][:0], mask=t["mask"][:0]).shape == (0, 4, 16)


# ------------------------------------------------------------------------------------------ verification
def _verify_problem(seed, V, nodes, spread=2.5, greedy=0.2, hit=0.7, tnum=1 << 16):
    rng = np.random.default_rng(seed)
    rs = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    R = int(rs[-1])
    lg = (rng.standard_normal((R, V)) * spread * eo.ONE).astype(np.int64)
    parent = ref.parents(rng, nodes)
    u = rng.integers(0, 1 << 20, R).astype(np.int32)
    u[rng.random(R) < greedy] = -1
    t = ref.verify(lg, u, np.zeros(R, np.int32), parent, rs, tnum, 1)[0]        # the target's choices
    tok = rng.integers(0, V, R).astype(np.int32)
    for b in range(len(nodes)):
        for i in range(rs[b] + 1, rs[b + 1]):
            if rng.random() < hit:
                tok[i] = t[rs[b] + parent[i]]
    return dict(logits=lg, u20=u, tokens=tok, parent=parent, row_start=rs, tnum=tnum, max_len=max(nodes + [1]))


def _verify(torch, exp_t, p, logits=None):
    d = {n: _dev(torch, p[n]) for n in ("logits", "u20", "tokens", "parent", "row_start")}
    if logits is not None:
        d["logits"] = logits
    got = torch.ops.exact.tree_verify(d["logits"], d["u20"], d["tokens"], d["parent"], d["row_start"], exp_t, p["tnum"],
                                      p["max_len"])
    return [x.cpu().numpy() for x in got]


def _same(got, want):
    return all(np.array_equal(a, b) and a.dtype == b.dtype for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [1, 2, 31, 1000, 1024, 1025, 4099, 30001, 65537])
def test_verify(gpu, exp_t, V):
    for seed, nodes in enumerate([[1], [5, 0, 33], [70, 2]]):
        p = _verify_problem(seed, V, nodes, tnum=[1 << 16, 81920, 1, 1 << 20][seed + (V % 2)])
        assert _same(_verify(gpu, exp_t, p), ref.verify(**p)), (V, nodes)


@pytest.mark.gpu
@pytest.mark.parametrize("V", [151936, 152064, 262147])
def test_verify_vocabularies(gpu, exp_t, V):
    p = _verify_problem(V, V, [4, 9])
    assert _same(_verify(gpu, exp_t, p), ref.verify(**p))


@pytest.mark.gpu
@pytest.mark.parametrize("V,tnum", [(327680, 1 << 16), (327681, 1 << 16), (400001, 81920), (5000, (1 << 31) - 1),
                                    (5000, 1 << 31), (5000, 1 << 32)])
def test_verify_any_length_any_temperature(gpu, exp_t, V, tnum):
    """Either side of what the clusters hold in registers, and of what their 32-bit products can scale."""
    p = _verify_problem(V, V, [3, 2], spread=2.5 * (1 << 16) / tnum, tnum=tnum)
    assert _same(_verify(gpu, exp_t, p), ref.verify(**p))
    for i in range(5):                                       # scaled logits around 2^30
        p["logits"][i] = np.random.default_rng(i).integers(-3, 3, V) + (((1 << 46) // tnum) + 1 if i % 2 else -((1 << 46) // tnum))
    assert _same(_verify(gpu, exp_t, p), ref.verify(**p))


@pytest.mark.gpu
def test_verify_edges(gpu, exp_t):
    """Ties, extreme logits, the ends of the random numbers' range, rows of a wider array, a short path buffer."""
    torch = gpu
    for V in (97, 5000, 152064):
        p = _verify_problem(V, V, [12, 6], greedy=0.0)
        lg = p["logits"]
        lg[0] = 0                                            # all equal
        lg[1] = -(1 << 40); lg[1, V - 1] = 1 << 40           # one token
        lg[2] = -(1 << 40); lg[2, 0] = lg[2, V // 2] = 5     # two
        lg[3] = -(1 << 46)
        lg[4, 7] = lg[4, 70] = lg[4].max() + 1
        p["u20"][:6] = [0, (1 << 20) - 1, 1 << 19, (1 << 20) - 1, 0, 1]
        p["u20"][6:9] = -1
        lg[6] = 3                                            # argmax of equal logits: the lowest index
        lg[7, V - 1] = lg[7].max() + 1
        lg[8, 0] = lg[8, 90] = lg[8].max() + 9
        assert _same(_verify(torch, exp_t, p), ref.verify(**p)), V
        wide = torch.full((len(lg), V + 5), 1 << 50, dtype=torch.int64, device="cuda")
        wide[:, :V] = _dev(torch, lg)
        assert _same(_verify(torch, exp_t, p, wide[:, :V]), ref.verify(**p))
        p["max_len"] = 2
        assert _same(_verify(torch, exp_t, p), ref.verify(**p))


@pytest.mark.gpu
def test_verify_is_the_sampler(gpu, exp_t):
    """A row's token is the one that the engine's sampler draws with that seed and position."""
    p = _verify_problem(4, 2000, [6], greedy=0.0, tnum=eo.temp_num(0.7))
    p["u20"] = np.array([eo.u20(99, i) for i in range(6)], np.int32)
    got = _verify(gpu, exp_t, p)[0]
    assert got.tolist() == [eo.sample_int(p["logits"][i], 99, i, p["tnum"])[0] for i in range(6)]


@pytest.mark.gpu
def test_verify_refusals(gpu, exp_t):
    torch = gpu
    p = _verify_problem(1, 50, [4])
    d = [_dev(torch, p[n]) for n in ("logits", "u20", "tokens", "parent", "row_start")]
    f = torch.ops.exact.tree_verify
    from exact_llm_b200 import ExbError
    for args, error in [((d[0].int(), *d[1:], exp_t, 1, 3), ValueError), ((*d, exp_t, 1, 0), ValueError),
                        ((d[0], d[1].long(), *d[2:], exp_t, 1, 3), TypeError), ((d[0], d[1][:2], *d[2:], exp_t, 1, 3), ValueError),
                        ((*d, exp_t[:9], 1, 3), ValueError), ((*d, exp_t, 0, 3), ExbError), ((*d, exp_t, 1 << 33, 3), ExbError),
                        ((d[0].t().contiguous().t(), *d[1:], exp_t, 1, 3), ValueError)]:
        with pytest.raises(error):
            f(*args)
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    s, n, path, tok = f(d[0][:0], none, none, none, torch.zeros(3, dtype=torch.int32, device="cuda"), exp_t, 1 << 16, 2)
    assert s.numel() == 0 and n.tolist() == [0, 0] and (path == -1).all() and (tok == -1).all()


# ------------------------------------------------------------------------------------------ cache rows
def _paths(rng, nodes, acc):
    out = np.full((len(nodes), max(acc + [1])), -1, np.int32)
    for b, (t, a) in enumerate(zip(nodes, acc)):
        if a:
            out[b, :a] = np.sort(rng.choice(t, a, replace=False))
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("L,KV,hd,page", [(1, 1, 16, 1), (3, 2, 32, 7), (2, 4, 64, 16), (24, 2, 64, 64), (5, 3, 128, 100)])
def test_compact(gpu, L, KV, hd, page):
    torch = gpu
    for seed, (ctx, nodes, acc) in enumerate([([0], [1], [1]), ([13, 0, 64], [9, 64, 20], [4, 31, 20]), ([5, 9], [3, 3], [0, 3])]):
        rng = np.random.default_rng(seed)
        table, pool = ref.paged(rng, [c + t for c, t in zip(ctx, nodes)], page)
        cache = [rng.integers(-100, 100, (L, pool, KV, page, hd)).astype(np.int16),
                 rng.integers(0, 20, (L, pool, KV, page)).astype(np.int8),
                 rng.integers(-2**31, 2**31, (L, pool, KV, page, hd)).astype(np.int32)]
        path, n = _paths(rng, nodes, acc), np.array(acc, np.int32)
        dev = [_dev(torch, x) for x in cache]
        new = torch.ops.exact.kv_compact_(*dev, _dev(torch, table), _dev(torch, np.array(ctx, np.int32)),
                                          _dev(torch, path), _dev(torch, n))
        want, lens = ref.compact(cache, table, np.array(ctx, np.int32), path, n)
        assert np.array_equal(new.cpu().numpy(), lens)
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(dev, want))


@pytest.mark.gpu
def test_compact_malformed(gpu):
    """A path that is not strictly increasing, or leaves the table, moves nothing in its sequence."""
    torch = gpu
    rng = np.random.default_rng(0)
    table, pool = ref.paged(rng, [40, 40], 16)
    cache = [rng.integers(-9, 9, (2, pool, 2, 16, 32)).astype(np.int16), rng.integers(0, 9, (2, pool, 2, 16)).astype(np.int8),
             rng.integers(-9, 9, (2, pool, 2, 16, 32)).astype(np.int32)]
    good = [0, 3, 5, 8]
    for first, n0, ctx0 in (([0, 3, 3, 8], 4, 10), ([0, 5, 4, 8], 4, 10), ([-1, 1, 2, 3], 4, 10), ([0, 1, 2, 38], 4, 10),
                            (good, 5, 10), (good, -1, 10), (good, 4, -3), ([0, 1, 2, 2**31 - 1], 4, 10)):
        dev = [_dev(torch, x) for x in cache]
        ctx, n = np.array([ctx0, 20], np.int32), np.array([n0, 4], np.int32)
        path = np.array([first, good], np.int32)
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        new = torch.ops.exact.kv_compact_(*dev, _dev(torch, table), _dev(torch, ctx), _dev(torch, path), _dev(torch, n), status)
        want, _ = ref.compact(cache, table, ctx, path, np.array([0, 4]))
        assert new.tolist() == [ctx0, 24] and int(status) == 8
        assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(dev, want))
    t2 = table.copy()
    t2[0, 0] = pool                                          # a page that is not there
    dev = [_dev(torch, x) for x in cache]
    new = torch.ops.exact.kv_compact_(*dev, _dev(torch, t2), _dev(torch, np.array([10, 20], np.int32)),
                                      _dev(torch, np.array([good, good], np.int32)), _dev(torch, np.array([4, 0], np.int32)))
    assert new.tolist() == [10, 20] and all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(dev, cache))


@pytest.mark.gpu
@pytest.mark.parametrize("L,KV,hd,page", [(1, 1, 16, 1), (2, 3, 32, 7), (3, 2, 64, 64), (2, 2, 128, 300)])
def test_copy_pages(gpu, L, KV, hd, page):
    torch = gpu
    rng = np.random.default_rng(page)
    pool = 9
    cache = [rng.integers(-99, 99, (L, pool, KV, page, hd)).astype(np.int16), rng.integers(0, 20, (L, pool, KV, page)).astype(np.int8),
             rng.integers(-2**31, 2**31, (L, pool, KV, page, hd)).astype(np.int32)]
    src, dst = np.array([7, 7, 2, 0], np.int32), np.array([1, 8, 4, 3], np.int32)      # one page to two targets
    rows = np.array([page, (page + 1) // 2, 0, min(1, page)], np.int32)
    want = [x.copy() for x in cache]
    for s, d, r in zip(src, dst, rows):
        for x, y in zip(cache, want):
            y[:, d, :, :r] = x[:, s, :, :r]
    dev = [_dev(torch, x) for x in cache]
    torch.ops.exact.kv_copy_pages_(*dev, _dev(torch, src), _dev(torch, dst), _dev(torch, rows))
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(dev, want))
    status = torch.zeros(1, dtype=torch.int32, device="cuda")                           # entries out of range: skipped
    torch.ops.exact.kv_copy_pages_(*dev, _dev(torch, np.array([pool, 0, 0, 0], np.int32)),
                                   _dev(torch, np.array([0, -1, 1, 2], np.int32)),
                                   _dev(torch, np.array([1, 1, page + 1, -1], np.int32)), status)
    assert int(status) == 8 and all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(dev, want))


@pytest.mark.gpu
def test_cache_strides(gpu):
    """Caches whose layers, heads and positions are stored in another order."""
    torch = gpu
    rng = np.random.default_rng(2)
    table, pool = ref.paged(rng, [30], 8)
    cache = [rng.integers(-9, 9, (2, pool, 3, 8, 32)).astype(np.int16), rng.integers(0, 9, (2, pool, 3, 8)).astype(np.int8),
             rng.integers(-9, 9, (2, pool, 3, 8, 32)).astype(np.int32)]
    path, n, ctx = np.array([[1, 4, 6]], np.int32), np.array([3], np.int32), np.array([20], np.int32)
    perm = (1, 3, 0, 2)
    dev = []
    for x in cache:
        order = perm + (4,) * (x.ndim == 5)
        dev.append(_dev(torch, x).permute(order).contiguous().permute(np.argsort(order).tolist()))
    torch.ops.exact.kv_compact_(*dev, _dev(torch, table), _dev(torch, ctx), _dev(torch, path), _dev(torch, n))
    want, _ = ref.compact(cache, table, ctx, path, n)
    free = [i for i in range(pool) if i not in table]
    torch.ops.exact.kv_copy_pages_(*dev, *[_dev(torch, np.array([x], np.int32)) for x in (table[0, 1], free[0], 5)])
    for y in want:
        y[:, free[0], :, :5] = y[:, table[0, 1], :, :5]
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(dev, want))


@pytest.mark.gpu
def test_cache_far_pages(gpu):
    """Pages more than 2^29 elements apart."""
    torch = gpu
    rng = np.random.default_rng(3)
    table, pool = ref.paged(rng, [40], 16)
    cache = [rng.integers(-9, 9, (2, pool, 2, 16, 32)).astype(np.int16), rng.integers(0, 9, (2, pool, 2, 16)).astype(np.int8),
             rng.integers(-9, 9, (2, pool, 2, 16, 32)).astype(np.int32)]
    path, n, ctx = np.array([[1, 4, 11]], np.int32), np.array([3], np.int32), np.array([20], np.int32)
    dev = [_far(torch, cache[0], 1), _dev(torch, cache[1]), _far(torch, cache[2], 1)]
    torch.ops.exact.kv_compact_(*dev, _dev(torch, table), _dev(torch, ctx), _dev(torch, path), _dev(torch, n))
    want, _ = ref.compact(cache, table, ctx, path, n)
    free = [i for i in range(pool) if i not in table][0]
    torch.ops.exact.kv_copy_pages_(*dev, *[_dev(torch, np.array([x], np.int32)) for x in (table[0, 1], free, 5)])
    for y in want:
        y[:, free, :, :5] = y[:, table[0, 1], :, :5]
    assert all(np.array_equal(a.cpu().numpy(), b) for a, b in zip(dev, want))


@pytest.mark.gpu
def test_cache_refusals(gpu):
    torch = gpu
    k, ks, v = (torch.zeros(2, 4, 2, 16, 32, dtype=torch.int16, device="cuda"), torch.zeros(2, 4, 2, 16, dtype=torch.int8, device="cuda"),
                torch.zeros(2, 4, 2, 16, 32, dtype=torch.int32, device="cuda"))
    i = torch.zeros(1, dtype=torch.int32, device="cuda")
    t = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    for f in (lambda: torch.ops.exact.kv_compact_(k[0], ks[0], v[0], t, i, t, i), lambda: torch.ops.exact.kv_compact_(k, ks, v, t, i, t, t),
              lambda: torch.ops.exact.kv_copy_pages_(k, ks, v, i, t[0], i),
              lambda: torch.ops.exact.kv_copy_pages_(k, ks, v[:, :3], i, i, i),
              lambda: torch.ops.exact.kv_copy_pages_(k.transpose(3, 4), ks, v, i, i, i)):
        with pytest.raises(ValueError):
            f()
    with pytest.raises(TypeError):
        torch.ops.exact.kv_copy_pages_(k.int(), ks, v, i, i, i)
