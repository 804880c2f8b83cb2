"""Edges of the drafted-tree operators and of the engine's step on trees: sums, scores and random numbers at
the ends of their ranges, malformed row ranges and arguments."""
import ctypes

import numpy as np
import pytest

from tests import tree_ref as ref
from tests.test_tree_ops import WIDE, _attend, _same, _verify, _verify_problem, exp_t, gpu  # noqa: F401


# ------------------------------------------------------------------------------------------ attention
@pytest.mark.gpu
@pytest.mark.parametrize("positions", [(1 << 18) - 1, 1 << 18, (1 << 18) + 1, 349526, 1 << 19, (1 << 20) + 1])
def test_attention_flat_rows_of_long_caches(gpu, exp_t, positions):  # noqa: F811
    """2^18 equal scores and more: the row's sum is 2^42 or more and a probability at most 4."""
    p = ref.problem(positions, H=1, KV=1, hd=16, page=4096, ctx=[positions - 1], nodes=[1], vscale=2.0**13)
    p["q"][:] = 0
    want = ref.attention(**p)
    assert want.any() == (positions <= 1 << 20)
    assert np.array_equal(_attend(gpu, exp_t, p).cpu().numpy(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("positions,qscale", [(400000, 0.02), (700001, 0.1), (1500000, 0.3)])
def test_attention_small_probabilities(gpu, exp_t, positions, qscale):  # noqa: F811
    """The same with scores of a small spread: probabilities of 0 to 4 side by side, two heads a group."""
    p = ref.problem(positions, H=2, KV=1, hd=16, page=1024, ctx=[positions - 3], nodes=[3], qscale=qscale, vscale=2.0**13)
    want = ref.attention(**p)
    assert want.any()
    assert np.array_equal(_attend(gpu, exp_t, p).cpu().numpy(), want)


@pytest.mark.gpu
@WIDE
@pytest.mark.parametrize("below", [0, 16])
def test_attention_lowest_32_bit_score(gpu, exp_t, wide, below):  # noqa: F811
    """A row whose largest score is -2^31 exactly sees its positions all the same."""
    p = ref.problem(12, H=4, KV=2, hd=64, page=32, ctx=[300], nodes=[5])
    p["q"][:], p["k"][:] = -16384, 16384 + below             # q.k = -2^34: times 2^13, shifted by 16
    p["k"][p["table"][0, 0]] = 16384
    p["qs"][:], p["ks"][:] = 9, 7
    want = ref.attention(**p)
    assert want.any()
    assert np.array_equal(_attend(gpu, exp_t, p, None, wide).cpu().numpy(), want)


@pytest.mark.gpu
@WIDE
@pytest.mark.parametrize("hd,nodes", [(16, 3), (128, 100)])
def test_attention_overlapping_rows(gpu, exp_t, wide, hd, nodes):  # noqa: F811
    """Where row_start falls, the range that falls and the ones that begin before an earlier one's end are left out:
    their rows are zeros, and the others have their values."""
    torch = gpu
    p = ref.problem(13, H=14, KV=2, hd=hd, page=64, ctx=[70, 20, 30, 9], nodes=[2 * nodes, 0, nodes, 5], words=8)
    a, b, R = 2 * nodes, 3 * nodes, 3 * nodes + 5
    want = ref.attention(**p)
    want[a:b] = 0
    bad = dict(p, row_start=np.array([0, a, nodes, b, R], np.int32))       # 1: falls; 2: begins inside 0's rows
    table = np.full((4, 64), -1, np.int32)
    table[:, :p["table"].shape[1]] = p["table"]
    table[2, :] = 0                                          # (all of its positions would be there)
    bad["table"] = table
    for _ in range(2):
        junk = torch.full((R, 14, hd), -1, dtype=torch.int64, device="cuda")
        del junk                                             # what the output's memory holds before the call
        status = torch.zeros(1, dtype=torch.int32, device="cuda")
        got = _attend(torch, exp_t, bad, status, wide).cpu().numpy()
        assert int(status) == 8
        assert np.array_equal(got, want)


@pytest.mark.gpu
@WIDE
@pytest.mark.parametrize("falls", [(4,), (31,), (32,), (33, 34), (5, 32, 64), (69,)])
def test_attention_overlapping_rows_of_many(gpu, exp_t, wide, falls):  # noqa: F811
    """The same among 70 sequences: the two ranges around an entry that is too low are out, no other."""
    torch = gpu
    rng = np.random.default_rng(14)
    nodes, ctx = rng.integers(1, 7, 70), rng.integers(0, 50, 70)
    p = ref.problem(14, H=8, KV=2, hd=32, page=16, ctx=[int(x) for x in ctx], nodes=[int(x) for x in nodes])
    want = ref.attention(**p)
    rs = p["row_start"].copy()
    for i in falls:
        rs[i] = max(rs[i] - 9, 0)
    for b in range(70):
        if rs[b] < rs[:b + 1].max() or rs[b + 1] < rs[b]:
            want[p["row_start"][b]:p["row_start"][b + 1]] = 0
        else:                                                # the others are as they were
            assert (rs[b], rs[b + 1]) == (p["row_start"][b], p["row_start"][b + 1])
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    junk = torch.full(want.shape, -1, dtype=torch.int64, device="cuda")
    del junk
    got = _attend(torch, exp_t, dict(p, row_start=rs), status, wide).cpu().numpy()
    assert int(status) == 8
    assert np.array_equal(got, want)


# ------------------------------------------------------------------------------------------ verification
@pytest.mark.gpu
@pytest.mark.parametrize("V,tnum", [(1, 1 << 16), (97, 1 << 16), (5000, 81920), (152064, 1 << 16), (300000, 1 << 16),
                                    (400001, 1 << 16), (97, 1 << 32)])
def test_verify_numbers_past_the_range(gpu, exp_t, V, tnum):  # noqa: F811
    """u20 from 2^20 on: the last index, on every path."""
    torch = gpu
    p = _verify_problem(V, V, [6], greedy=0.0, tnum=tnum)
    p["u20"][:] = [1 << 20, 2**31 - 1, (1 << 20) - 1, (1 << 20) + 1, 0, 1 << 30]
    inside = dict(p, u20=np.where(p["u20"] < 1 << 20, p["u20"], 0))
    want = ref.verify(**inside)[0]
    want[p["u20"] >= 1 << 20] = V - 1
    p["tokens"][:] = V                                       # nothing agrees
    junk = [torch.full((n,), -77, dtype=torch.int32, device="cuda") for n in (1, 6, 6, 6, 6)]
    del junk
    sampled, n, path, tok = _verify(torch, exp_t, p)
    assert np.array_equal(sampled, want)
    assert n.tolist() == [1] and path[0, 0] == 0 and tok[0, 0] == V - 1


@pytest.mark.gpu
@pytest.mark.parametrize("V", [262143, 262144, 262145, 327680])
def test_verify_flat_rows(gpu, exp_t, V):  # noqa: F811
    """Equal logits of 2^18 entries and more: sums around 2^42."""
    p = _verify_problem(1, V, [5], greedy=0.0)
    p["logits"][:4] = 12345
    p["u20"][:] = [0, 1, (1 << 20) - 1, 1 << 19, 77]
    assert _same(_verify(gpu, exp_t, p), ref.verify(**p))


# ------------------------------------------------------------------------------------------ the engine's step
@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 300, 5], [0, -1, 5], [0, 4, 3, 5], [0, 5, 2, 5], [0, 2**31 - 1, 5]])
def test_tree_step_row_ranges(cuda_ok, starts):
    """A row_start that falls, or leaves the rows in between, is refused before any node is read or kept: the arrays
    passed hold the last entry's rows and no more."""
    from exact_llm_b200._lib import lib
    from tests.test_tree_decode import SMALL, _model, _prompt
    m = _model(SMALL, max_batch=4, max_seq=400)
    for s in range(3):
        m.forward(_prompt(SMALL, 3), m.new_cache(s))
    B, R = len(starts) - 1, starts[-1]
    arr = [np.ascontiguousarray(x, np.int32) for x in
           (range(B), starts, [1] * R, [-1] + list(range(R - 1)), np.zeros(B), np.zeros(B * 4), np.zeros(B * 4))]
    seqs, rs, ids, par, n, path, tok = [x.ctypes.data_as(ctypes.POINTER(ctypes.c_int32)) for x in arr]
    rc = lib.exb_tree_step(m.h, B, seqs, rs, ids, par, None, 1 << 16, 4, n, path, tok, None, None)
    assert rc == 1 and "row_start must rise" in lib.exb_last_error().decode()
    assert [lib.exb_seq_len(m.h, s) for s in range(3)] == [3, 3, 3]


@pytest.mark.gpu
def test_tree_step_no_length(cuda_ok):
    """A max_len of 0 or less is refused by the engine, not taken for the default."""
    from exact_llm_b200 import ExbError
    from tests.test_tree_decode import SMALL, _model, _prompt
    m = _model(SMALL, max_batch=1, max_seq=40)
    m.forward(_prompt(SMALL, 10), m.new_cache(0))
    for n in (0, -1):
        with pytest.raises(ExbError, match="max_len"):
            m.tree_step([(0, [1, 2], [-1, 0])], max_len=n)


def _check_step(m, p, ids, par, nodes, layers):
    """One step of slot 0 (which holds p) on a tree: the logits of `nodes`, the tokens and the cache are those of plain
    steps along the paths (slot 1, forked from slot 0)."""
    from exact_llm_b200 import Cache
    ((path, toks),), lg = m.tree_step([(0, ids, par)], want_logits=True)

    def way(i):
        out = []
        while i >= 0:
            out.append(ids[i])
            i = par[i]
        return np.array(out[::-1], np.int32)

    for i in nodes:
        c = m.fork(0, 1, len(p))
        assert np.array_equal(m.forward(way(i), c, last_only=True)[-1], lg[i]), i
    assert path[0] == 0 and all(par[b] == a and ids[b] == t for a, b, t in zip(path, path[1:], toks))
    assert toks == [int(np.argmax(lg[i])) for i in path]
    assert not any(par[i] == path[-1] and ids[i] == toks[-1] for i in range(len(ids)))
    m.forward(way(path[-1]), m.fork(0, 1, len(p)))
    for i in range(layers):
        a, b = m.kv_cache(i, Cache(m, 0)), m.kv_cache(i, Cache(m, 1))
        assert a["kq"].shape[1] == len(p) + len(path)
        assert all(np.array_equal(a[n], b[n]) for n in ("kq", "sk", "v"))
    return path


def _tree(rng, V, chain, n):
    """`chain` from the root on, and random nodes around it."""
    ids, par, on = [int(chain[0])], [-1], 0
    for i in range(1, n):
        if i % 3 == 1 and i // 3 + 1 < len(chain):
            ids.append(int(chain[i // 3 + 1]))
            par.append(on)
            on = i
        else:
            ids.append(int(rng.integers(0, V)))
            par.append(int(rng.integers(max(0, i - 70), i)))
    return ids, par


@pytest.mark.gpu
def test_tree_step_long_context(cuda_ok):
    """One layer of the 7B architecture, 4500 tokens in a cache of 8192 and a tree of 70 nodes: the attention's tcgen05
    kernels, and masks of two words."""
    from exact_llm_b200 import configs
    from tests.test_tree_decode import _model, _prompt
    c = configs.arch("qwen2.5-7b", NL=1)
    m = _model(c, max_batch=2, max_seq=8192)
    p = _prompt(c, 4500, 6)
    m.forward(p, m.new_cache(0), want_logits=False)
    first = int(m.last_next[-1])
    cache, chain = m.fork(0, 1), [first]
    for _ in range(5):                                       # what plain steps give
        m.forward(np.array(chain[-1:], np.int32), cache, want_logits=False)
        chain.append(int(m.last_next[-1]))
    ids, par = _tree(np.random.default_rng(6), c["V"], chain, 70)
    assert len(_check_step(m, p, ids, par, [0, 1, 4, 7, 33, 63, 64, 69], 1)) >= 5


@pytest.mark.gpu
@pytest.mark.parametrize("moe,rows", [(False, 512), (True, 256)], ids=["dense", "moe"])
def test_tree_step_most_rows(cuda_ok, moe, rows):
    """As many nodes as a step takes, in one tree and in two; one more is refused."""
    from exact_llm_b200 import ExbError
    from tests.test_tree_decode import MOE, SMALL, _model, _prompt
    c = MOE if moe else SMALL
    rng = np.random.default_rng(rows)
    m = _model(c, max_batch=3, max_seq=900)
    p = _prompt(c, 50, 7)
    m.forward(p, m.new_cache(0))
    chain = [int(m.last_next[-1])]
    cache = m.fork(0, 1)
    for _ in range(9):
        m.forward(np.array(chain[-1:], np.int32), cache)
        chain.append(int(m.last_next[-1]))
    ids, par = _tree(rng, c["V"], chain, rows + 1)
    with pytest.raises(ExbError, match="rows"):
        m.tree_step([(0, ids, par)])
    keep = m.fork(0, 2)
    assert len(_check_step(m, p, ids[:-1], par[:-1], [0, 1, 63, 64, 200, rows - 1], c["NL"])) >= 9
    a, b = rows // 3, rows - rows // 3                       # slots 2 and 1, of the same prompt
    m.fork(2, 0), m.fork(2, 1)
    (one,), lg1 = m.tree_step([(0, ids[:a], par[:a])], want_logits=True)
    both, lg = m.tree_step([(1, ids[:b], par[:b]), (keep, ids[:a], par[:a])], want_logits=True)
    assert both[1] == one and np.array_equal(lg[b:], lg1)
