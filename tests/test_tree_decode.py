"""Decoding by drafted trees equals one-token decoding, bit for bit: tokens, logits, cache."""
import numpy as np
import pytest

SMALL = dict(D=256, H=4, KV=2, hd=64, I=512, V=1024, NL=2, theta=1e6, tie=True, lin="group")
MOE = dict(D=256, H=4, KV=4, hd=64, I=128, V=1024, NL=2, theta=1e6, tie=False, lin="channel", NE=8, TOPK=2, MI=128,
           SI=256)


def test_ngram_tree():
    from exact_llm_b200 import drafting
    t = [1, 2, 3, 4, 9, 1, 2, 3, 5, 8, 1, 2, 3]
    ids, par = drafting.ngram_tree(t, nodes=6, depth=3)
    assert ids[0] == 5 and par[0] == -1                      # the latest continuation first
    assert all(p < i for i, p in enumerate(par)) and len(ids) == 6
    assert (4, -1) in list(zip(ids, par))                    # the earlier one beside it
    assert drafting.ngram_tree([7]) == ([], [])
    assert drafting.ngram_tree([1, 2, 3]) == ([], [])


def test_sampler_numbers():
    from exact_llm_b200 import drafting
    from oracle import exact_oracle as eo
    assert [drafting.u20(5, i) for i in range(50)] == [eo.u20(5, i) for i in range(50)]


def _model(c, **kw):
    from exact_llm_b200 import ExactModel
    return ExactModel.synthetic(c, 31, **kw)


def _prompt(c, n, seed=0):
    rng = np.random.default_rng(seed)
    return np.tile(rng.integers(0, c["V"], max(3, n // 3)), 4)[:n].astype(np.int32)


def _true_draft(tokens, wrong):
    """a draft that knows the answer: a chain of it, with wrong branches in between"""
    def draft(hist):
        at = len(hist)
        ids, par, last = [], [], -1
        for i, t in enumerate(tokens[at:at + 5]):
            if (at + i) % wrong == 0:
                ids.append((t + 1) % 1000)                   # a wrong sibling first
                par.append(last)
            ids.append(t)
            par.append(last)
            last = len(ids) - 1
        return ids, par
    return draft


@pytest.mark.gpu
@pytest.mark.parametrize("c", [SMALL, MOE, dict(SMALL, hd=32, H=8, KV=2)], ids=["dense", "moe", "hd32"])
def test_tree_decoding_is_decoding(cuda_ok, c):
    n, p = 24, _prompt(c, 40)
    m = _model(c, max_batch=2, max_seq=96)
    lg, rows, want = m.greedy(p, n)
    kv = [m.kv_cache(i) for i in range(c["NL"])]
    full = p.tolist() + want
    for draft in (None, lambda hist: ([], []), _true_draft(full, 2), _true_draft(full, 3)):
        got, steps = m.generate_drafted(p, n, draft, slot=1)
        assert got[:n] == want
        # the last token is not in the cache yet, on neither side
        cache = [m.kv_cache(i, m_cache(m, 1)) for i in range(c["NL"])]
        k = min(len(p) + n - 1, cache[0]["kq"].shape[1])
        assert k >= len(p) + n - 1
        for a, b in zip(kv, cache):
            for name in ("kq", "sk", "v"):
                assert np.array_equal(a[name][:, :k], b[name][:, :k]), name
    assert m.generate_drafted(p, n, _true_draft(full, 100), slot=1)[1] <= -(-(n - 1) // 5)


def m_cache(m, slot):
    from exact_llm_b200 import Cache
    return Cache(m, slot)


@pytest.mark.gpu
def test_tree_decoding_sampled(cuda_ok):
    c = SMALL
    n, p = 20, _prompt(c, 30, 1)
    m = _model(c, max_batch=1, max_seq=80)
    receipt, _ = m.generate_sampled(p, n, 77, 0.8)
    full = p.tolist() + receipt["tokens"]
    for draft in (None, _true_draft(full, 3)):
        got, _ = m.generate_drafted(p, n, draft, seed=77, temp=0.8)
        assert got == receipt["tokens"]
    assert m.verify_receipt(receipt) == (True, None)


@pytest.mark.gpu
def test_tree_step_logits_and_batch(cuda_ok):
    """Trees of several sequences in one step: every node's logits are those of its path as a plain
    continuation; forked slots go on from a shared prompt."""
    c = SMALL
    rng = np.random.default_rng(5)
    m = _model(c, max_batch=4, max_seq=200)
    p = _prompt(c, 33, 2)
    m.forward(p, m.new_cache(0))
    m.fork(0, 1)
    m.fork(0, 2, 20)
    lens = [33, 33, 20]
    trees = []
    for s, T in zip(range(3), (70, 1, 9)):
        par = [-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, T)]
        trees.append((s, rng.integers(0, c["V"], T).tolist(), par))
    res, lg = m.tree_step(trees, want_logits=True)
    kv = [[m.kv_cache(i, m_cache(m, s)) for i in range(c["NL"])] for s in range(3)]
    assert [m_cache(m, s).n for s in range(3)] == [n + len(r[0]) for n, r in zip(lens, res)]
    r = 0
    for s, (_, ids, par) in enumerate(trees):
        for i in range(len(ids)):
            way, j = [], i
            while j >= 0:
                way.append(ids[j])
                j = par[j]
            if i < 12 or i % 9 == 0:
                want = m(np.array(p[:lens[s]].tolist() + way[::-1], np.int32))[-1]         # slot 0, anew
                assert np.array_equal(lg[r], want), (s, i)
            r += 1
        nodes, toks = res[s]
        assert nodes[0] == 0 and toks[-1] == int(np.argmax(lg[r - len(ids) + nodes[-1]]))
        for a, b, t in zip(nodes, nodes[1:], toks):
            assert par[b] == a and ids[b] == t
        m(np.array(p[:lens[s]].tolist() + [ids[j] for j in nodes], np.int32))
        for i in range(c["NL"]):
            again = m.kv_cache(i)
            for name in ("kq", "sk", "v"):
                assert np.array_equal(kv[s][i][name], again[name])


@pytest.mark.gpu
def test_tree_step_at_model_size(cuda_ok):
    """One layer of the 7B architecture, a tree of 40 behind 300 tokens."""
    from exact_llm_b200 import configs
    c = configs.arch("qwen2.5-7b", NL=1)
    m = _model(c, max_batch=1, max_seq=400)
    p = _prompt(c, 300, 3)
    n = 12
    lg, rows, want = m.greedy(p, n)
    got, steps = m.generate_drafted(p, n, _true_draft(p.tolist() + want, 2))
    assert got[:n] == want and steps < n - 1


@pytest.mark.gpu
def test_tree_step_refusals(cuda_ok):
    from exact_llm_b200 import ExbError
    m = _model(SMALL, max_batch=2, max_seq=40)
    m.forward(_prompt(SMALL, 30), m.new_cache(0))
    ok = [1, 2, 3], [-1, 0, 0]
    for trees, kw in [([(0, [1, 2], [-1, 1])], {}), ([(0, [1], [0])], {}), ([(0, [1024], [-1])], {}), ([(2, *ok)], {}),
                      ([(0, *ok), (0, *ok)], {}), ([(0, [1] * 11, [-1] + [0] * 10)], {}), ([(0, *ok)], dict(u20=[0, 1 << 20, 0])),
                      ([(0, *ok)], dict(tnum=0)), ([(0, *ok)], dict(max_len=600)), ([(0, *ok), (1, [], [])], {})]:
        with pytest.raises(ExbError):
            m.tree_step(trees, **kw)
    assert m_cache(m, 0).n == 30
    for a in ((0, 0), (0, 2), (0, 1, 31), (-1, 1)):
        with pytest.raises(ExbError):
            m.fork(*a)
    with pytest.raises(ValueError):
        m.tree_step([(0, [1, 2], [-1])])
    m.trace_enable(True)
    with pytest.raises(ExbError, match="tensor-core path"):
        m.tree_step([(0, *ok)])
