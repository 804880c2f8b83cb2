"""Drafts for tree decoding, on the host: token trees from the text itself, and the sampler's numbers."""

_M64 = (1 << 64) - 1


def u20(seed, pos):
    """The sampler's random number for output position ``pos``, in [0, 2^20) (exact_llm.py:243-248)."""
    z = (seed + (pos + 1) * 0x9E3779B97F4A7C15) & _M64
    z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & _M64
    z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & _M64
    return (z ^ (z >> 31)) >> 44


def ngram_tree(tokens, nodes=16, depth=6, most=3):
    """What followed earlier occurrences of the last ``most`` .. 1 tokens, merged into one tree:
    (ids, parents), parent -1 for the nodes right after the last token, else an earlier node.  Longer
    matches and later occurrences come first; at most ``nodes`` nodes, ``depth`` tokens deep."""
    ids, par, child = [], [], {}
    n = len(tokens)
    for k in range(min(most, n - 1), 0, -1):
        last = tokens[n - k:]
        for at in range(n - k - 1, -1, -1):
            if tokens[at:at + k] != last:
                continue
            node = -1
            for t in tokens[at + k:at + k + depth]:
                nxt = child.get((node, t))
                if nxt is None:
                    if len(ids) == nodes:
                        break
                    nxt = child[node, t] = len(ids)
                    ids.append(t)
                    par.append(node)
                node = nxt
            if len(ids) == nodes:
                return ids, par
    return ids, par
