"""The reference's operator API for the hot path, backed by libexactb200.so.

``torch.ops.exact.gemv(x16, wT, Mg)`` is the operator the reference's engine calls for every
batch-1 group-128 linear (experiments/speed_fair_kaggle.py:698-702, caller TLinG.__call__ at
:737-738):

    x16  int16 (K,)      the quantised activation row
    wT   int8  (N, K)    weights, one contiguous K-byte row per output
    Mg   int64 (N, K/128) group scales
    ->   int64 (N,)      out[n] = sum_g Mg[n, g] * sum_{k in g} x16[k] * wT[n, k]   (exact)

As in the reference, the output is allocated by the op, the kernel runs on the current CUDA
stream, there is no host synchronisation (the op can be captured in a CUDA graph) and the fake
(meta) implementation gives the output shape for tracing.  Unlike the reference, shapes, dtypes,
devices and alignment are checked and a failing launch raises.  Importing this module registers
the ops; it needs torch.

Operators of speculative decoding, without a counterpart in the reference (its engine decodes one
token at a time).  The arithmetic is the exact program's, so a tree gives the bits of one-token steps:

``torch.ops.exact.tree_attention(q, qs, k, ks, v, table, ctx, row_start, mask, exp_t, status=None)``
    attention of drafted trees over a paged cache -> int64 (R, H, hd)
``torch.ops.exact.tree_verify(logits, u20, tokens, parent, row_start, exp_t, tnum, max_len)``
    -> sampled int32 (R), n int32 (B), path int32 (B, max_len), tokens int32 (B, max_len)
``torch.ops.exact.kv_compact_(k, ks, v, table, ctx, path, n, status=None)``
    accepted rows moved next to the sequence's older rows, in place -> new lengths int32 (B)
``torch.ops.exact.kv_copy_pages_(k, ks, v, src, dst, rows, status=None)``
    the first rows[i] positions of page src[i] copied to page dst[i], in place

    q int16 (R, H, hd), qs int32 (R, H)       query rows after RoPE and qrow, their shifts
    k int16 (P, KV, page, hd), ks int8 (P, KV, page), v int32 (P, KV, page, hd)
                                              the cache of one layer; a leading layer dimension for
                                              kv_compact_ and kv_copy_pages_; any strides that keep a
                                              row's hd values together and 16-byte aligned
    table int32 (B, pages)                    page of every ``page`` positions of each sequence
    ctx int32 (B)                             positions cached before the tree; node i is at ctx + i
    row_start int32 (B + 1)                   sequence b's rows are row_start[b] .. row_start[b+1]-1
    mask int64 (R, W)                         the nodes that a row sees: bit i % 64 of word i // 64
                                              (``tree_masks`` makes it from the parents)
    exp_t int32 (10242)                       the Q24 table (``tables.exp_table``)
    logits int64 (R, V), tnum                 rows as the head gives them, round(2^16 / temperature)
    u20 int32 (R)                             the random number of every row, -1 for the argmax
    tokens, parent int32 (R)                  drafted token and parent node (before its child; root -1)
    status int32 (1)                          gets bit 8 or-ed in where an index was out of range; the
                                              entry is left out, never read or written

They run on the current stream of the tensors' device, never synchronise and can be captured.
"""
import torch

from ._lib import KvView, check, lib


def _check_args(x16, wT, Mg):
    if x16.dtype != torch.int16 or wT.dtype != torch.int8 or Mg.dtype != torch.int64:
        raise TypeError("exact::gemv wants x16 int16, wT int8, Mg int64")
    if x16.dim() != 1 or wT.dim() != 2 or Mg.dim() != 2:
        raise ValueError("exact::gemv wants x16 (K,), wT (N, K), Mg (N, K/128)")
    N, K = wT.shape
    if K % 128 or x16.shape[0] != K or tuple(Mg.shape) != (N, K // 128):
        raise ValueError(f"exact::gemv shapes: x16 {tuple(x16.shape)}, wT {tuple(wT.shape)}, Mg {tuple(Mg.shape)}"
                         " (K a multiple of 128)")
    return N, K


@torch.library.custom_op("exact::gemv", mutates_args=())
def gemv(x16: torch.Tensor, wT: torch.Tensor, Mg: torch.Tensor) -> torch.Tensor:
    N, K = _check_args(x16, wT, Mg)
    if not (x16.is_cuda and wT.device == x16.device and Mg.device == x16.device):
        raise ValueError("exact::gemv runs on one CUDA device (all three tensors on it)")
    x16, wT, Mg = x16.contiguous(), wT.contiguous(), Mg.contiguous()
    out = torch.empty((N,), dtype=torch.int64, device=x16.device)
    stream = torch.cuda.current_stream(x16.device).cuda_stream
    with torch.cuda.device(x16.device):
        check(lib.exb_gemv(x16.data_ptr(), wT.data_ptr(), Mg.data_ptr(), K, N, out.data_ptr(), stream))
    return out


@gemv.register_fake
def _gemv_fake(x16, wT, Mg):
    return torch.empty((wT.shape[0],), dtype=torch.int64, device=x16.device)


# ------------------------------------------------------------------------------------------ drafted trees
_lib = torch.library.Library("exact", "FRAGMENT")
_lib.define("tree_attention(Tensor q, Tensor qs, Tensor k, Tensor ks, Tensor v, Tensor table, Tensor ctx, "
            "Tensor row_start, Tensor mask, Tensor exp_t, Tensor(a!)? status=None) -> Tensor")
_lib.define("tree_verify(Tensor logits, Tensor u20, Tensor tokens, Tensor parent, Tensor row_start, Tensor exp_t, "
            "int tnum, int max_len) -> (Tensor, Tensor, Tensor, Tensor)")
_lib.define("kv_compact_(Tensor(a!) k, Tensor(b!) ks, Tensor(c!) v, Tensor table, Tensor ctx, Tensor path, Tensor n, "
            "Tensor(d!)? status=None) -> Tensor")
_lib.define("kv_copy_pages_(Tensor(a!) k, Tensor(b!) ks, Tensor(c!) v, Tensor src, Tensor dst, Tensor rows, "
            "Tensor(d!)? status=None) -> ()")

EXP_LEN = 256 * 40 + 2


def tree_masks(parent, row_start, words=None):
    """Visibility words of drafted trees, on the host: int64 (R, words), a node's own bit and those of
    its ancestors.  ``parent`` (R) holds each row's parent node within its sequence (-1 for a root, else
    a node before it), ``row_start`` (B + 1) the sequences' rows; both are sequences of whole numbers or
    CPU tensors.  ``words`` defaults to what the largest tree needs."""
    parent = [int(p) for p in parent]
    starts = [int(s) for s in row_start]
    if not starts or starts[0] != 0 or starts[-1] != len(parent) or any(a > b for a, b in zip(starts, starts[1:])):
        raise ValueError("tree_masks: row_start must rise from 0 to the number of rows")
    most = max((b - a for a, b in zip(starts, starts[1:])), default=0)
    need = max(1, -(-most // 64))
    words = need if words is None else int(words)
    if words < need:
        raise ValueError(f"tree_masks: {most} nodes need {need} words")
    out = torch.zeros((len(parent), words), dtype=torch.int64)
    for a, b in zip(starts, starts[1:]):
        bits = []
        for i, p in enumerate(parent[a:b]):
            if p >= i or p < -1:
                raise ValueError(f"tree_masks: the parent of node {i} is {p}, not an earlier node")
            bits.append((bits[p] if p >= 0 else 0) | (1 << i))
            for w in range(words):
                x = (bits[i] >> (64 * w)) & (2**64 - 1)
                out[a + i, w] = x - 2**64 if x >> 63 else x
    return out


def _want(name, t, dtype, *shape):
    """dtype, shape (None: any size), contiguity and device class of an argument"""
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, not {t.dtype}")
    if t.dim() != len(shape) or any(w is not None and w != s for w, s in zip(shape, t.shape)):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple('any' if w is None else w for w in shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def _one_device(first, *rest):
    for t in rest:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on {first.device} and {t.device}: exact:: operators run on one CUDA device")


def _view(op, k, ks, v, layered):
    """exb_kv_view of a cache; with ``layered`` a leading layer dimension"""
    if k.dtype != torch.int16 or ks.dtype != torch.int8 or v.dtype != torch.int32:
        raise TypeError(f"{op}: k int16, ks int8, v int32")
    n = 5 if layered else 4
    if k.dim() != n or v.shape != k.shape or ks.shape != k.shape[:-1]:
        raise ValueError(f"{op}: cache shapes k {tuple(k.shape)}, ks {tuple(ks.shape)}, v {tuple(v.shape)}; "
                         f"want {n}-dimensional k and v of one shape and ks without the last dimension")
    if k.stride(-1) != 1 or v.stride(-1) != 1:
        raise ValueError(f"{op}: the values of a cache row must lie together")
    sh = k.shape if layered else (1, *k.shape)
    sk, ss, sv = k.stride()[:-1], ks.stride(), v.stride()[:-1]
    if not layered:
        sk, ss, sv = (0, *sk), (0, *ss), (0, *sv)
    return KvView(k.data_ptr(), ks.data_ptr(), v.data_ptr(), *sh, *sk, *ss, *sv)


def _status(t):
    if t is None:
        return None
    _want("status", t, torch.int32, 1)
    return t.data_ptr()


class _on:
    """The tensors' device made current, and its current stream."""

    def __init__(self, device):
        self.guard = torch.cuda.device(device) if device.index != torch.cuda.current_device() else None
        self.device = device

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return torch.cuda.current_stream(self.device).cuda_stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _check_attention(q, qs, k, table, ctx, row_start, mask, exp_t):
    if q.dtype != torch.int16 or q.dim() != 3 or not q.is_contiguous():
        raise ValueError("exact::tree_attention: q must be contiguous int16 (R, H, hd)")
    R, H, hd = q.shape
    if k.dim() != 4 or k.shape[3] != hd or k.shape[1] < 1 or H % k.shape[1]:
        raise ValueError(f"exact::tree_attention: q {tuple(q.shape)} does not fit the cache {tuple(k.shape)}")
    B = ctx.shape[0] if ctx.dim() == 1 else -1
    _want("qs", qs, torch.int32, R, H)
    _want("ctx", ctx, torch.int32, B)
    _want("table", table, torch.int32, B, None)
    _want("row_start", row_start, torch.int32, B + 1)
    _want("mask", mask, torch.int64, R, None)
    _want("exp_t", exp_t, torch.int32, EXP_LEN)
    return R, H, hd, B


def _tree_attention(q, qs, k, ks, v, table, ctx, row_start, mask, exp_t, status=None):
    R, H, hd, B = _check_attention(q, qs, k, table, ctx, row_start, mask, exp_t)
    kv = _view("exact::tree_attention", k, ks, v, False)
    _one_device(q, qs, k, ks, v, table, ctx, row_start, mask, exp_t, status)
    st = _status(status)
    out = torch.empty((R, H, hd), dtype=torch.int64, device=q.device)
    if R == 0:
        return out
    nb = lib.exb_tree_attention_workspace_bytes(R, H, B)
    ws = torch.empty(nb, dtype=torch.uint8, device=q.device)
    with _on(q.device) as stream:
        check(lib.exb_tree_attention(kv, q.data_ptr(), qs.data_ptr(), R, H, table.data_ptr(), B, table.shape[1],
                                     ctx.data_ptr(), row_start.data_ptr(), mask.data_ptr(), mask.shape[1],
                                     exp_t.data_ptr(), out.data_ptr(), ws.data_ptr(), nb, st, stream))
    return out


def _check_verify(logits, u20, tokens, parent, row_start, exp_t, tnum, max_len):
    if logits.dtype != torch.int64 or logits.dim() != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("exact::tree_verify: logits must be int64 (R, V) with rows in one piece")
    R, V = logits.shape
    if V < 1 or max_len < 1:
        raise ValueError("exact::tree_verify: V >= 1 and max_len >= 1")
    if row_start.dim() != 1 or row_start.shape[0] < 1:
        raise ValueError("exact::tree_verify: row_start (B + 1)")
    for name, t in (("u20", u20), ("tokens", tokens), ("parent", parent)):
        _want(name, t, torch.int32, R)
    _want("row_start", row_start, torch.int32, None)
    _want("exp_t", exp_t, torch.int32, EXP_LEN)
    return R, V, row_start.shape[0] - 1


def _verify_outputs(R, B, max_len, device):
    i32 = dict(dtype=torch.int32, device=device)
    return (torch.empty(R, **i32), torch.empty(B, **i32), torch.empty((B, max_len), **i32),
            torch.empty((B, max_len), **i32))


def _tree_verify(logits, u20, tokens, parent, row_start, exp_t, tnum, max_len):
    R, V, B = _check_verify(logits, u20, tokens, parent, row_start, exp_t, tnum, max_len)
    _one_device(logits, u20, tokens, parent, row_start, exp_t)
    sampled, n, path, out = _verify_outputs(R, B, max_len, logits.device)
    with _on(logits.device) as stream:
        check(lib.exb_tree_verify(logits.data_ptr(), logits.stride(0) if R > 1 else V, R, V, u20.data_ptr(), tnum,
                                  tokens.data_ptr(), parent.data_ptr(), row_start.data_ptr(), B, max_len,
                                  exp_t.data_ptr(), sampled.data_ptr(), n.data_ptr(), path.data_ptr(), out.data_ptr(),
                                  stream))
    return sampled, n, path, out


def _check_compact(k, table, ctx, path, n):
    B = ctx.shape[0] if ctx.dim() == 1 else -1
    _want("ctx", ctx, torch.int32, B)
    _want("table", table, torch.int32, B, None)
    _want("path", path, torch.int32, B, None)
    _want("n", n, torch.int32, B)
    return B


def _kv_compact(k, ks, v, table, ctx, path, n, status=None):
    B = _check_compact(k, table, ctx, path, n)
    kv = _view("exact::kv_compact_", k, ks, v, True)
    _one_device(k, ks, v, table, ctx, path, n, status)
    st = _status(status)
    new = torch.empty(B, dtype=torch.int32, device=k.device)
    if B:
        with _on(k.device) as stream:
            check(lib.exb_kv_compact(kv, table.data_ptr(), B, table.shape[1], ctx.data_ptr(), path.data_ptr(),
                                     path.shape[1], n.data_ptr(), new.data_ptr(), st, stream))
    return new


def _kv_copy_pages(k, ks, v, src, dst, rows, status=None):
    kv = _view("exact::kv_copy_pages_", k, ks, v, True)
    _want("src", src, torch.int32, None)
    count = src.shape[0]
    _want("dst", dst, torch.int32, count)
    _want("rows", rows, torch.int32, count)
    _one_device(k, ks, v, src, dst, rows, status)
    st = _status(status)
    if count:
        with _on(k.device) as stream:
            check(lib.exb_kv_copy_pages(kv, src.data_ptr(), dst.data_ptr(), rows.data_ptr(), count, st, stream))


_lib.impl("tree_attention", _tree_attention, "CUDA")
_lib.impl("tree_verify", _tree_verify, "CUDA")
_lib.impl("kv_compact_", _kv_compact, "CUDA")
_lib.impl("kv_copy_pages_", _kv_copy_pages, "CUDA")


@torch.library.register_fake("exact::tree_attention")
def _tree_attention_fake(q, qs, k, ks, v, table, ctx, row_start, mask, exp_t, status=None):
    _check_attention(q, qs, k, table, ctx, row_start, mask, exp_t)
    return torch.empty(q.shape, dtype=torch.int64, device=q.device)


@torch.library.register_fake("exact::tree_verify")
def _tree_verify_fake(logits, u20, tokens, parent, row_start, exp_t, tnum, max_len):
    R, _, B = _check_verify(logits, u20, tokens, parent, row_start, exp_t, tnum, max_len)
    return _verify_outputs(R, B, max_len, logits.device)


@torch.library.register_fake("exact::kv_compact_")
def _kv_compact_fake(k, ks, v, table, ctx, path, n, status=None):
    return torch.empty(_check_compact(k, table, ctx, path, n), dtype=torch.int32, device=k.device)


@torch.library.register_fake("exact::kv_copy_pages_")
def _kv_copy_pages_fake(k, ks, v, src, dst, rows, status=None):
    return None
