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
    u20 int32 (R)                             the random number of every row, below 2^20 (from there on the
                                              row's token is V - 1); -1 for the argmax
    tokens, parent int32 (R)                  drafted token and parent node (before its child; root -1)
    status int32 (1)                          gets bit 8 or-ed in where an index was out of range; the
                                              entry is left out, never read or written

They run on the current stream of the tensors' device, never synchronise and can be captured.  They are in
libexactb200_torch.so; where it was not built, or for another torch, each of them raises ImportError when called.
"""
import ctypes
import os

import torch

from ._lib import HERE, check, lib

TORCH_OPS_PATH = os.path.join(HERE, "libexactb200_torch.so")


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
# Schemas, checks and calls are in torch_ops.cpp, which gets the entry points of the library loaded by _lib.
_ENTRIES = ("exb_last_error", "exb_tree_attention_workspace_bytes", "exb_tree_attention", "exb_tree_verify",
            "exb_kv_compact", "exb_kv_copy_pages")
_TREE_OPS = ("tree_attention", "tree_verify", "kv_compact_", "kv_copy_pages_")


def _missing(name, why):
    def op(*args, **kwargs):
        raise ImportError(f"torch.ops.exact.{name}: {why}; build it with `python exact_llm_b200/build.py`")
    return op


def _load_tree_ops(path):
    """Register the operators of ``path``.  Without it ``exact::gemv`` is all there is, and the others raise when called."""
    why = f"{path} is missing"
    if os.path.exists(path):
        try:
            torch.ops.load_library(path)
            bind = ctypes.CDLL(path).exb_torch_bind
            bind((ctypes.c_void_p * len(_ENTRIES))(*(ctypes.cast(getattr(lib, n), ctypes.c_void_p) for n in _ENTRIES)))
            return
        except (OSError, AttributeError) as e:               # of another torch, or older than this module
            why = f"{path} does not load ({e})"
    for name in _TREE_OPS:
        setattr(torch.ops.exact, name, _missing(name, why))


_load_tree_ops(TORCH_OPS_PATH)


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
