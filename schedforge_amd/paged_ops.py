"""What a paged KV cache keeps and reads, over PagedKVCache's device pools:

  speculative decoding   append_drafts, tree_mask, tree_attention, accept_drafts
  eviction by weight     attention_weights, weighted_decode_attention, evict_paged_kv
  sparse attention       page_bounds, refresh_page_bounds, sparse_decode_attention

The reference has no counterparts: its caches grow at the end and are read whole.
Tensors stay on the device and no call waits for it; each runs on `stream`, or the
current one, and the caller orders calls on different streams.  Arguments live on the
cache's device and are contiguous; a `workspace` (uint8, as large as the *_workspace query
of the C ABI says) may be passed to calls that are captured or repeated, else it is
allocated.

Calls can be captured, except where pages change hands (append_drafts into pages that are
not reserved yet, evict_paged_kv): the tables are uploaded there, and a replay would upload
them again as they are not any more.  A replay leaves the host's side alone: cache.length,
the bound on all lengths, is what it was when the call was captured.

Sequences may have lengths of their own: `seq_lens` (int32 [B] on the device), none above
cache.length.  Without it every sequence holds cache.length tokens.

Keys and queries come rotated (RoPE): drafts at their sequence's length plus their depth in
the tree.  Tokens that move keep their rotation, so after an eviction a token's position is
the caller's count, not its place in the cache.

The pools of a compiled layer (DecoderExecutablePlan.t) are no PagedKVCache: its callers use
the C ABI.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import numpy as np
import torch

from . import _abi
from ._abi import BF16, F32, check
from .kvcache import PagedKVCache

_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}


@contextlib.contextmanager
def _on(cache: PagedKVCache, stream: Optional[torch.cuda.Stream]):
    """The cache's device and the call's stream, so that what a call allocates is that stream's."""
    if stream is not None and (not isinstance(stream, torch.cuda.Stream) or stream.device != cache.device):
        raise ValueError(f"stream must be a torch.cuda.Stream of {cache.device}")
    with torch.cuda.device(cache.device):
        s = stream if stream is not None else torch.cuda.current_stream()
        with torch.cuda.stream(s):
            yield s.cuda_stream


def _tensor(cache: PagedKVCache, t, name: str, dtypes, shape) -> torch.Tensor:
    dtypes = dtypes if isinstance(dtypes, tuple) else (dtypes,)
    if not isinstance(t, torch.Tensor) or t.dtype not in dtypes:
        raise ValueError(f"{name} must be a tensor of {' or '.join(str(d) for d in dtypes)}")
    if t.device != cache.device:
        raise ValueError(f"{name} must be on {cache.device}")
    if tuple(t.shape) != tuple(shape) or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous of shape {tuple(shape)}; got {tuple(t.shape)}")
    return t


def _lens(cache: PagedKVCache, seq_lens) -> Optional[int]:
    return None if seq_lens is None else _tensor(cache, seq_lens, "seq_lens", torch.int32, (cache.config.batch,)).data_ptr()


def _args(cache: PagedKVCache, query, out, seq_lens, kv_splits: int, scale: float):
    """The argument block, and the output (made like the query if not given)."""
    c = cache.config
    if not isinstance(query, torch.Tensor) or query.dim() != 4:
        raise ValueError("query must be a tensor [batch][q_heads][rows][head_dim]")
    hq, rows = int(query.shape[1]), int(query.shape[2])
    if hq <= 0 or hq % c.kv_heads:
        raise ValueError("invalid attention configuration")
    _tensor(cache, query, "query", tuple(_DTYPES), (c.batch, hq, rows, c.head_dim))
    out = torch.empty_like(query) if out is None else _tensor(cache, out, "out", tuple(_DTYPES), query.shape)
    a = _abi.PagedAttnArgs()
    a.q, a.q_dtype = query.data_ptr(), _DTYPES[query.dtype]
    a.k_pool, a.v_pool, a.kv_dtype = cache.k_pool.data_ptr(), cache.v_pool.data_ptr(), cache.pool_dtype
    a.page_table, a.seq_lens = cache.table.data_ptr(), _lens(cache, seq_lens)
    a.out, a.out_dtype = out.data_ptr(), _DTYPES[out.dtype]
    a.batch, a.q_heads, a.kv_heads, a.rows, a.head_dim = c.batch, hq, c.kv_heads, rows, c.head_dim
    a.page_tokens, a.pages_per_seq, a.num_pages = c.page_tokens, c.pages_per_seq, c.num_pages
    a.max_context, a.kv_splits, a.scale = cache.length, kv_splits, scale
    return a, out


def _workspace(cache: PagedKVCache, workspace, size: int) -> torch.Tensor:
    if workspace is None:
        return torch.empty(max(size, 1), dtype=torch.uint8, device=cache.device)
    return _tensor(cache, workspace, "workspace", torch.uint8, workspace.shape if isinstance(workspace, torch.Tensor) else ())


def _uncaptured(what: str) -> None:
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} changes the page tables and cannot be captured")


# ---------------------------------------------------------------- speculative decoding
def tree_mask(parents, device="cuda") -> torch.Tensor:
    """Ancestor-or-self bits of drafted trees, int32 words [B][T][ceil(T / 32)] as tree_attention
    takes them.  parents: int [B][T] on the host, parents[b][t] < t, -1 for a child of the last
    committed token."""
    p = np.asarray(parents)
    if p.ndim != 2 or p.shape[1] == 0 or (p < -1).any() or (p >= np.arange(p.shape[1])[None]).any():
        raise ValueError("parents: [batch][nodes] of earlier nodes, or -1")
    b, t = p.shape
    seen = np.zeros((b, t, -(-t // 32) * 32), bool)
    rows = np.arange(b)
    for n in range(t):
        seen[:, n] = np.where(p[:, n, None] >= 0, seen[rows, np.maximum(p[:, n], 0)], False)
        seen[:, n, n] = True
    words = np.packbits(seen, axis=-1, bitorder="little").view("<i4")
    return torch.from_numpy(np.ascontiguousarray(words)).to(device)


def append_drafts(cache: PagedKVCache, keys: torch.Tensor, values: torch.Tensor, seq_lens=None,
                  stream: Optional[torch.cuda.Stream] = None) -> None:
    """K / V of drafted tokens [B][Hkv][T][D] (fp32 or bf16) written behind each sequence's committed
    tokens.  The pages are reserved; cache.length and seq_lens stay (accept_drafts moves them on)."""
    c = cache.config
    if not isinstance(keys, torch.Tensor) or keys.dim() != 4 or keys.shape[2] == 0:
        raise ValueError("drafted keys must be a tensor [batch][kv_heads][tokens][head_dim]")
    t = int(keys.shape[2])
    for name, x in (("keys", keys), ("values", values)):
        _tensor(cache, x, name, keys.dtype if keys.dtype in _DTYPES else tuple(_DTYPES), (c.batch, c.kv_heads, t, c.head_dim))
    lens = _lens(cache, seq_lens)
    with _on(cache, stream) as s:
        grows = any(len(p) * c.page_tokens < cache.length + t for p in cache.page_table)
        if grows:
            _uncaptured("appending into new pages")
        cache.alloc.reserve(t)
        if grows:
            cache._sync_table(wait=False)
        dt = _DTYPES[keys.dtype]
        check(cache.lib.sfg_hip_kv_append_pool_v1(
            keys.data_ptr(), values.data_ptr(), dt, cache.k_pool.data_ptr(), cache.v_pool.data_ptr(), cache.pool_dtype,
            cache.table.data_ptr(), lens, cache.length, 0, c.batch, c.kv_heads, t, c.head_dim, c.page_tokens,
            c.pages_per_seq, c.num_pages, s))


def tree_attention(cache: PagedKVCache, query: torch.Tensor, mask: torch.Tensor, seq_lens=None, out=None,
                   scale: float = 0.0, kv_splits: int = 0, workspace=None,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Attention of drafted tokens (append_drafts) over the committed ones and each other: query
    [B][Hq][T][D]; row t sees draft u iff its bit in mask ([B or 1][T][ceil(T / 32)] int32, tree_mask) is set."""
    with _on(cache, stream) as s:
        a, out = _args(cache, query, out, seq_lens, kv_splits, scale)
        b, w = cache.config.batch, -(-a.rows // 32)
        shared = isinstance(mask, torch.Tensor) and mask.dim() == 3 and mask.shape[0] == 1
        _tensor(cache, mask, "mask", torch.int32, (1 if shared else b, a.rows, w))
        ws = _workspace(cache, workspace, cache.lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(a)))
        check(cache.lib.sfg_hip_attn_tree_v1(ctypes.byref(a), mask.data_ptr(), 0 if shared else a.rows * w, ws.data_ptr(),
                                             ws.numel(), s))
    return out


def accept_drafts(cache: PagedKVCache, path: torch.Tensor, counts: torch.Tensor, seq_lens: torch.Tensor,
                  longest: Optional[int] = None, stream: Optional[torch.cuda.Stream] = None) -> None:
    """Keeps the accepted drafts: draft path[b][i] (int32 [B][n], ascending) becomes the i-th token behind
    sequence b's committed ones for i < counts[b], and seq_lens grows by counts.  longest: the most that any
    sequence accepts, if the host knows it (default: n); counts beyond it are cut to it, and cache.length, the
    bound on all lengths, grows by it."""
    c = cache.config
    if not isinstance(path, torch.Tensor) or path.dim() != 2 or path.shape[1] == 0:
        raise ValueError("path must be a tensor [batch][nodes]")
    n = int(path.shape[1])
    longest = n if longest is None else longest
    if longest < 0 or longest > n or cache.length + longest > c.capacity:
        raise ValueError("paged KV capacity exceeded")
    _tensor(cache, path, "path", torch.int32, (c.batch, n))
    _tensor(cache, counts, "counts", torch.int32, (c.batch,))
    lens = _lens(cache, seq_lens)
    if lens is None:
        raise ValueError("accept_drafts needs the sequences' lengths")
    if longest == 0:
        return
    with _on(cache, stream) as s:
        check(cache.lib.sfg_hip_kv_compact_v1(
            cache.k_pool.data_ptr(), cache.v_pool.data_ptr(), cache.pool_dtype, cache.table.data_ptr(), lens,
            path.data_ptr(), 1, n, counts.data_ptr(), lens, longest, c.batch, c.kv_heads, c.head_dim, c.page_tokens,
            c.pages_per_seq, c.num_pages, s))
    cache.alloc.length += longest


# ---------------------------------------------------------------- eviction by accumulated weight
def attention_weights(cache: PagedKVCache) -> torch.Tensor:
    """Accumulators of the cache's tokens, fp32 [B][Hkv][pages_per_seq * page_tokens], zero.  Entries behind the
    cached tokens have to be zero: evict_paged_kv leaves them so, after truncate_paged_kv the caller clears them."""
    c = cache.config
    return torch.zeros((c.batch, c.kv_heads, c.pages_per_seq * c.page_tokens), dtype=torch.float32, device=cache.device)


def _weights(cache: PagedKVCache, weights) -> torch.Tensor:
    c = cache.config
    return _tensor(cache, weights, "weights", torch.float32, (c.batch, c.kv_heads, c.pages_per_seq * c.page_tokens))


def weighted_decode_attention(cache: PagedKVCache, query: torch.Tensor, weights: torch.Tensor, seq_lens=None, out=None,
                              scale: float = 0.0, kv_splits: int = 0, workspace=None,
                              stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Causal attention of the newest tokens (query [B][Hq][rows][D]) that adds to `weights`
    (attention_weights) what each cached token drew, summed over the rows and the heads of its kv head."""
    _weights(cache, weights)
    with _on(cache, stream) as s:
        a, out = _args(cache, query, out, seq_lens, kv_splits, scale)
        ws = _workspace(cache, workspace, cache.lib.sfg_hip_attn_weights_workspace_v1(ctypes.byref(a)))
        check(cache.lib.sfg_hip_attn_weights_v1(ctypes.byref(a), weights.data_ptr(), weights.shape[2], ws.data_ptr(),
                                                ws.numel(), s))
    return out


def evict_paged_kv(cache: PagedKVCache, weights: torch.Tensor, budget: int, recent: int, seq_lens=None,
                   stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Cuts every sequence back to `budget` tokens: the newest `recent` and, per kv head, the others of the
    largest weight (ties to the older).  K, V and weights are compacted in place, seq_lens (if given) and
    cache.length shrink, the pages behind return to the free list.  Returns the kept positions, int32
    [B][Hkv][budget], -1 behind."""
    c = cache.config
    _weights(cache, weights)
    if cache.length <= 0:
        raise ValueError("cannot evict from an empty paged KV cache")
    if budget <= 0 or recent < 0 or recent > budget:
        raise ValueError("invalid eviction budget")
    lens = _lens(cache, seq_lens)
    with _on(cache, stream) as s:
        if budget < cache.length:
            _uncaptured("eviction")
        keep = torch.empty((c.batch, c.kv_heads, budget), dtype=torch.int32, device=cache.device)
        counts = torch.empty(c.batch, dtype=torch.int32, device=cache.device)
        check(cache.lib.sfg_hip_kv_select_v1(weights.data_ptr(), weights.shape[2], lens, cache.length, budget, recent,
                                             keep.data_ptr(), counts.data_ptr(), weights.data_ptr(), c.batch, c.kv_heads, s))
        if budget < cache.length:
            check(cache.lib.sfg_hip_kv_compact_v1(
                cache.k_pool.data_ptr(), cache.v_pool.data_ptr(), cache.pool_dtype, cache.table.data_ptr(), None,
                keep.data_ptr(), c.kv_heads, budget, counts.data_ptr(), counts.data_ptr() if lens is None else lens, budget,
                c.batch, c.kv_heads, c.head_dim, c.page_tokens, c.pages_per_seq, c.num_pages, s))
            cache.alloc.truncate(budget)
            cache._sync_table(wait=False)
    return keep


# ---------------------------------------------------------------- sparse attention
def page_bounds(cache: PagedKVCache) -> torch.Tensor:
    """Room for the pages' key bounds, [num_pages][Hkv][2][D] in the pool's type (bf16 or fp32), zero."""
    c = cache.config
    return torch.zeros((c.num_pages, c.kv_heads, 2, c.head_dim), device=cache.device,
                       dtype=torch.float32 if cache.pool_dtype == F32 else torch.bfloat16)


def _bounds(cache: PagedKVCache, bounds) -> torch.Tensor:
    c = cache.config
    return _tensor(cache, bounds, "bounds", torch.float32 if cache.pool_dtype == F32 else torch.bfloat16,
                   (c.num_pages, c.kv_heads, 2, c.head_dim))


def refresh_page_bounds(cache: PagedKVCache, bounds: torch.Tensor, fresh: Optional[int] = None, seq_lens=None,
                        stream: Optional[torch.cuda.Stream] = None) -> None:
    """The bounds of the pages that hold the newest `fresh` tokens (default: all): after every append with
    its tokens, after truncation, acceptance or eviction with all."""
    c = cache.config
    _bounds(cache, bounds)
    if cache.length <= 0:
        raise ValueError("cannot bound the pages of an empty paged KV cache")
    lens = _lens(cache, seq_lens)
    with _on(cache, stream) as s:
        check(cache.lib.sfg_hip_kv_page_bounds_v1(
            cache.k_pool.data_ptr(), cache.pool_dtype, cache.table.data_ptr(), lens, cache.length,
            cache.length if fresh is None else fresh, bounds.data_ptr(), c.batch, c.kv_heads, c.head_dim, c.page_tokens,
            c.pages_per_seq, c.num_pages, s))


def sparse_decode_attention(cache: PagedKVCache, query: torch.Tensor, bounds: torch.Tensor, top_pages: int,
                            sink_pages: int = 1, recent_pages: int = 1, seq_lens=None, out=None, selected=None,
                            scale: float = 0.0, kv_splits: int = 0, workspace=None,
                            stream: Optional[torch.cuda.Stream] = None):
    """Causal attention of the newest tokens (query [B][Hq][rows][D]) over at most top_pages pages per row
    and kv head: the first sink_pages, the newest recent_pages and the others of the highest score by
    `bounds` (refresh_page_bounds).  Returns (out, selected): selected int32 [B][rows][Hkv][top_pages]
    holds the logical pages ascending, -1 behind."""
    c = cache.config
    _bounds(cache, bounds)
    if top_pages <= 0:
        raise ValueError("sparse attention reads at least one page")
    with _on(cache, stream) as s:
        a, out = _args(cache, query, out, seq_lens, kv_splits, scale)
        shape = (c.batch, a.rows, c.kv_heads, top_pages)
        selected = torch.empty(shape, dtype=torch.int32, device=cache.device) if selected is None else selected
        _tensor(cache, selected, "selected", torch.int32, shape)
        ws = _workspace(cache, workspace, cache.lib.sfg_hip_attn_sparse_workspace_v1(ctypes.byref(a), top_pages))
        check(cache.lib.sfg_hip_attn_sparse_v1(ctypes.byref(a), bounds.data_ptr(), top_pages, sink_pages, recent_pages,
                                               selected.data_ptr(), ws.data_ptr(), ws.numel(), s))
    return out, selected
