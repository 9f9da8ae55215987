"""A paged KV cache held in 8 bits, and a serving step over it with nothing on the host:

  plan_step             pages given back and taken, slots and positions of the new tokens
  rotate                rotary positions of queries and keys (RotaryAngles: scaled contexts)
  append_quantized_kv   keys and values into the cache, one scale for each page, kv head and pool
  quantized_attention   causal attention of each sequence's newest rows over the cache

The reference has no counterparts: its caches hold fp32 and its page allocator is the host's
(kvcache.py).  Here the page tables, the free list and the lengths live on the device, so a step
whose sequences grow by other counts each time is captured once and replayed: counts (and keep)
are tensors that the caller writes between replays.

A step's tokens are packed: rows starts[b] .. starts[b + 1] are sequence b's, oldest first; rows
behind starts[batch] are padding, with position and slot -1, and are left as they were.

Tensors stay on the device and no call waits for it; each runs on `stream`, or the current one,
and the caller orders calls on different streams.  A `workspace` (uint8, as large as
attention_workspace says) may be passed to calls that are captured or repeated, else it is
allocated; calls that overlap need workspaces of their own.

Nothing here computes gradients: rows that require them are refused while autograd records.
"""
from __future__ import annotations

import ctypes
import dataclasses
from typing import Optional

import numpy as np
import torch

from . import _abi
from ._abi import BF16, F32, FP8, I8, check
from .paged_ops import _on, _tensor, _workspace

_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}
_POOLS = {"int8": (I8, torch.int8), "fp8": (FP8, torch.float8_e4m3fn)}
_SCALINGS = {"plain": _abi.ROPE_PLAIN, "linear": _abi.ROPE_LINEAR, "base": _abi.ROPE_BASE, "bands": _abi.ROPE_BANDS,
             "ramp": _abi.ROPE_RAMP}
_LAYOUTS = {"half": _abi.ROPE_HALF, "interleaved": _abi.ROPE_INTERLEAVED}


@dataclasses.dataclass
class QuantizedKVConfig:
    batch: int = 1
    kv_heads: int = 1
    head_dim: int = 1
    page_tokens: int = 16
    capacity: int = 0                  # tokens of the longest sequence
    num_pages: Optional[int] = None    # pages shared by all sequences (default: capacity for each)
    pool_dtype: str = "int8"           # or "fp8" (e4m3)

    def validate(self) -> None:
        if (self.batch <= 0 or self.kv_heads <= 0 or self.head_dim <= 0 or self.page_tokens <= 0 or self.capacity <= 0
                or (self.num_pages is not None and self.num_pages <= 0)):
            raise ValueError("invalid quantized KV configuration")
        if self.pool_dtype not in _POOLS:
            raise ValueError(f"unknown quantized KV pool dtype {self.pool_dtype}")

    @property
    def pages_per_seq(self) -> int:
        return (self.capacity + self.page_tokens - 1) // self.page_tokens


class QuantizedKVCache:
    """Pools, scales, page tables [B][pages_per_seq], lengths [B] and the free list, all on the device.  Page ids
    leave the free list from its end: the highest first."""

    def __init__(self, config: QuantizedKVConfig, device="cuda"):
        config.validate()
        self.config = config
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())  # where the pools are, whatever is current later
        self.lib = _abi.load()
        self.num_pages = config.num_pages or config.batch * config.pages_per_seq
        self.pool_dtype, store = _POOLS[config.pool_dtype]
        n, h, pt, d = self.num_pages, config.kv_heads, config.page_tokens, config.head_dim
        make = lambda shape, dtype, value: torch.full(shape, value, dtype=dtype, device=self.device)  # noqa: E731
        self.k_pool = make((n, h, pt, d), torch.int8, 0).view(store)
        self.v_pool = make((n, h, d, pt), torch.int8, 0).view(store)
        self.scales = make((n, h, 2), torch.float32, 0.0)
        self.page_table = make((config.batch, config.pages_per_seq), torch.int32, -1)
        self.seq_lens = make((config.batch,), torch.int32, 0)
        self.free_pages = torch.arange(n, dtype=torch.int32, device=self.device)
        self.free_count = make((1,), torch.int32, n)

    @property
    def capacity(self) -> int:
        """Positions that a page table covers."""
        return self.config.pages_per_seq * self.config.page_tokens


@dataclasses.dataclass
class StepPlan:
    """Where a step's tokens go: starts int32 [B + 1], positions int32 [T], slots int64 [T] (-1: padding)."""
    starts: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


def plan_step(cache: QuantizedKVCache, counts: torch.Tensor, max_tokens: int, keep: Optional[torch.Tensor] = None,
              out: Optional[StepPlan] = None, stream: Optional[torch.cuda.Stream] = None) -> StepPlan:
    """Gives back the pages behind each sequence's first keep[b] tokens (int32 [B]; None: all are kept; 0 ends a
    sequence), then grants sequence b the counts[b] tokens (int32 [B]) that it asks for and takes their pages: all of
    them or none, in the sequences' order, as far as the table's capacity, max_tokens rows and the free pages go (a
    sequence that does not fit stops the later ones that need what it waited for).  Moves cache.seq_lens; sequence b
    got nothing where starts[b + 1] == starts[b].  `out`: a plan of max_tokens rows to write into."""
    c = cache.config
    if max_tokens <= 0:
        raise ValueError("a step needs room for at least one row")
    _tensor(cache, counts, "counts", torch.int32, (c.batch,))
    if keep is not None:
        _tensor(cache, keep, "keep", torch.int32, (c.batch,))
    with _on(cache, stream) as s:
        if out is None:
            make = lambda n, dtype: torch.empty(n, dtype=dtype, device=cache.device)  # noqa: E731
            out = StepPlan(make(c.batch + 1, torch.int32), make(max_tokens, torch.int32), make(max_tokens, torch.int64))
        a = _abi.KvPlanArgs()
        a.keep, a.counts = None if keep is None else keep.data_ptr(), counts.data_ptr()
        a.seq_lens, a.page_table = cache.seq_lens.data_ptr(), cache.page_table.data_ptr()
        a.free_pages, a.free_count = cache.free_pages.data_ptr(), cache.free_count.data_ptr()
        a.starts = _tensor(cache, out.starts, "starts", torch.int32, (c.batch + 1,)).data_ptr()
        a.positions = _tensor(cache, out.positions, "positions", torch.int32, (max_tokens,)).data_ptr()
        a.slots = _tensor(cache, out.slots, "slots", torch.int64, (max_tokens,)).data_ptr()
        a.batch, a.pages_per_seq, a.num_pages = c.batch, c.pages_per_seq, cache.num_pages
        a.page_tokens, a.max_tokens = c.page_tokens, max_tokens
        check(cache.lib.sfg_hip_kv_plan_v1(ctypes.byref(a), s))
    return out


# ---------------------------------------------------------------- rotary positions
class RotaryAngles:
    """Angles per position of rotary_dim / 2 pairs, on the device as 64-bit turns, and the factor on cosine and sine.

    scaling: "plain"; for contexts longer than the weights were trained on, by `factor`: "linear" (positions divided),
    "base" (a larger theta), "bands" (pairs that turn less than `low` times over the original `context` divided, those
    over `high` times kept, mixed between), "ramp" (the same by pair index, with a factor on cosine and sine).
    sfg_rope_scaling in include/sfg_hip.h has the formulas.  inv_freq: angles of the caller's own (float64 [pairs] on
    the host) instead."""

    def __init__(self, rotary_dim: int, theta: float = 10000.0, scaling: str = "plain", factor: float = 1.0,
                 context: float = 0.0, low: float = 1.0, high: float = 32.0, inv_freq=None, magnitude: Optional[float] = None,
                 device="cuda"):
        if rotary_dim <= 0 or rotary_dim % 2:
            raise ValueError("rotary_dim must be positive and even")
        lib = _abi.load()
        self.rotary_dim = int(rotary_dim)
        pairs = self.rotary_dim // 2
        found = ctypes.c_float(1.0)
        if inv_freq is None:
            if scaling not in _SCALINGS:
                raise ValueError(f"unknown rotary scaling {scaling}")
            w = np.empty(pairs, np.float64)
            how = _abi.RopeScaling(_SCALINGS[scaling], theta, factor, context, low, high)
            check(lib.sfg_hip_rope_inv_freq_host_v1(w.ctypes.data, ctypes.byref(found), self.rotary_dim, ctypes.byref(how)))
        else:
            w = np.ascontiguousarray(inv_freq, np.float64)
            if w.shape != (pairs,):
                raise ValueError("inv_freq: one angle for each pair")
        turns = np.empty(pairs, np.uint64)
        check(lib.sfg_hip_rope_turns_host_v1(turns.ctypes.data, w.ctypes.data, pairs))
        self.inv_freq = w
        self.magnitude = float(found.value if magnitude is None else magnitude)
        self.device = torch.device(device)
        if self.device.type == "cuda" and self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.turns = torch.from_numpy(turns.view(np.int64)).to(self.device)


def _no_gradients(*tensors) -> None:
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in tensors):
        raise ValueError("gradients are not computed: call under torch.no_grad(), or with detached tensors")


def _rows(where, t, name: str, dtypes, shape=None) -> int:
    """A row's stride, in elements, of t [T][heads][D], whose heads lie one behind the other."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.dtype not in dtypes or 0 in t.shape:
        raise ValueError(f"{name} must be a tensor [tokens][heads][head_dim] of {' or '.join(str(d) for d in dtypes)}")
    if t.device != where.device:
        raise ValueError(f"{name} must be on {where.device}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} must have shape {tuple(shape)}; got {tuple(t.shape)}")
    n, h, d = t.shape
    stride = t.stride(0) if n > 1 else h * d
    if (d > 1 and t.stride(2) != 1) or (h > 1 and t.stride(1) != d) or stride < h * d:
        raise ValueError(f"{name}: the heads of a row must lie one behind the other, and rows apart")
    return stride


def rotate(angles: RotaryAngles, positions: torch.Tensor, q: Optional[torch.Tensor] = None, k: Optional[torch.Tensor] = None,
           layout: str = "half", q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
           stream: Optional[torch.cuda.Stream] = None):
    """Turns the first angles.rotary_dim values of each head by the row's position (int32 [T]; negative: the row is left
    as it is) and copies the others.  q [T][Hq][D], k [T][Hkv][D] (fp32 or bf16; parts of a wider row will do); pairs
    (i, i + rotary_dim / 2) in the "half" layout, (2 i, 2 i + 1) in the "interleaved" one.  q_out = q rotates in place;
    by default outputs are allocated.  Returns (q_out, k_out)."""
    if layout not in _LAYOUTS:
        raise ValueError(f"unknown rotary layout {layout}")
    _no_gradients(q, k, q_out, k_out)
    given = [x for x in (q, k) if x is not None]
    if not given:
        raise ValueError("rotate needs queries or keys")
    if (q is None and q_out is not None) or (k is None and k_out is not None):
        raise ValueError("an output without its input")
    a = _abi.RopeArgs()
    kinds = (given[0].dtype,) if isinstance(given[0], torch.Tensor) and given[0].dtype in _DTYPES else tuple(_DTYPES)
    for x, name in ((q, "q"), (k, "k")):
        if x is not None:
            _rows(angles, x, name, kinds)
            if x.shape[0] != given[0].shape[0] or x.shape[2] != given[0].shape[2]:
                raise ValueError("q and k must have as many rows and the same head_dim")
    tokens, _, dim = given[0].shape
    if angles.rotary_dim > dim:
        raise ValueError(f"rotary_dim {angles.rotary_dim} > head_dim {dim}")
    _tensor(angles, positions, "positions", torch.int32, (tokens,))
    with _on(angles, stream) as s:
        out = []
        for x, o, name in ((q, q_out, "q"), (k, k_out, "k")):
            if x is None:
                out.append(None)
                continue
            if o is None:
                o = torch.empty(x.shape, dtype=x.dtype, device=x.device)
            setattr(a, name, x.data_ptr())
            setattr(a, name + "_out", o.data_ptr())
            setattr(a, name + "_stride", _rows(angles, x, name, kinds))
            setattr(a, name + "_out_stride", _rows(angles, o, name + "_out", kinds, x.shape))
            out.append(o)
        a.dtype, a.layout, a.magnitude = _DTYPES[given[0].dtype], _LAYOUTS[layout], angles.magnitude
        a.positions, a.turns = positions.data_ptr(), angles.turns.data_ptr()
        a.tokens, a.head_dim, a.rotary_dim = tokens, dim, angles.rotary_dim
        a.q_heads, a.kv_heads = (0 if q is None else q.shape[1]), (0 if k is None else k.shape[1])
        check(_abi.load().sfg_hip_rope_v1(ctypes.byref(a), s))
    return tuple(out)


# ---------------------------------------------------------------- the cache
def append_quantized_kv(cache: QuantizedKVCache, keys: torch.Tensor, values: torch.Tensor, slots: torch.Tensor,
                        stream: Optional[torch.cuda.Stream] = None) -> None:
    """Stores keys and values [T][Hkv][D] (fp32 or bf16, rotated; parts of a wider row will do) at slots (int64 [T],
    StepPlan.slots).  The tokens of a page lie side by side, their slots ascending by one.  A page's scale is the
    largest magnitude it has held over 127 (fp8: 448), and earlier tokens are coded anew where it grows; a NaN or an
    infinity makes it, and so all that the page and head hold, NaN until its first token is written again."""
    c = cache.config
    key_stride = _rows(cache, keys, "keys", tuple(_DTYPES))
    shape = (keys.shape[0], c.kv_heads, c.head_dim)
    _rows(cache, keys, "keys", tuple(_DTYPES), shape)
    value_stride = _rows(cache, values, "values", (keys.dtype,), shape)
    _tensor(cache, slots, "slots", torch.int64, (shape[0],))
    a = _abi.Kv8AppendArgs()
    a.keys, a.values, a.dtype, a.key_stride, a.value_stride = keys.data_ptr(), values.data_ptr(), _DTYPES[keys.dtype], key_stride, value_stride
    a.k_pool, a.v_pool, a.pool_dtype = cache.k_pool.data_ptr(), cache.v_pool.data_ptr(), cache.pool_dtype
    a.scales, a.slots = cache.scales.data_ptr(), slots.data_ptr()
    a.tokens, a.kv_heads, a.head_dim, a.page_tokens, a.num_pages = shape[0], c.kv_heads, c.head_dim, c.page_tokens, cache.num_pages
    with _on(cache, stream) as s:
        check(cache.lib.sfg_hip_kv8_append_v1(ctypes.byref(a), s))


def _attention(cache: QuantizedKVCache, tokens: int, q_heads: int, starts, max_rows, max_context, kv_splits: int, scale: float):
    c = cache.config
    if starts is None and tokens % c.batch:
        raise ValueError("rows without starts: as many for every sequence")
    if q_heads <= 0 or q_heads % c.kv_heads:
        raise ValueError("invalid attention configuration")
    a = _abi.Kv8AttnArgs()
    a.batch, a.tokens, a.q_heads, a.kv_heads, a.head_dim = c.batch, tokens, q_heads, c.kv_heads, c.head_dim
    a.max_rows = max_rows if max_rows is not None else (tokens // c.batch if starts is None else tokens)
    a.page_tokens, a.pages_per_seq, a.num_pages = c.page_tokens, c.pages_per_seq, cache.num_pages
    a.max_context = cache.capacity if max_context is None else max_context
    a.pool_dtype, a.kv_splits, a.scale = cache.pool_dtype, kv_splits, scale
    return a


def attention_workspace(cache: QuantizedKVCache, tokens: int, q_heads: int, dtype: torch.dtype, starts=True,
                        max_rows: Optional[int] = None, max_context: Optional[int] = None, kv_splits: int = 0,
                        out_dtype: Optional[torch.dtype] = None) -> int:
    """Bytes of workspace for quantized_attention with queries of these sizes, or of no larger tokens, max_rows and
    max_context.  dtype: the queries'; out_dtype: the output's (default: the same)."""
    if dtype not in _DTYPES or (out_dtype is not None and out_dtype not in _DTYPES):
        raise ValueError(f"queries and outputs must be of {' or '.join(str(d) for d in _DTYPES)}")
    a = _attention(cache, tokens, q_heads, starts, max_rows, max_context, kv_splits, 0.0)
    a.q_dtype, a.out_dtype = _DTYPES[dtype], _DTYPES[dtype if out_dtype is None else out_dtype]
    return cache.lib.sfg_hip_attn_kv8_workspace_v1(ctypes.byref(a))


def quantized_attention(cache: QuantizedKVCache, query: torch.Tensor, starts: Optional[torch.Tensor] = None,
                        max_rows: Optional[int] = None, max_context: Optional[int] = None, out: Optional[torch.Tensor] = None,
                        scale: float = 0.0, kv_splits: int = 0, workspace=None,
                        stream: Optional[torch.cuda.Stream] = None) -> torch.Tensor:
    """Causal attention of each sequence's newest rows (query [T][Hq][D], fp32 or bf16; their keys and values are in the
    cache) over its cached tokens: of a sequence's R rows and L tokens row i sees token j iff j <= L - R + i; a row that
    sees nothing is NaN.  starts: int32 [B + 1] (StepPlan.starts), None: as many rows for every sequence.  max_rows: the
    most rows of any sequence (default: all T; rows past it are not computed); max_context: no sequence is longer
    (default: the capacity).  Both are the bounds that a captured call is built for: with a max_rows of thousands
    sequences are not split, so a decode step is better captured with its own.  T * Hq stays below 2^22."""
    if not isinstance(query, torch.Tensor) or query.dim() != 3:
        raise ValueError("query must be a tensor [tokens][q_heads][head_dim]")
    _no_gradients(query, out)
    tokens, q_heads = int(query.shape[0]), int(query.shape[1])
    q_stride = _rows(cache, query, "query", tuple(_DTYPES), (tokens, q_heads, cache.config.head_dim))
    a = _attention(cache, tokens, q_heads, starts, max_rows, max_context, kv_splits, scale)
    if starts is not None:
        a.starts = _tensor(cache, starts, "starts", torch.int32, (cache.config.batch + 1,)).data_ptr()
    with _on(cache, stream) as s:
        if out is None:
            out = torch.empty(query.shape, dtype=query.dtype, device=query.device)
        a.q, a.q_dtype, a.q_stride = query.data_ptr(), _DTYPES[query.dtype], q_stride
        a.out_stride = _rows(cache, out, "out", tuple(_DTYPES), query.shape)
        a.out, a.out_dtype = out.data_ptr(), _DTYPES[out.dtype]
        a.k_pool, a.v_pool, a.scales = cache.k_pool.data_ptr(), cache.v_pool.data_ptr(), cache.scales.data_ptr()
        a.page_table, a.seq_lens = cache.page_table.data_ptr(), cache.seq_lens.data_ptr()
        ws = _workspace(cache, workspace, cache.lib.sfg_hip_attn_kv8_workspace_v1(ctypes.byref(a)))
        check(cache.lib.sfg_hip_attn_kv8_v1(ctypes.byref(a), ws.data_ptr(), ws.numel(), s))
    return out
