"""The operators that choose what a paged KV cache keeps and reads: what is measured of them.

Five kinds of pass, all over the paged pools (K [page][Hkv][page_tokens][D],
V [page][Hkv][D][page_tokens], one page-table row per sequence):

  tree     attention of a tree of drafted tokens over the cache (sfg_hip_attn_tree_v1);
  accept   the drafts' K / V appended, then the accepted path moved behind the committed
           tokens (sfg_hip_kv_append_pool_v1, sfg_hip_kv_compact_v1);
  weights  decode attention that adds each cached token's attention weight to its
           accumulator (sfg_hip_attn_weights_v1);
  evict    the tokens to keep by accumulated weight, and the cache compacted to them
           (sfg_hip_kv_select_v1, sfg_hip_kv_compact_v1);
  sparse   the page bounds of the newest tokens refreshed, then attention over the pages that
           the bounds select for each query (sfg_hip_kv_page_bounds_v1, sfg_hip_attn_sparse_v1).
"""
from __future__ import annotations

import ctypes
import math
import zlib

import numpy as np
import torch

own = False

PT = 16   # tokens of a page

# (query heads, kv heads, head dim) of this repository's decode configurations: the medium
# profile, the bf16 decode benchmark's model, the large profile
MEDIUM, BASE, LARGE = (16, 4, 64), (16, 4, 128), (32, 8, 128)


def _case(kind, model, dtype, batch, longest, name=None, **more):
    hq, hkv, d = model
    c = {"kind": kind, "dtype": dtype, "batch": batch, "query_heads": hq, "kv_heads": hkv, "head_dim": d,
         "longest": longest, **more}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one user's speculative step: a small tree over a short conversation, the smallest call
        _case("tree", LARGE, "bf16", 1, 900, nodes=8, name="tree-1x8"),
        # a serving batch of ordinary trees over ragged caches
        _case("tree", LARGE, "bf16", 8, 4096, nodes=32, name="tree-8x32"),
        # the widest trees over long caches, the largest call
        _case("tree", LARGE, "bf16", 16, 8192, nodes=64, name="tree-16x64"),
        # fp32 plan (the operator interface's own type), an odd tree
        _case("tree", MEDIUM, "f32", 4, 2001, nodes=13, name="f32-tree-4x13"),
        # one user's accepted path; and that of a whole batch with wide trees
        _case("accept", LARGE, "bf16", 1, 900, nodes=8, name="accept-1x8"),
        _case("accept", LARGE, "bf16", 64, 1024, nodes=64, name="accept-64x64"),
        # the decode step of one long conversation, and of a serving batch, under an eviction policy
        _case("weights", LARGE, "bf16", 1, 4096, rows=1, name="weights-1"),
        _case("weights", BASE, "bf16", 32, 8192, rows=1, name="weights-32"),
        # one user's cache cut back after a chunk of its prompt; a batch halving its caches
        _case("evict", BASE, "bf16", 1, 1501, budget=1024, recent=128, name="evict-1"),
        _case("evict", LARGE, "bf16", 16, 4096, budget=2048, recent=256, name="evict-16"),
        # a decode step over long caches reading 64 pages of up to 2048 per head
        _case("sparse", LARGE, "bf16", 16, 32768, rows=1, fresh=1, top=64, sink=1, recent=2, name="sparse-16x32k"),
        # the first step after a prompt: every page's bounds are made
        _case("sparse", BASE, "bf16", 2, 6000, rows=1, fresh=6000, top=32, sink=1, recent=1, name="sparse-prompt-2x6000"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("tree", "tree", "accept", "weights", "evict", "sparse", "sparse"))
    model, dtype = rng.choice((MEDIUM, BASE, LARGE)), rng.choice(("bf16", "bf16", "f32"))
    batch = _log(rng, 1, 16)
    if kind == "tree":
        return _case(kind, model, dtype, batch, _log(rng, 64, 8192 if dtype == "bf16" else 3000), nodes=_log(rng, 1, 64))
    if kind == "accept":
        return _case(kind, model, dtype, _log(rng, 1, 64), _log(rng, 32, 1024), nodes=_log(rng, 2, 64))
    if kind == "weights":
        return _case(kind, model, dtype, batch, _log(rng, 64, 8192), rows=rng.choice((1, 1, 1, 4)))
    if kind == "evict":
        longest = _log(rng, 128, 8192)
        budget = max(16, int(longest * rng.uniform(0.2, 0.9)))
        return _case(kind, model, dtype, batch, longest, budget=budget, recent=int(budget * rng.uniform(0.0, 0.5)))
    longest = _log(rng, 300, 32768)
    return _case(kind, model, dtype, batch, longest, rows=rng.choice((1, 1, 3)), fresh=rng.choice((1, 1, 40, longest)),
                 top=_log(rng, 4, 128), sink=rng.randint(0, 1), recent=rng.randint(1, 2))


# ---------------------------------------------------------------- inputs
def _gen(seed, name):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + zlib.crc32(name.encode())) % (1 << 62))


def _normal(seed, name, shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=_gen(seed, name))


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _rows(case):
    return case["nodes"] if case["kind"] == "tree" else case["rows"]


def _lengths(case):
    """The sequences' cached tokens: the longest, and others spread evenly below it.  The work follows from
    the case alone; an eviction's caches are all over the budget."""
    lo = max(1, case.get("rows", 1), case.get("budget", 0) + 1)
    hi = max(lo, case["longest"])
    n = case["batch"]
    return np.array([hi - int((hi - lo) * ((k * 0.6180339887) % 1.0)) for k in range(n)], np.int32)


def _capacity(case):
    """Positions that the page tables cover: the longest cache and the drafts behind it."""
    return -(-(case["longest"] + case.get("nodes", 0)) // PT) * PT


def _tree(rng, batch, nodes):
    """Ancestor-or-self bits [B][T][words] of random trees: a node's parent is an earlier node or the last committed token."""
    seen = np.zeros((batch, nodes, nodes), bool)
    for b in range(batch):
        for t in range(nodes):
            # the drafts of a position follow each other: parents are recent nodes
            parent = int(rng.integers(max(-1, t - 9), t)) if t else -1
            if parent >= 0:
                seen[b, t] = seen[b, parent]
            seen[b, t, t] = True
    return seen


def _words(bits):
    """Bits [..., T] as little-endian 32-bit words [..., ceil(T / 32)]."""
    t = bits.shape[-1]
    pad = np.zeros((*bits.shape[:-1], -(-t // 32) * 32), bool)
    pad[..., :t] = bits
    return np.packbits(pad, axis=-1, bitorder="little").view(np.int32)


def _path(rng, bits, t):
    """The longest node of a few drawn ones, as the path of its ancestors: what a verification accepts."""
    best = max((int(rng.integers(0, t)) for _ in range(3)), key=lambda n: int(bits[n].sum()))
    return np.flatnonzero(bits[best])


def _inputs(case, seed):
    b, hq, hkv, d = (case[n] for n in ("batch", "query_heads", "kv_heads", "head_dim"))
    dt = _dtype(case)
    cap = _capacity(case)
    per = cap // PT
    rng = np.random.default_rng(seed % (1 << 32))
    s = {"case": case, "lens": torch.from_numpy(_lengths(case)).cuda(),
         "table": torch.from_numpy(rng.permutation(b * per).astype(np.int32).reshape(b, per)).cuda()}
    # keys: channels with their own offset and pages whose tokens resemble each other
    k = _normal(seed, "k", (b * per, hkv, PT, d)) + _normal(seed, "kp", (b * per, hkv, 1, d), 0.7) + _normal(seed, "kc", (1, hkv, 1, d))
    s["k"] = k.to(dt)
    del k
    s["v"] = _normal(seed, "v", (b * per, hkv, d, PT)).to(dt)
    kind = case["kind"]
    if kind in ("tree", "weights", "sparse"):
        s["q"] = _normal(seed, "q", (b, hq, _rows(case), d), 1.5).to(dt)
        s["out"] = torch.empty_like(s["q"])
    if kind == "tree":
        s["mask"] = torch.from_numpy(_words(_tree(rng, b, case["nodes"]))).cuda()
    if kind == "accept":
        t = case["nodes"]
        bits = _tree(rng, b, t)
        paths = [_path(rng, bits[n], t) for n in range(b)]
        keep = np.full((b, 1, t), -1, np.int32)
        for n, p in enumerate(paths):
            keep[n, 0, : len(p)] = p
        s["keep"] = torch.from_numpy(keep).cuda()
        s["counts"] = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
        s["new_lens"] = torch.empty(b, dtype=torch.int32, device="cuda")
        s["dk"], s["dv"] = (_normal(seed, n, (b, hkv, t, d)).to(dt) for n in ("dk", "dv"))
    if kind in ("weights", "evict"):
        # accumulated weights so far: heavy-tailed, older tokens have gathered more
        w = torch.exp(2.0 * _normal(seed, "w", (b, hkv, cap)))
        s["weights"] = w * (cap / (cap + 4.0 * torch.arange(cap, device="cuda")))
        s["weights"][torch.arange(cap, device="cuda")[None, None].expand(b, hkv, cap) >= s["lens"][:, None, None]] = 0.0
    if kind == "evict":
        s["keep"] = torch.empty((b, hkv, case["budget"]), dtype=torch.int32, device="cuda")
        s["counts"] = torch.empty(b, dtype=torch.int32, device="cuda")
        s["new_lens"] = torch.empty(b, dtype=torch.int32, device="cuda")
        s["kept"] = torch.empty((b, hkv, cap), device="cuda")
    if kind == "sparse":
        s["selected"] = torch.empty((b, case["rows"], hkv, case["top"]), dtype=torch.int32, device="cuda")
        # the bounds as the last step left them: those of all but the fresh tokens
        s["bounds"] = torch.zeros((b * per, hkv, 2, d), dtype=dt, device="cuda")
        old = (s["lens"] - case["fresh"]).clamp(min=0)
        if case["fresh"] < case["longest"]:
            _bounds(s, torch.zeros_like(old), old, case["longest"])
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:
        _prepare_own(s)
    return s


# ---------------------------------------------------------------- the framework's calls
def _prepare_own(s):
    from schedforge_amd import _abi
    case, lib = s["case"], _abi.load()
    s["lib"], s["check"] = lib, _abi.check
    dt = _abi.F32 if case["dtype"] == "f32" else _abi.BF16
    s["dt"] = dt
    b, hq, hkv, d = (case[n] for n in ("batch", "query_heads", "kv_heads", "head_dim"))
    p = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    s["p"] = p
    if "q" not in s:
        return
    a = _abi.PagedAttnArgs()
    a.q, a.q_dtype, a.k_pool, a.v_pool, a.kv_dtype = p["q"], dt, p["k"], p["v"], dt
    a.page_table, a.seq_lens, a.out, a.out_dtype = p["table"], p["lens"], p["out"], dt
    a.batch, a.q_heads, a.kv_heads, a.rows, a.head_dim = b, hq, hkv, _rows(case), d
    a.page_tokens, a.pages_per_seq, a.num_pages = PT, s["table"].shape[1], s["k"].shape[0]
    a.max_context, a.kv_splits, a.scale = case["longest"], 0, 0.0
    s["args"] = a
    ref = ctypes.byref(a)
    n = {"tree": lambda: lib.sfg_hip_attn_tree_workspace_v1(ref),
         "weights": lambda: lib.sfg_hip_attn_weights_workspace_v1(ref),
         "sparse": lambda: lib.sfg_hip_attn_sparse_workspace_v1(ref, case.get("top", 0))}[case["kind"]]()
    s["ws"] = torch.empty(max(1, n), dtype=torch.uint8, device="cuda")
    p["ws"] = s["ws"].data_ptr()


def _run_own(s):
    lib, case, p = s["lib"], s["case"], s["p"]
    stream = torch.cuda.current_stream().cuda_stream
    kind = case["kind"]
    b, hkv, d, per, pages = case["batch"], case["kv_heads"], case["head_dim"], s["table"].shape[1], s["k"].shape[0]
    if kind == "tree":
        s["check"](lib.sfg_hip_attn_tree_v1(ctypes.byref(s["args"]), p["mask"], s["mask"].stride(0), p["ws"],
                                            s["ws"].numel(), stream))
        return s["out"]
    if kind == "accept":
        t = case["nodes"]
        s["check"](lib.sfg_hip_kv_append_pool_v1(p["dk"], p["dv"], s["dt"], p["k"], p["v"], s["dt"], p["table"],
                                                 p["lens"], 0, 0, b, hkv, t, d, PT, per, pages, stream))
        s["check"](lib.sfg_hip_kv_compact_v1(p["k"], p["v"], s["dt"], p["table"], p["lens"], p["keep"], 1, t,
                                             p["counts"], p["new_lens"], t, b, hkv, d, PT, per, pages, stream))
        return {"k": s["k"], "v": s["v"], "lens": s["new_lens"]}
    if kind == "weights":
        s["check"](lib.sfg_hip_attn_weights_v1(ctypes.byref(s["args"]), p["weights"], s["weights"].shape[2], p["ws"],
                                               s["ws"].numel(), stream))
        return {"out": s["out"], "weights": s["weights"]}
    if kind == "evict":
        n = case["budget"]
        s["check"](lib.sfg_hip_kv_select_v1(p["weights"], s["weights"].shape[2], p["lens"], case["longest"], n,
                                            case["recent"], p["keep"], p["counts"], p["kept"], b, hkv, stream))
        s["check"](lib.sfg_hip_kv_compact_v1(p["k"], p["v"], s["dt"], p["table"], None, p["keep"], hkv, n, p["counts"],
                                             p["new_lens"], n, b, hkv, d, PT, per, pages, stream))
        return {"k": s["k"], "v": s["v"], "keep": s["keep"], "lens": s["new_lens"], "weights": s["kept"]}
    s["check"](lib.sfg_hip_kv_page_bounds_v1(p["k"], s["dt"], p["table"], p["lens"], case["longest"], case["fresh"],
                                             p["bounds"], b, hkv, d, PT, per, pages, stream))
    s["check"](lib.sfg_hip_attn_sparse_v1(ctypes.byref(s["args"]), p["bounds"], case["top"], case["sink"], case["recent"],
                                          p["selected"], p["ws"], s["ws"].numel(), stream))
    return {"out": s["out"], "selected": s["selected"], "bounds": s["bounds"]}


# ---------------------------------------------------------------- the plain forms
def _tokens(pool, table, d_last):
    """A pool's tokens in logical order, [B][Hkv][capacity][D] in its own type."""
    t = pool[table.long()]                                  # [B][per][Hkv][pt][D] or [..][D][pt]
    if not d_last:
        t = t.transpose(-1, -2)
    b, per, h, pt, d = t.shape
    return t.permute(0, 2, 1, 3, 4).reshape(b, h, per * pt, d)


def _softmax(x):
    """Softmax weights over the last dimension; hidden entries hold -inf."""
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _attend(q, k, v, seen, scale):
    """q [B][Hq][T][D], k / v [B][Hkv][L][D], seen [B][T][L]: out and the weights [B][Hkv][G][T][L]."""
    b, hq, t, d = q.shape
    hkv, n = k.shape[1], k.shape[2]
    g = hq // hkv
    x = torch.matmul(q.float().reshape(b, hkv, g * t, d), k.float().transpose(-1, -2)) * scale
    x = x.reshape(b, hkv, g, t, n).masked_fill(~seen[:, None, None], -math.inf)
    w = _softmax(x)
    out = torch.matmul(w.reshape(b, hkv, g * t, n), v.float())
    return out.reshape(b, hq, t, d), w


def _bounds(s, begin, end, tokens):
    """Refreshes the bounds of the pages that hold tokens [begin, end) of each sequence, at most `tokens` of them."""
    table = s["table"]
    n = min(table.shape[1], (tokens + PT - 1) // PT + 1)
    at = (end[:, None] + PT - 1) // PT - 1 - torch.arange(n, device="cuda")        # logical pages, the newest first
    due = (at >= 0) & ((at + 1) * PT > begin[:, None])
    at = at.clamp(min=0)
    page = torch.gather(table, 1, at).long()
    k = s["k"][page]                                                               # [B][n][Hkv][pt][D]
    live = (at[:, :, None] * PT + torch.arange(PT, device="cuda")) < end[:, None, None]
    live = live[:, :, None, :, None]
    new = torch.stack((k.masked_fill(~live, math.inf).amin(3), k.masked_fill(~live, -math.inf).amax(3)), 3)
    s["bounds"][page[due]] = new[due]


def _move(s, src, dst):
    """Token src[b][h][i] of each sequence and kv head written at position dst[b][h][i], all read before."""
    b, h = (torch.arange(n, device="cuda") for n in src.shape[:2])
    b, h = b[:, None, None], h[None, :, None]
    frm, to = s["table"][b, (src // PT).long()].long(), s["table"][b, (dst // PT).long()].long()
    v = s["v"].transpose(-1, -2)
    k_moved, v_moved = s["k"][frm, h, (src % PT).long()], v[frm, h, (src % PT).long()]
    s["k"][to, h, (dst % PT).long()] = k_moved
    v[to, h, (dst % PT).long()] = v_moved


def _run_tree(s):
    case, lens = s["case"], s["lens"].long()
    t = case["nodes"]
    k, v = _tokens(s["k"], s["table"], True), _tokens(s["v"], s["table"], False)
    at = torch.arange(k.shape[2], device="cuda")[None] - lens[:, None]            # draft index of each position
    u = at.clamp(0, t - 1)[:, None].expand(-1, t, -1)
    word = torch.gather(s["mask"].long(), 2, u // 32)
    bit = ((word >> (u % 32)) & 1).bool()
    seen = (at < 0)[:, None] | (bit & ((at >= 0) & (at < t))[:, None])
    out, _ = _attend(s["q"], k, v, seen, 1.0 / math.sqrt(case["head_dim"]))
    s["out"].copy_(out)
    return s["out"]


def _run_accept(s):
    case, lens = s["case"], s["lens"].long()
    b, hkv, t = case["batch"], case["kv_heads"], case["nodes"]
    i = torch.arange(t, device="cuda")
    at = (lens[:, None] + i)[:, None].expand(b, hkv, t)
    bb, hh = torch.arange(b, device="cuda")[:, None, None], torch.arange(hkv, device="cuda")[None, :, None]
    page = s["table"][bb, at // PT].long()
    s["k"][page, hh, at % PT] = s["dk"]
    s["v"].transpose(-1, -2)[page, hh, at % PT] = s["dv"]
    live = (i[None] < s["counts"][:, None])[:, None]
    src = lens[:, None, None] + torch.where(live, s["keep"].long(), i)
    _move(s, src.expand(b, hkv, t), at)
    s["new_lens"].copy_(lens + s["counts"])
    return {"k": s["k"], "v": s["v"], "lens": s["new_lens"]}


def _causal(case, lens, n):
    """Which of n positions each of the newest `rows` tokens sees, [B][rows][n]."""
    r = case["rows"]
    end = lens[:, None] - r + 1 + torch.arange(r, device="cuda")
    return torch.arange(n, device="cuda")[None, None] < end[:, :, None]


def _run_weights(s):
    case, lens = s["case"], s["lens"].long()
    k, v = _tokens(s["k"], s["table"], True), _tokens(s["v"], s["table"], False)
    out, w = _attend(s["q"], k, v, _causal(case, lens, k.shape[2]), 1.0 / math.sqrt(case["head_dim"]))
    s["out"].copy_(out)
    s["weights"] += w.sum((2, 3))
    return {"out": s["out"], "weights": s["weights"]}


def _run_evict(s):
    case, lens = s["case"], s["lens"].long()[:, None, None]
    n, cap = case["budget"], s["weights"].shape[2]
    pos = torch.arange(cap, device="cuda")
    key = s["weights"].masked_fill((pos >= lens - case["recent"]) & (pos < lens), math.inf)
    key = key.masked_fill((pos >= lens).expand_as(key), -math.inf)
    order = torch.sort(key, dim=2, descending=True, stable=True).indices[:, :, :n]
    keep = order.sort(dim=2).values                          # every cache here is longer than the budget
    s["keep"].copy_(keep)
    s["kept"].zero_()
    s["kept"][:, :, :n] = torch.gather(s["weights"], 2, keep)
    _move(s, keep, pos[:n].expand_as(keep))
    s["new_lens"].fill_(n)
    return {"k": s["k"], "v": s["v"], "keep": s["keep"], "lens": s["new_lens"], "weights": s["kept"]}


def _run_sparse(s):
    case, lens = s["case"], s["lens"].long()
    b, hq, hkv, d, r, top = (case[n] for n in ("batch", "query_heads", "kv_heads", "head_dim", "rows", "top"))
    g = hq // hkv
    _bounds(s, (lens - case["fresh"]).clamp(min=0), lens, case["fresh"])
    per = s["table"].shape[1]
    q = s["q"].reshape(b, hkv, g, r, d)
    # scores in 64 bits: they decide which pages are read
    up, down = q.double().clamp(min=0).sum(2), q.double().clamp(max=0).sum(2)     # [B][Hkv][r][D]
    bd = s["bounds"][s["table"].long()].double()                                  # [B][per][Hkv][2][D]
    lo, hi = (bd[:, :, :, i].permute(0, 2, 3, 1) for i in (0, 1))                 # [B][Hkv][D][per]
    score = torch.matmul(up, hi) + torch.matmul(down, lo)                         # [B][Hkv][r][per]
    end = lens[:, None] - r + 1 + torch.arange(r, device="cuda")                  # tokens seen [B][r]
    pages = ((end + PT - 1) // PT)[:, None, :, None]
    pos = torch.arange(per, device="cuda")
    score = score.masked_fill((pos < case["sink"]) | (pos >= pages - case["recent"]), math.inf)
    score = score.masked_fill(pos >= pages, -math.inf)
    order = torch.sort(score, dim=3, descending=True, stable=True).indices[..., :top]
    order = torch.where(order < pages, order, per).sort(dim=3).values             # unused entries last
    taken = order < per
    if order.shape[3] < top:
        order, taken = (torch.nn.functional.pad(x, (0, top - x.shape[3])) for x in (order, taken))
    s["selected"].copy_(torch.where(taken, order, -1).permute(0, 2, 1, 3))
    page = s["table"][torch.arange(b, device="cuda")[:, None, None, None], order.clamp(max=per - 1)].long()
    h = torch.arange(hkv, device="cuda")[None, :, None, None]
    k = s["k"][page, h].float().reshape(b, hkv, r, top * PT, d)
    v = s["v"][page, h].transpose(-1, -2).float().reshape(b, hkv, r, top * PT, d)
    tok = order[..., None] * PT + torch.arange(PT, device="cuda")
    seen = (taken[..., None] & (tok < end[:, None, :, None, None])).reshape(b, hkv, r, top * PT)
    x = torch.matmul(q.float().transpose(2, 3), k.transpose(-1, -2)) / math.sqrt(d)   # [B][Hkv][r][G][n]
    w = _softmax(x.masked_fill(~seen[:, :, :, None], -math.inf))
    s["out"].copy_(torch.matmul(w, v).transpose(2, 3).reshape(b, hq, r, d))
    return {"out": s["out"], "selected": s["selected"], "bounds": s["bounds"]}


def run(s):
    if own:
        return _run_own(s)
    return {"tree": _run_tree, "accept": _run_accept, "weights": _run_weights, "evict": _run_evict,
            "sparse": _run_sparse}[s["case"]["kind"]](s)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    b, hq, hkv, d = (case[n] for n in ("batch", "query_heads", "kv_heads", "head_dim"))
    kind, lens = case["kind"], [int(n) for n in _lengths(case)]
    if kind == "tree":
        t = case["nodes"]
        seen = sum(n + t for n in lens)
        return {"bytes": 2 * hkv * d * e * seen + 2 * b * hq * t * d * e + b * t * -(-t // 32) * 4,
                "flops": 4.0 * hq * d * t * seen}
    if kind == "accept":
        # the drafts read and written; of the accepted ones (a fourth, say) read and written again
        return {"bytes": 2 * b * hkv * d * e * case["nodes"] * 2.5, "flops": 0}
    if kind == "weights":
        r = case["rows"]
        return {"bytes": sum(lens) * hkv * (2 * d * e + 8) + 2 * b * hq * r * d * e, "flops": 4.0 * hq * d * r * sum(lens)}
    if kind == "evict":
        n = case["budget"]
        return {"bytes": b * hkv * (n * (4 * d * e + 4) + 4 * _capacity(case)) + sum(lens) * hkv * 4, "flops": 0}
    r, top = case["rows"], case["top"]
    per = [-(-n // PT) for n in lens]
    fresh = sum(min(p, -(-case["fresh"] // PT)) for p in per)
    taken = sum(min(p, top) for p in per)
    return {"bytes": hkv * (sum(per) * 2 * d * e + fresh * (PT + 2) * d * e + taken * PT * 2 * d * e * r) + 2 * b * hq * r * d * e,
            "flops": 4.0 * hq * r * taken * PT * d + 4.0 * hkv * r * d * sum(per)}


# ---------------------------------------------------------------- the definitions in 64 bits
def _logical(s, name, b):
    """Sequence b's tokens [Hkv][capacity][D] in 64 bits."""
    t = s[name][s["table"][b].long()].double()
    t = t if name == "k" else t.permute(0, 1, 3, 2)
    return torch.cat(tuple(t.unbind(0)), dim=1)


def _rows64(q, k, v, seen, d):
    """One kv head: q [rows][D] against k, v [L][D]; seen [rows][L]."""
    x = (q @ k.T) * (d ** -0.5)
    x[~seen] = -math.inf
    p = torch.softmax(x, dim=1)
    return p @ v, p


def exact(case, seed):
    s = _inputs(case, seed)
    kind, lens = case["kind"], [int(n) for n in _lengths(case)]
    b, hq, hkv, d = (case[n] for n in ("batch", "query_heads", "kv_heads", "head_dim"))
    g = hq // hkv
    if kind in ("tree", "weights"):
        out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
        weights = s["weights"].double() if kind == "weights" else None
        t = _rows(case)
        for n in range(b):
            k, v = _logical(s, "k", n), _logical(s, "v", n)
            seen = torch.zeros((t, k.shape[1]), dtype=torch.bool, device="cuda")
            if kind == "tree":
                seen[:, : lens[n]] = True
                for u in range(t):
                    seen[:, lens[n] + u] = (s["mask"][n, :, u // 32].long() & (1 << (u % 32))) != 0
            else:
                for i in range(t):
                    seen[i, : lens[n] - t + i + 1] = True
            for h in range(hq):
                o, p = _rows64(s["q"][n, h].double(), k[h // g], v[h // g], seen, d)
                out[n, h] = o
                if weights is not None:
                    weights[n, h // g] += p.sum(0)
        return out if kind == "tree" else {"out": out, "weights": weights}
    if kind in ("accept", "evict"):
        # moves alone: the values themselves, token by token through each sequence's own list
        k, v = s["k"].double(), s["v"].double()
        keep = np.full((b, hkv, case.get("budget", case.get("nodes"))), -1, np.int64)
        new = np.zeros(b, np.int64)
        kept = torch.zeros((b, hkv, _capacity(case)), dtype=torch.float64, device="cuda")
        for n in range(b):
            pages = s["table"][n].long()
            kk, vv = _logical(s, "k", n), _logical(s, "v", n)
            if kind == "accept":
                t, c = case["nodes"], int(s["counts"][n])
                kk[:, lens[n]: lens[n] + t], vv[:, lens[n]: lens[n] + t] = s["dk"][n].double(), s["dv"][n].double()
                path = lens[n] + s["keep"][n, 0, :c].long()
                kk[:, lens[n]: lens[n] + c], vv[:, lens[n]: lens[n] + c] = kk[:, path].clone(), vv[:, path].clone()
                new[n] = lens[n] + c
            else:
                w = s["weights"][n].cpu().numpy().astype(np.float64)
                old, most = lens[n] - case["recent"], case["budget"] - case["recent"]
                for h in range(hkv):
                    heavy = np.lexsort((np.arange(old), -w[h, :old]))[:most]
                    keep[n, h] = np.concatenate((np.sort(heavy), np.arange(old, lens[n])))
                    at = torch.from_numpy(keep[n, h]).cuda()
                    kk[h, : case["budget"]], vv[h, : case["budget"]] = kk[h, at].clone(), vv[h, at].clone()
                    kept[n, h, : case["budget"]] = torch.from_numpy(w[h, keep[n, h]]).cuda()
                new[n] = case["budget"]
            per = pages.numel()
            k[pages] = kk.reshape(hkv, per, PT, d).transpose(0, 1)
            v[pages] = vv.reshape(hkv, per, PT, d).permute(1, 0, 3, 2)
        found = {"k": k, "v": v, "lens": torch.from_numpy(new.astype(np.int32))}
        return found if kind == "accept" else {**found, "keep": torch.from_numpy(keep.astype(np.int32)), "weights": kept}
    r, top = case["rows"], case["top"]
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    selected = torch.full((b, r, hkv, top), -1, dtype=torch.int32)
    bounds = s["bounds"].double()
    for n in range(b):
        k, v, pages = _logical(s, "k", n), _logical(s, "v", n), s["table"][n].long()
        last = -(-lens[n] // PT)
        whole = k[:, : last * PT].reshape(hkv, last, PT, d).clone()
        tail = lens[n] - (last - 1) * PT
        lo, hi = whole.amin(2), whole.amax(2)
        lo[:, -1], hi[:, -1] = whole[:, -1, :tail].amin(1), whole[:, -1, :tail].amax(1)
        for p in range(max(0, lens[n] - case["fresh"]) // PT, last):
            bounds[pages[p], :, 0], bounds[pages[p], :, 1] = lo[:, p], hi[:, p]
        for i in range(r):
            end = lens[n] - r + i + 1
            count = -(-end // PT)
            for h in range(hkv):
                q = s["q"][n, h * g: (h + 1) * g, i].double()
                score = torch.maximum(q[:, None] * lo[h, None, :count], q[:, None] * hi[h, None, :count]).sum((0, 2)).cpu().numpy()
                first = set(range(min(case["sink"], count))) | set(range(max(0, count - case["recent"]), count))
                rest = [p for p in np.lexsort((np.arange(count), -score)) if p not in first]
                take = sorted(first | set(int(p) for p in rest[: max(0, top - len(first))]))
                selected[n, i, h, : len(take)] = torch.tensor(take, dtype=torch.int32)
                tok = torch.cat([torch.arange(p * PT, min((p + 1) * PT, end)) for p in take]).cuda()
                seen = torch.ones((g, tok.numel()), dtype=torch.bool, device="cuda")
                out[n, h * g: (h + 1) * g, i] = _rows64(q, k[h, tok], v[h, tok], seen, d)[0]
    return {"out": out, "selected": selected, "bounds": bounds}
