"""The operators of a serving step over a paged cache held in 8 bits: what is measured of them.

Four kinds of pass, in the order of a step:

  plan    block tables, slot map, positions and row starts made on the GPU from the sequences' lengths
          and token counts, pages given back and taken from the free list (sfg_hip_kv_plan_v1);
  rotate  rotary positions of queries and keys: half and interleaved layouts, part of the head,
          scaled for long contexts (sfg_hip_rope_v1);
  append  keys and values stored in 8 bits at their slots, one scale for each page, kv head and
          pool (sfg_hip_kv8_append_v1);
  attend  causal attention of each sequence's newest rows over the cache (sfg_hip_attn_kv8_v1).

Pools: K [page][Hkv][page_tokens][D], V [page][Hkv][D][page_tokens], int8 or e4m3 codes; scales fp32
[page][Hkv][2] (K's, V's).  A token's value is code * scale.
"""
from __future__ import annotations

import ctypes
import math
import zlib

import numpy as np
import torch

own = False

# (query heads, kv heads, head dim) of this repository's decode configurations: the medium
# profile, the bf16 decode benchmark's model, the large profile
MEDIUM, BASE, LARGE = (16, 4, 64), (16, 4, 128), (32, 8, 128)
MOST = {"i8": 127.0, "fp8": 448.0}   # the largest code


def _case(kind, model, dtype, name=None, **more):
    hq, hkv, d = model
    c = {"kind": kind, "dtype": dtype, "query_heads": hq, "kv_heads": hkv, "head_dim": d, **more}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the decode step of a serving batch: one token a sequence, a new page for every sixteenth
        _case("plan", LARGE, "i8", batch=64, longest=8192, page=16, rows=1, chunk=0, spare=1.0, name="plan-64"),
        # prompts of many requests admitted at once, more than the free pages hold
        _case("plan", LARGE, "i8", batch=256, longest=16384, page=16, rows=200, chunk=3000, spare=0.9, name="plan-256-prompts"),
        # one user's token: the smallest call; a prompt of 8192 tokens deep inside a long context;
        # the operator interface's own type, a quarter of each head
        _case("rotate", LARGE, "bf16", tokens=1, far=4096, layout="half", part=1.0, scaling="plain", name="rotate-1"),
        _case("rotate", LARGE, "bf16", tokens=8192, far=131072, layout="half", part=1.0, scaling="ramp", name="rotate-8192"),
        _case("rotate", MEDIUM, "f32", tokens=1001, far=1000000, layout="interleaved", part=0.25, scaling="linear",
              name="rotate-f32-part"),
        # the decode step of a batch, into pages that hold earlier tokens; whole prompts into new pages
        _case("append", LARGE, "bf16", cache="i8", batch=64, longest=1024, page=16, rows=1, chunk=0, name="append-64"),
        _case("append", LARGE, "bf16", cache="fp8", batch=4, longest=4500, page=16, rows=1500, chunk=3600, name="append-prompts"),
        # one user's token over a short conversation; the decode benchmark's batch and context;
        # two very long contexts; a chunk of a prompt beside decoding sequences; fp32 rows of a
        # drafted continuation over larger pages
        _case("attend", LARGE, "bf16", cache="i8", batch=1, longest=900, page=16, rows=1, chunk=0, name="attend-1"),
        _case("attend", LARGE, "bf16", cache="i8", batch=64, longest=8192, page=16, rows=1, chunk=0, name="attend-64"),
        _case("attend", LARGE, "bf16", cache="fp8", batch=2, longest=131072, page=16, rows=1, chunk=0, name="attend-2x128k"),
        _case("attend", LARGE, "bf16", cache="fp8", batch=8, longest=6000, page=16, rows=1, chunk=512, name="attend-chunk"),
        _case("attend", MEDIUM, "f32", cache="i8", batch=4, longest=2001, page=64, rows=5, chunk=0, name="attend-f32-rows"),
    ]


def _log(rng, lo, hi):
    """A whole number spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("plan", "rotate", "append", "append", "attend", "attend", "attend"))
    model = rng.choice((MEDIUM, BASE, LARGE))
    dtype, cache, page = rng.choice(("bf16", "bf16", "f32")), rng.choice(("i8", "fp8")), rng.choice((16, 16, 32, 64))
    if kind == "plan":
        rows = rng.choice((1, _log(rng, 1, 200)))
        return _case(kind, model, cache, batch=_log(rng, 1, 256), longest=_log(rng, 64, 16384), page=page, rows=rows,
                     chunk=rng.choice((0, _log(rng, 1, 3000))), spare=rng.choice((1.0, 1.0, 0.7)))
    if kind == "rotate":
        return _case(kind, model, dtype, tokens=_log(rng, 1, 8192 if dtype == "bf16" else 4096), far=_log(rng, 16, 1000000),
                     layout=rng.choice(("half", "interleaved")), part=rng.choice((1.0, 1.0, 0.5, 0.25)),
                     scaling=rng.choice(("plain", "linear", "base", "bands", "ramp")))
    rows, chunk = rng.choice((1, 1, _log(rng, 1, 16))), rng.choice((0, 0, _log(rng, 1, 512)))
    if kind == "append":
        if rng.random() < 0.4:
            rows, chunk = _log(rng, 16, 1000), 0
        return _case(kind, model, dtype, cache=cache, batch=_log(rng, 1, 64 if rows <= 64 else 8), longest=_log(rng, 64, 2048),
                     page=page, rows=rows, chunk=chunk)
    batch = _log(rng, 1, 32)
    return _case(kind, model, dtype, cache=cache, batch=min(batch, 8) if chunk else batch,
                 longest=_log(rng, 32, 4096 if chunk else 16384), page=page, rows=rows, chunk=min(chunk, 256) if dtype == "f32" else chunk)


# ---------------------------------------------------------------- inputs
def _gen(seed, name):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + zlib.crc32(name.encode())) % (1 << 62))


def _normal(seed, name, shape, std=1.0):
    return torch.empty(shape, device="cuda").normal_(0.0, std, generator=_gen(seed, name))


def _dtype(case):
    return torch.float32 if case["dtype"] == "f32" else torch.bfloat16


def _rows(case):
    """New tokens of each sequence: `rows`, the first sequence's `chunk` if there is one."""
    r = np.full(case["batch"], case["rows"], np.int64)
    if case["chunk"]:
        r[0] = case["chunk"]
    return r


def _lengths(case):
    """The sequences' tokens, new ones included: the longest, and others spread evenly below it.  The work
    follows from the case alone."""
    r = _rows(case)
    hi = max(case["longest"], int(r.max()))
    return np.array([max(int(r[k]), hi - int((hi - 1) * ((k * 0.6180339887) % 1.0))) for k in range(case["batch"])], np.int64)


def _table(rng, lens, page, per, spare):
    """Pages for every sequence, drawn from a shuffled pool: table [B][per] (-1: none) and the pages left over."""
    need = -(-lens // page)
    ids = rng.permutation(int(need.sum()) + spare).astype(np.int32)
    table = np.full((len(lens), per), -1, np.int32)
    table[np.arange(per)[None] < need[:, None]] = ids[: need.sum()]
    return table, ids[need.sum():]


def _frequencies(case, rotary):
    """Angle per position of each pair, in 64 bits, and the factor on cosine and sine."""
    kind, theta = case["scaling"], 500000.0 if case["far"] > 65536 else 10000.0
    i = torch.arange(rotary // 2, dtype=torch.float64)
    if kind == "base" and rotary > 2:
        theta *= 8.0 ** (rotary / (rotary - 2))
    w = theta ** (-2.0 * i / rotary)
    turns = 8192.0 * w / (2.0 * math.pi)
    if kind == "linear":
        w = w / 8.0
    if kind == "bands":
        t = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        w = w * (t + (1.0 - t) / 8.0)
    if kind == "ramp":
        at = [rotary * math.log(8192.0 / (b * 2.0 * math.pi)) / (2.0 * math.log(theta)) for b in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rotary - 1)
        t = ((i - lo) / max(hi - lo, 0.001)).clamp(0.0, 1.0)
        w = w * (1.0 - t + t / 8.0)
    return w.cuda(), 0.1 * math.log(8.0) + 1.0 if kind == "ramp" else 1.0


def _code(x, scale, cache):
    """Codes of x (any float type) under a scale that broadcasts: the quotient in fp32, rounded to the nearest
    code, ties to even, and cut to the largest; 0 where the scale is 0."""
    y = (x.double() / torch.where(scale > 0, scale, 1.0).double()).float()
    y = torch.where(scale > 0, y, 0.0).clamp(-MOST[cache], MOST[cache])
    return y.round().to(torch.int8) if cache == "i8" else y.to(torch.float8_e4m3fn).view(torch.int8)


def _value(code, cache):
    return code.float() if cache == "i8" else code.view(torch.float8_e4m3fn).float()


def _fill(s, pages, hkv, page, d, cache, seed):
    """Pools that hold what earlier steps appended: channels with their own offset, pages with their own range."""
    k = _normal(seed, "k", (pages, hkv, page, d)) + _normal(seed, "kp", (pages, hkv, 1, d), 0.7) + _normal(seed, "kc", (1, hkv, 1, d))
    ks = (k.abs().amax((2, 3)).double() / MOST[cache]).float()
    s["k"] = _code(k, ks[:, :, None, None], cache)
    del k
    v = _normal(seed, "v", (pages, hkv, d, page)) * torch.exp(_normal(seed, "vp", (pages, hkv, 1, 1), 0.5))
    vs = (v.abs().amax((2, 3)).double() / MOST[cache]).float()
    s["v"] = _code(v, vs[:, :, None, None], cache)
    s["scales"] = torch.stack((ks, vs), 2)


def _inputs(case, seed):
    kind, (hq, hkv, d) = case["kind"], (case[n] for n in ("query_heads", "kv_heads", "head_dim"))
    rng = np.random.default_rng(seed % (1 << 32))
    dev = lambda a, t: torch.from_numpy(np.ascontiguousarray(a)).to("cuda", t)  # noqa: E731
    s = {"case": case}
    if kind == "rotate":
        t, rotary = case["tokens"], int(d * case["part"]) // 2 * 2
        # queries and keys as the projection leaves them, side by side with the values
        qkv = _normal(seed, "qkv", (t, (hq + 2 * hkv) * d), 1.5).to(_dtype(case))
        s["q"], s["k"] = qkv[:, : hq * d].view(t, hq, d), qkv[:, hq * d: (hq + hkv) * d].view(t, hkv, d)
        # runs of consecutive positions, the last of them the farthest
        start = rng.integers(0, max(1, case["far"] - t), size=max(1, t // 700))
        run = np.sort(rng.integers(0, len(start), size=t))
        s["positions"] = dev(np.minimum(start[run] + np.arange(t) - np.searchsorted(run, run), case["far"] - 1), torch.int32)
        s["w"], s["magnitude"] = _frequencies(case, rotary)
        s["q_out"], s["k_out"] = (torch.empty((t, h, d), dtype=_dtype(case), device="cuda") for h in (hq, hkv))
        return s
    rows, lens, page = _rows(case), _lengths(case), case["page"]
    starts = np.concatenate(([0], np.cumsum(rows)))
    s["total"] = int(starts[-1])
    per = -(-int(lens.max()) // page)
    if kind == "plan":
        held = lens - rows                                       # before the step
        table, _ = _table(rng, held, page, per, 0)
        need = int((-(-lens // page) - -(-held // page)).sum())
        spare = int(need * case["spare"])
        used = int((table >= 0).sum())
        ids = rng.permutation(used + spare).astype(np.int32)
        table[table >= 0] = ids[:used]
        free = np.full(used + spare, -1, np.int32)
        free[:spare] = ids[used:]
        s["table"], s["free"], s["free_count"] = dev(table, torch.int32), dev(free, torch.int32), dev(np.array([spare]), torch.int32)
        s["lens"], s["keep"], s["counts"] = dev(held, torch.int32), dev(held, torch.int32), dev(rows, torch.int32)
        s["starts"] = torch.empty(case["batch"] + 1, dtype=torch.int32, device="cuda")
        s["positions"] = torch.empty(s["total"], dtype=torch.int32, device="cuda")
        s["slots"] = torch.empty(s["total"], dtype=torch.int64, device="cuda")
        return s
    table, _ = _table(rng, lens, page, per, 0)
    s["table"], s["lens"], s["starts"] = dev(table, torch.int32), dev(lens, torch.int32), dev(starts, torch.int32)
    _fill(s, int((table >= 0).sum()), hkv, page, d, case["cache"], seed)
    if kind == "append":
        t = s["total"]
        s["keys"] = (_normal(seed, "nk", (t, hkv, d), 1.2) + _normal(seed, "kc", (1, hkv, 1, d))[0, :, 0]).to(_dtype(case))
        s["values"] = _normal(seed, "nv", (t, (hq + 2 * hkv) * d)).to(_dtype(case))[:, (hq + hkv) * d:].view(t, hkv, d)
        b = np.repeat(np.arange(case["batch"]), rows)
        pos = np.arange(t) - starts[b] + (lens - rows)[b]
        s["slots"] = dev(table[b, pos // page].astype(np.int64) * page + pos % page, torch.int64)
    else:
        s["q"] = _normal(seed, "q", (s["total"], hq, d), 1.5).to(_dtype(case))
        s["out"] = torch.empty_like(s["q"])
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
    kind, (hq, hkv, d) = case["kind"], (case[n] for n in ("query_heads", "kv_heads", "head_dim"))
    s["lib"], s["check"] = lib, _abi.check
    p = {n: t.data_ptr() for n, t in s.items() if isinstance(t, torch.Tensor)}
    dt = _abi.F32 if case["dtype"] == "f32" else _abi.BF16
    if kind == "rotate":
        turns = np.empty(s["w"].numel(), np.uint64)
        w = s["w"].cpu().numpy()
        _abi.check(lib.sfg_hip_rope_turns_host_v1(turns.ctypes.data, w.ctypes.data, w.size))
        s["turns"] = torch.from_numpy(turns.view(np.int64)).cuda()
        a = _abi.RopeArgs()
        a.q, a.k, a.q_out, a.k_out, a.dtype = p["q"], p["k"], p["q_out"], p["k_out"], dt
        a.q_stride, a.k_stride = s["q"].stride(0), s["k"].stride(0)
        a.q_out_stride, a.k_out_stride = s["q_out"].stride(0), s["k_out"].stride(0)
        a.positions, a.turns, a.magnitude = p["positions"], s["turns"].data_ptr(), s["magnitude"]
        a.layout = _abi.ROPE_HALF if case["layout"] == "half" else _abi.ROPE_INTERLEAVED
        a.tokens, a.q_heads, a.kv_heads, a.head_dim, a.rotary_dim = case["tokens"], hq, hkv, d, 2 * w.size
    elif kind == "plan":
        a = _abi.KvPlanArgs()
        a.keep, a.counts, a.seq_lens, a.page_table = p["keep"], p["counts"], p["lens"], p["table"]
        a.free_pages, a.free_count, a.starts, a.positions, a.slots = p["free"], p["free_count"], p["starts"], p["positions"], p["slots"]
        a.batch, a.pages_per_seq, a.num_pages, a.page_tokens = case["batch"], s["table"].shape[1], s["free"].numel(), case["page"]
        a.max_tokens = s["total"]
    elif kind == "append":
        a = _abi.Kv8AppendArgs()
        a.keys, a.values, a.dtype = p["keys"], p["values"], dt
        a.key_stride, a.value_stride = s["keys"].stride(0), s["values"].stride(0)
        a.k_pool, a.v_pool, a.pool_dtype, a.scales, a.slots = p["k"], p["v"], _cache_type(_abi, case), p["scales"], p["slots"]
        a.tokens, a.kv_heads, a.head_dim, a.page_tokens, a.num_pages = s["total"], hkv, d, case["page"], s["k"].shape[0]
    else:
        a = _abi.Kv8AttnArgs()
        a.q, a.q_dtype, a.q_stride, a.out, a.out_dtype, a.out_stride = p["q"], dt, hq * d, p["out"], dt, hq * d
        a.k_pool, a.v_pool, a.pool_dtype, a.scales = p["k"], p["v"], _cache_type(_abi, case), p["scales"]
        a.page_table, a.seq_lens, a.starts = p["table"], p["lens"], p["starts"]
        a.batch, a.tokens, a.max_rows = case["batch"], s["total"], int(_rows(case).max())
        a.q_heads, a.kv_heads, a.head_dim = hq, hkv, d
        a.page_tokens, a.pages_per_seq, a.num_pages = case["page"], s["table"].shape[1], s["k"].shape[0]
        a.max_context, a.kv_splits, a.scale = int(_lengths(case).max()), 0, 0.0
        s["ws"] = torch.empty(max(1, lib.sfg_hip_attn_kv8_workspace_v1(ctypes.byref(a))), dtype=torch.uint8, device="cuda")
    s["args"], s["ref"] = a, ctypes.byref(a)


def _cache_type(abi, case):
    return abi.I8 if case["cache"] == "i8" else abi.FP8


def _run_own(s):
    lib, kind, stream = s["lib"], s["case"]["kind"], torch.cuda.current_stream().cuda_stream
    if kind == "plan":
        s["check"](lib.sfg_hip_kv_plan_v1(s["ref"], stream))
    elif kind == "rotate":
        s["check"](lib.sfg_hip_rope_v1(s["ref"], stream))
    elif kind == "append":
        s["check"](lib.sfg_hip_kv8_append_v1(s["ref"], stream))
    else:
        s["check"](lib.sfg_hip_attn_kv8_v1(s["ref"], s["ws"].data_ptr(), s["ws"].numel(), stream))
    return _outputs(s)


def _outputs(s):
    """A pass's outputs.  Codes come as they are stored: both sides have to agree on each of them."""
    names = {"plan": ("table", "lens", "free", "free_count", "starts", "positions", "slots"), "rotate": ("q_out", "k_out"),
             "append": ("k", "v", "scales"), "attend": ("out",)}[s["case"]["kind"]]
    return {n: s[n] for n in names}


# ---------------------------------------------------------------- the plain forms
def _before(x):
    """Sums of the entries before each one."""
    return torch.cumsum(x, 0) - x


def _run_plan(s):
    case, table, free = s["case"], s["table"], s["free"]
    page, per, n, t = case["page"], table.shape[1], free.numel(), s["total"]
    lens = s["lens"].long().clamp(0, per * page)
    keep = torch.minimum(s["keep"].long().clamp(min=0), lens)
    count = s["free_count"].long().clamp(0, n)
    # pages behind the kept tokens go back, each sequence's last one first
    first, end = (keep + page - 1) // page, (lens + page - 1) // page
    logical = torch.arange(per, device="cuda")[None]
    gone = (logical >= first[:, None]) & (logical < end[:, None])
    at = count + _before(end - first)[:, None] + (end[:, None] - 1 - logical)
    stack = torch.cat((free, free.new_empty(1)))                  # the entry behind takes what is not written
    stack[torch.where(gone, at, n)] = torch.where(gone, table, 0)
    table.masked_fill_(gone, -1)
    count = count + (end - first).sum()
    # sequences in order, as far as capacity, free pages and rows go
    want = s["counts"].long().clamp(min=0)
    want = torch.where(keep + want <= per * page, want, 0)
    need = (keep + want + page - 1) // page - first
    fits = ((need == 0) | (torch.cumsum(need, 0) <= count)) & (torch.cumsum(want, 0) <= t)
    want, need = torch.where(fits, want, 0), torch.where(fits, need, 0)
    taken = (logical >= first[:, None]) & (logical < (first + need)[:, None])
    at = count - 1 - _before(need)[:, None] - (logical - first[:, None])
    table.copy_(torch.where(taken, stack[at.clamp(0, n)], table))
    free.copy_(stack[:n])
    s["free_count"].copy_(count - need.sum())
    s["lens"].copy_(keep + want)
    ends = torch.cumsum(want, 0)
    s["starts"].copy_(torch.cat((ends.new_zeros(1), ends)))
    i = torch.arange(t, device="cuda")
    b = torch.searchsorted(ends, i, right=True).clamp(max=case["batch"] - 1)
    pos = keep[b] + i - (ends - want)[b]
    live = i < ends[-1]
    pos = torch.where(live, pos, 0)
    slot = table[b, pos // page].long() * page + pos % page
    s["positions"].copy_(torch.where(live, pos, -1))
    s["slots"].copy_(torch.where(live, slot, -1))


def _run_rotate(s):
    case, n = s["case"], s["w"].numel()
    angle = s["positions"].double()[:, None] * s["w"]             # far positions: 64 bits
    cos, sin = ((f(angle) * s["magnitude"]).float()[:, None] for f in (torch.cos, torch.sin))
    for x, out in ((s["q"], s["q_out"]), (s["k"], s["k_out"])):
        x = x.float()
        turned, rest = x[..., : 2 * n], x[..., 2 * n:]
        if case["layout"] == "half":
            a, b = turned[..., :n], turned[..., n:]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), 2)
        else:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), 3).flatten(2)
        out.copy_(torch.cat((turned, rest), 2))


def _run_append(s):
    case, slots = s["case"], s["slots"]
    page, cache, t = case["page"], case["cache"], slots.numel()
    at, off = slots // page, slots % page
    # the tokens of a page follow each other: its first one speaks for it
    i = torch.arange(t, device="cuda")
    lead = torch.cat((slots.new_ones(1, dtype=torch.bool), at[1:] != at[:-1]))
    run = torch.cumsum(lead, 0) - 1                               # the page's number in this call
    first = torch.full((t,), t - 1, device="cuda").scatter_reduce(0, run, i, "amin")  # behind the last one: unused
    pid, fresh = at[first], off[first] == 0
    used = i <= run[-1]
    for pool, new, which in ((s["k"], s["keys"], 0), (s["v"].transpose(2, 3), s["values"], 1)):
        x = new.float()
        top = torch.zeros((t, x.shape[1]), device="cuda").scatter_reduce(0, run[:, None].expand(-1, x.shape[1]), x.abs().amax(2), "amax")
        old = torch.where(fresh[:, None], 0.0, s["scales"][pid, :, which])
        scale = torch.maximum(old, (top.double() / MOST[cache]).float())
        # the page's earlier tokens under the scale as it is now, then the new ones
        codes = pool[pid]                                          # [run][Hkv][page][D]
        again = _code(_value(codes, cache) * old[:, :, None, None], scale[:, :, None, None], cache)
        earlier = (torch.arange(page, device="cuda")[None] < off[first][:, None]) & used[:, None]
        earlier = earlier[:, None, :, None] & (scale > old)[:, :, None, None]
        codes = torch.where(earlier, again, codes).transpose(1, 2)
        codes[run, off] = _code(x, scale[run][:, :, None], cache)
        # (pages behind the last run are the last token's: written once more, with what they hold)
        same = torch.where(used, i, run[-1])
        pool[pid] = codes[same].transpose(1, 2)
        s["scales"][pid, :, which] = scale[same]


def _run_attend(s):
    case, lens, starts = s["case"], s["lens"].long(), s["starts"].long()
    b, hq, hkv, d, page = (case[n] for n in ("batch", "query_heads", "kv_heads", "head_dim", "page"))
    g, r = hq // hkv, int(case["chunk"] and max(case["chunk"], case["rows"]) or case["rows"])
    per = s["table"].shape[1]
    at = s["table"].long().clamp(min=0)
    k = _value(s["k"][at], case["cache"]) * s["scales"][at][..., 0, None, None]        # [B][per][Hkv][page][D]
    k = k.permute(0, 2, 4, 1, 3).reshape(b, hkv, d, per * page)
    v = _value(s["v"][at], case["cache"]) * s["scales"][at][..., 1, None, None]        # [B][per][Hkv][D][page]
    v = v.permute(0, 2, 1, 4, 3).reshape(b, hkv, per * page, d)
    rows = starts[1:] - starts[:-1]
    i = torch.arange(r, device="cuda")
    q = s["q"][(starts[:-1, None] + i).clamp(max=s["total"] - 1)].float()              # [B][r][Hq][D]
    q = q.reshape(b, r, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b, hkv, g * r, d)
    x = torch.matmul(q, k).reshape(b, hkv, g, r, per * page) / math.sqrt(d)
    seen = torch.arange(per * page, device="cuda") <= (lens - rows)[:, None, None] + i[None, :, None]
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x = torch.exp(x.sub_(x.amax(-1, keepdim=True)))
    out = torch.matmul((x / x.sum(-1, keepdim=True)).reshape(b, hkv, g * r, per * page), v)
    out = out.reshape(b, hkv, g, r, d).permute(0, 3, 1, 2, 4).reshape(b, r, hq, d)
    t = torch.arange(s["total"], device="cuda")
    n = torch.searchsorted(starts[1:], t, right=True)
    s["out"].copy_(out[n, t - starts[n]])


def run(s):
    if own:
        return _run_own(s)
    {"plan": _run_plan, "rotate": _run_rotate, "append": _run_append, "attend": _run_attend}[s["case"]["kind"]](s)
    return _outputs(s)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind, (hq, hkv, d) = case["kind"], (case[n] for n in ("query_heads", "kv_heads", "head_dim"))
    e = 4 if case["dtype"] == "f32" else 2
    if kind == "rotate":
        n = int(d * case["part"]) // 2
        return {"bytes": case["tokens"] * (2 * (hq + hkv) * d * e + 4) + 8 * n, "flops": case["tokens"] * (hq + hkv) * n * 6}
    rows, lens, page = _rows(case), _lengths(case), case["page"]
    t = int(rows.sum())
    if kind == "plan":
        pages = int((-(-lens // page) - -(-(lens - rows) // page)).sum())
        return {"bytes": case["batch"] * 24 + t * 12 + pages * 8, "flops": 0}
    if kind == "append":
        pages = int((-(-lens // page) - (lens - rows) // page).sum())
        return {"bytes": t * (2 * hkv * d * (e + 1) + 8) + pages * hkv * 8, "flops": 4 * t * hkv * d}
    pages = int((-(-lens // page)).sum())
    pairs = int((rows * (lens - rows) + rows * (rows + 1) // 2).sum())
    return {"bytes": int(lens.sum()) * hkv * 2 * d + pages * (8 * hkv + 4) + 2 * t * hq * d * e, "flops": 4.0 * pairs * hq * d}


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_plan(s):
    """Sequence by sequence on the host: release, then grant from the top of the stack."""
    case, page = s["case"], s["case"]["page"]
    lens, keep, counts, stack = (s[n].tolist() for n in ("lens", "keep", "counts", "free"))
    count, table, per = int(s["free_count"]), s["table"].cpu().numpy().copy(), s["table"].shape[1]
    for b in range(case["batch"]):
        keep[b] = min(max(keep[b], 0), lens[b])
        for p in range(-(-lens[b] // page) - 1, -(-keep[b] // page) - 1, -1):
            stack[count], count, table[b, p] = int(table[b, p]), count + 1, -1
    asked, rows, left, starts, positions, slots = 0, 0, count, [0], [], []
    for b in range(case["batch"]):
        n = max(counts[b], 0)
        n = n if keep[b] + n <= per * page else 0
        first, end = -(-keep[b] // page), -(-(keep[b] + n) // page)
        asked, rows = asked + end - first, rows + n
        if (end > first and asked > left) or rows > s["total"]:
            n, end = 0, first
        for p in range(first, end):
            count -= 1
            table[b, p] = stack[count]
        for pos in range(keep[b], keep[b] + n):
            positions.append(pos)
            slots.append(int(table[b, pos // page]) * page + pos % page)
        lens[b] = keep[b] + n
        starts.append(starts[-1] + n)
    pad = [-1] * (s["total"] - len(slots))
    return {"table": torch.from_numpy(table), "lens": torch.tensor(lens, dtype=torch.int32),
            "free": torch.tensor(stack, dtype=torch.int32), "free_count": torch.tensor([count], dtype=torch.int32),
            "starts": torch.tensor(starts, dtype=torch.int32), "positions": torch.tensor(positions + pad, dtype=torch.int32),
            "slots": torch.tensor(slots + pad, dtype=torch.int64)}


def _exact_rotate(s):
    """Each pair as a complex number, times e^(i angle)."""
    case, n = s["case"], s["w"].numel()
    z = torch.polar(torch.full((case["tokens"], 1, n), s["magnitude"], dtype=torch.float64, device="cuda"),
                    (s["positions"].double()[:, None] * s["w"])[:, None])
    found = {}
    for name in ("q", "k"):
        x = s[name].double()
        if case["layout"] == "half":
            y = torch.complex(x[..., :n], x[..., n: 2 * n]) * z
            y = torch.cat((y.real, y.imag), 2)
        else:
            y = torch.view_as_real(torch.view_as_complex(x[..., : 2 * n].reshape(*x.shape[:2], n, 2)) * z).flatten(2)
        found[name + "_out"] = torch.cat((y, x[..., 2 * n:]), 2)
    return found


def _exact_append(s):
    """The scales alone (the codes are whole numbers): page by page on the host."""
    case, page = s["case"], s["case"]["page"]
    scales = s["scales"].double().cpu().numpy()
    top = np.stack([s[n].double().abs().amax(2).cpu().numpy() for n in ("keys", "values")], 2)
    begun = set()
    for i, slot in enumerate(s["slots"].tolist()):
        p = slot // page
        if p not in begun and slot % page == 0:
            scales[p] = 0.0
        begun.add(p)
        scales[p] = np.maximum(scales[p], top[i] / MOST[case["cache"]])
    return {"k": None, "v": None, "scales": torch.from_numpy(scales)}


def _exact_attend(s):
    case = s["case"]
    hq, hkv, d, page = (case[n] for n in ("query_heads", "kv_heads", "head_dim", "page"))
    g = hq // hkv
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    starts, lens = s["starts"].tolist(), s["lens"].tolist()
    for b in range(case["batch"]):
        t0, t1, n = starts[b], starts[b + 1], lens[b]
        pages = s["table"][b, : -(-n // page)].long()
        sk, sv = (s["scales"][pages, :, i].double()[:, :, None, None] for i in (0, 1))
        k = (_value(s["k"][pages], case["cache"]).double() * sk).transpose(0, 1).reshape(hkv, -1, d)[:, :n]
        v = (_value(s["v"][pages], case["cache"]).double() * sv).permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :n]
        hidden = torch.arange(n, device="cuda")[None] > n - (t1 - t0) + torch.arange(t1 - t0, device="cuda")[:, None]
        for h in range(hq):
            x = (s["q"][t0:t1, h].double() @ k[h // g].T) * d ** -0.5
            out[t0:t1, h] = torch.softmax(x.masked_fill_(hidden, -math.inf), 1) @ v[h // g]
    return {"out": out}


def exact(case, seed):
    return {"plan": _exact_plan, "rotate": _exact_rotate, "append": _exact_append, "attend": _exact_attend}[case["kind"]](_inputs(case, seed))
