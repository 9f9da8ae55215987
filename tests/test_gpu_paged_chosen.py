"""Tree attention, attention with accumulated weights, token selection, compaction, page bounds and sparse
attention over a paged cache (GPU only), through the C ABI, against 64-bit results on the host.

What no row may see (drafts off a row's path, tokens past a sequence's end, pages of no table) holds NaN and
infinities throughout.  Bounds of the errors: tests/_paged_chosen.py.  Selections, moves and bounds are exact.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

import oracle
from schedforge_amd import _abi
from schedforge_amd._abi import BF16, F32

from _helpers import KEEP_ALIVE, dev, host, stream
from _paged_chosen import (Cache, ancestors, attend, close, output, queries, random_tree, ref_rows, value, words,
                           workspace)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def run_tree(lib, c, qd, qt, mask, stride, out, ot, longest, splits=0, lens=True, ws=None):
    a = c.args(qd, out, qt, ot, longest, splits, lens)
    n = lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(a))
    ws = workspace(n) if ws is None else ws
    _abi.check(lib.sfg_hip_attn_tree_v1(ctypes.byref(a), mask.data_ptr(), stride, ws.data_ptr(), ws.numel(), stream()))


# (q heads, kv heads, D, page tokens, nodes, lengths, splits, q offset)
TREES = [
    (4, 4, 128, 16, 1, (33, 0, 1), 0, 0),            # one node; a sequence with nothing committed
    (8, 2, 128, 16, 8, (900, 0, 15, 16, 17), 0, 0),
    (8, 2, 64, 16, 5, (300, 31, 1), 3, 0),
    (4, 1, 128, 16, 33, (257, 0, 100), 0, 0),        # two mask words
    (16, 4, 64, 16, 64, (150, 3), 0, 0),             # 256 columns
    (3, 1, 64, 16, 13, (77, 48), 0, 0),
    (34, 2, 128, 16, 3, (40, 200), 0, 0),            # a group of 17
    (6, 3, 80, 16, 7, (50, 0, 129), 0, 0),           # head dims of the general kernel
    (2, 1, 33, 5, 9, (23, 64), 2, 0),
    (4, 2, 256, 16, 4, (70, 1), 40, 0),              # more splits than pages
    (4, 2, 128, 8, 6, (61, 8), 0, 0),                # 8-token pages
    (8, 2, 128, 16, 6, (64, 90), 0, 1),              # a query off its boundary
]


@pytest.mark.parametrize("types", ["bf16/bf16/bf16", "bf16/bf16/f32", "f32/bf16/f32", "f32/f32/f32", "bf16/f32/bf16"])
@pytest.mark.parametrize("hq,hkv,d,pt,t,lens,splits,offset", TREES)
def test_tree_attention(hq, hkv, d, pt, t, lens, splits, offset, types):
    lib = _abi.load()
    qt, kt, ot = types.split("/")
    rng = np.random.default_rng(hq * 31 + d + t)
    longest = max(lens)
    c = Cache(rng, lens, longest + t, hkv, d, pt, kt)
    bits = ancestors(random_tree(rng, c.b, t))
    q, qd, qdt = queries(rng, c.b, hq, t, d, qt, offset=offset)
    out, odt = output(q.shape, ot)
    # a draft that only its own subtree sees holds what the others must not meet
    hidden = t - 1
    c.upload(c.lens + t)
    if t > 1 and not bits[:, : t - 1, hidden].any():
        for n in range(c.b):
            pos = int(c.lens[n]) + hidden
            pg, at = int(c.table[n, pos // pt]), pos % pt
            bad = torch.tensor([float("inf"), float("nan")], device="cuda")
            v = c.vd.view(torch.bfloat16) if kt == "bf16" else c.vd
            v[pg, :, 0::2, at], v[pg, :, 1::2, at] = bad[0].to(v.dtype), bad[1].to(v.dtype)
            k = c.kd.view(torch.bfloat16) if kt == "bf16" else c.kd
            k[pg, :, at, :] = bad[1].to(k.dtype)
    run_tree(lib, c, qd, qdt, dev(words(bits)), t * -(-t // 32), out, odt, longest, splits)

    def see(n, h, i):
        s = np.arange(c.per * pt) < c.lens[n]
        s[c.lens[n]: c.lens[n] + t] = bits[n, i]
        return s
    ref, _, err, _ = ref_rows(c, q, see, types == "bf16/bf16/bf16", ot == "bf16")
    got = value(out)
    rows = slice(0, hidden) if t > 1 else slice(0, t)
    close(got[:, :, rows], ref[:, :, rows], err[:, :, rows], "tree")
    if t > 1:
        assert np.isnan(got[:, :, hidden]).any() or hidden == 0  # the row that sees it does meet it


def test_tree_of_one_mask_for_all_and_rows_that_see_nothing():
    """mask_stride 0; a row whose bits are clear sees the committed tokens alone, and nothing where there are none."""
    lib = _abi.load()
    rng = np.random.default_rng(5)
    for d, pt in ((128, 16), (40, 16)):
        c = Cache(rng, (0, 37), 60, 2, d, pt).upload((4, 41))
        bits = np.tril(np.ones((1, 4, 4), bool))
        bits[0, 2] = False
        q, qd, qdt = queries(rng, 2, 4, 4, d, "bf16")
        out, odt = output(q.shape, "f32")
        run_tree(lib, c, qd, qdt, dev(words(bits)), 0, out, odt, 37)

        def see(n, h, i):
            s = np.arange(c.per * pt) < c.lens[n]
            s[c.lens[n]: c.lens[n] + 4] = bits[0, i]
            return s
        ref, _, err, _ = ref_rows(c, q, see, False, False)
        assert np.isnan(ref[0, :, 2]).all()
        close(value(out), ref, err, f"shared mask D {d}")


@pytest.mark.parametrize("d,pt", [(128, 16), (64, 16), (48, 16)])
def test_bad_pages_and_lengths_are_not_followed(d, pt):
    """Page ids outside the pool hide their tokens; lengths outside [0, max_context] are clamped."""
    lib = _abi.load()
    rng = np.random.default_rng(d)
    c = Cache(rng, (100, 90, 64), 128, 2, d, pt).upload((104, 94, 68))
    table = c.table.copy()
    table[0, 1], table[1, 0], table[2, :] = -1, c.pages, 1 << 30
    c.td, c.ld = dev(table), dev(np.array([1000, -5, 64], np.int32))
    lens = np.array([100, 0, 64])
    bits = ancestors(random_tree(rng, 3, 4))
    q, qd, qdt = queries(rng, 3, 4, 4, d, "f32")
    out, odt = output(q.shape, "f32")
    # the second sequence's drafts are where its clamped length puts them
    run_tree(lib, c, qd, qdt, dev(words(bits)), 4, out, odt, 100)

    def see(n, h, i):
        s = np.arange(c.per * pt) < lens[n]
        s[lens[n]: lens[n] + 4] = bits[n, i]
        ok = (table[n] >= 0) & (table[n] < c.pages)
        return s & np.repeat(ok, pt)
    ref, _, err, _ = ref_rows(c, q, see, False, False)
    close(value(out), ref, err, "bad pages")


@pytest.mark.parametrize("kt", ["bf16", "f32"])
def test_visible_infinities_give_the_reference_result(kt):
    """An infinite value that every row sees makes that output dim infinite, an infinite key the row NaN or
    its value, as the formula in 64 bits has it; the other rows and sequences are finite."""
    lib = _abi.load()
    rng = np.random.default_rng(11)
    for qt, ot in (("bf16", "bf16"), ("f32", "f32")):
        c = Cache(rng, (70, 60), 90, 2, 128, 16, kt)
        c.v[0, 1, 33, 5] = np.inf
        c.v[0, 1, 40, 9] = -np.inf
        c.upload((73, 63))
        bits = ancestors(random_tree(rng, 2, 3))
        q, qd, qdt = queries(rng, 2, 4, 3, 128, qt)
        out, odt = output(q.shape, ot)
        run_tree(lib, c, qd, qdt, dev(words(bits)), 3, out, odt, 70)
        got = value(out)
        assert (got[0, 2:, :, 5] == np.inf).all() and (got[0, 2:, :, 9] == -np.inf).all()
        got[0, 2:, :, [5, 9]] = 0.0
        assert np.isfinite(got).all()


# (q heads, kv heads, D, page tokens, rows, lengths, splits)
WEIGHTS = [(8, 2, 128, 16, 1, (900, 0, 1, 16, 17), 0), (4, 4, 64, 16, 1, (300,), 3), (16, 4, 128, 16, 4, (257, 4, 3, 0), 0),
           (34, 2, 64, 16, 3, (40, 100), 0), (6, 3, 80, 16, 2, (50, 129), 0), (2, 1, 33, 5, 1, (23, 64), 9),
           (4, 1, 128, 16, 30, (60, 33), 0), (4, 2, 128, 8, 1, (61, 8), 0)]


@pytest.mark.parametrize("types", ["bf16/bf16/bf16", "f32/bf16/f32", "f32/f32/f32"])
@pytest.mark.parametrize("hq,hkv,d,pt,rows,lens,splits", WEIGHTS)
def test_attention_with_accumulated_weights(hq, hkv, d, pt, rows, lens, splits, types):
    """Two calls: the second adds to what the first left.  Entries past a sequence's end stay as they were."""
    lib = _abi.load()
    qt, kt, ot = types.split("/")
    rng = np.random.default_rng(hq + d + rows)
    longest = max(lens)
    c = Cache(rng, lens, longest, hkv, d, pt, kt).upload(lens)
    ld = longest + 3
    w0 = rng.uniform(0.0, 2.0, (c.b, hkv, ld)).astype(np.float32)
    wd = dev(w0)
    want, tol = w0.astype(np.float64), np.zeros(w0.shape)

    def see(n, h, i):
        return np.arange(c.per * pt) < c.lens[n] - rows + i + 1
    for _ in range(2):
        q, qd, qdt = queries(rng, c.b, hq, rows, d, qt)
        out, odt = output(q.shape, ot)
        a = c.args(qd, out, qdt, odt, longest, splits)
        ws = workspace(lib.sfg_hip_attn_weights_workspace_v1(ctypes.byref(a)))
        _abi.check(lib.sfg_hip_attn_weights_v1(ctypes.byref(a), wd.data_ptr(), ld, ws.data_ptr(), ws.numel(), stream()))
        ref, w, err, rel = ref_rows(c, q, see, types == "bf16/bf16/bf16", ot == "bf16")
        close(value(out), ref, err, "out")
        add = w.reshape(c.b, hkv, hq // hkv, rows, -1)[..., :longest]
        r = rel.reshape(c.b, hkv, hq // hkv, rows)
        want[..., :longest] += add.sum((2, 3))
        # each weight's own error, their sum's, and the accumulation's
        tol[..., :longest] += (add * r[..., None]).sum((2, 3)) + (hq // hkv * rows + 1) * 2.0 ** -24 * want[..., :longest]
    got = host(wd)
    for n in range(c.b):
        np.testing.assert_array_equal(got[n, :, c.lens[n]:], w0[n, :, c.lens[n]:])
    assert (np.abs(got - want) <= tol + 1e-30).all(), (np.abs(got - want) / (tol + 1e-30)).max()


def keep_reference(w, length, budget, recent):
    """Positions kept of one row of weights, by sorting (value descending, position ascending); NaN lowest."""
    if length <= budget:
        return np.arange(length)
    old = length - recent
    key = np.where(np.isnan(w[:old]), -np.inf, w[:old]) + 0.0
    nan_last = np.isnan(w[:old])
    order = np.lexsort((np.arange(old), nan_last, -key))[: budget - recent]
    return np.concatenate((np.sort(order), np.arange(old, length)))


def weights_of(rng, kind, shape):
    if kind == "heavy":
        return np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        return rng.integers(0, 3, shape).astype(np.float32)
    if kind == "equal":
        return np.full(shape, 0.25, np.float32)
    w = rng.standard_normal(shape).astype(np.float32)  # signs, both zeros, infinities, NaN, denormals
    flat = w.reshape(-1)
    for i, v in enumerate((np.inf, -np.inf, np.nan, 0.0, -0.0, 1e-42, -1e-42, -np.nan)):
        flat[i::17] = v
    return w


@pytest.mark.parametrize("kind", ["heavy", "ties", "equal", "odd"])
@pytest.mark.parametrize("lens,budget,recent", [
    ((1, 0, 2, 3), 1, 0), ((1, 0, 2, 3), 2, 2), ((100, 64, 65, 63), 64, 7), ((1500, 1024, 1025), 1024, 128),
    ((5000, 4097, 40), 33, 33), ((9000, 2049), 2048, 1), ((2048, 1024), 1023, 0), ((20000,), 17777, 5)])
def test_token_selection(lens, budget, recent, kind):
    lib = _abi.load()
    rng = np.random.default_rng(budget + len(kind))
    b, hkv, longest = len(lens), 3, max(lens)
    ld = longest + 2
    w = weights_of(rng, kind, (b, hkv, ld))
    for inplace in (False, True, None):
        wd = dev(w)
        kept = wd if inplace else torch.full((b, hkv, ld), 5.0, device="cuda")
        keep = torch.full((b, hkv, budget), 99, dtype=torch.int32, device="cuda")
        counts = torch.full((b,), 99, dtype=torch.int32, device="cuda")
        _abi.check(lib.sfg_hip_kv_select_v1(wd.data_ptr(), ld, dev(np.array(lens, np.int32)).data_ptr(), longest, budget, recent,
                                            keep.data_ptr(), counts.data_ptr(), None if inplace is None else kept.data_ptr(),
                                            b, hkv, stream()))
        got, n_got, k_got = host(keep), host(counts), host(kept)
        for n in range(b):
            assert n_got[n] == min(lens[n], budget)
            for h in range(hkv):
                ref = keep_reference(w[n, h], lens[n], budget, recent)
                np.testing.assert_array_equal(got[n, h, : ref.size], ref)
                assert (got[n, h, ref.size:] == -1).all()
                if inplace is not None:
                    np.testing.assert_array_equal(k_got[n, h, : ref.size], w[n, h, ref])
                    assert (k_got[n, h, ref.size:] == 0).all()
        if not inplace:
            np.testing.assert_array_equal(host(wd), w)


def compact(lib, c, kd, vd, base, keep, counts, new, max_keep=None):
    keep_heads, ld = keep.shape[1], keep.shape[2]
    _abi.check(lib.sfg_hip_kv_compact_v1(
        kd.data_ptr(), vd.data_ptr(), BF16 if c.dtype == "bf16" else F32, c.td.data_ptr(), None if base is None else base.data_ptr(),
        keep.data_ptr(), keep_heads, ld, counts.data_ptr(), new.data_ptr(), ld if max_keep is None else max_keep, c.b, c.hkv,
        c.d, c.pt, c.per, c.pages, stream()))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,pt,longest,n", [(128, 16, 700, 300), (64, 16, 90, 89), (128, 16, 1300, 1299), (80, 16, 200, 64),
                                            (33, 5, 64, 20), (256, 8, 100, 1), (1, 1, 9, 4), (128, 16, 5000, 2048)])
def test_compaction_per_head(d, pt, longest, n, dtype):
    """Every head keeps tokens of its own, in place; what is not a destination stays."""
    lib = _abi.load()
    rng = np.random.default_rng(n + d)
    lens = np.array([longest, max(n, longest // 2)], np.int32)
    c = Cache(rng, lens, longest, 2, d, pt, dtype, poison=False).upload(lens)
    keep = np.full((2, 2, n + 3), -7, np.int32)
    counts = np.array([n, n // 2], np.int32)
    for b in range(2):
        for h in range(2):
            keep[b, h, : counts[b]] = np.sort(rng.permutation(int(lens[b]))[: counts[b]])
    new = torch.zeros(2, dtype=torch.int32, device="cuda")
    compact(lib, c, c.kd, c.vd, None, dev(keep), dev(counts), new)
    k, v = c.logical(c.kd, c.vd)
    for b in range(2):
        for h in range(2):
            m = counts[b]
            for got, was in ((k, c.k), (v, c.v)):
                np.testing.assert_array_equal(got[b, h, :m], was[b, h, keep[b, h, :m]])
                np.testing.assert_array_equal(got[b, h, m:], was[b, h, m:])
    np.testing.assert_array_equal(host(new), counts)


@pytest.mark.parametrize("alias", ["none", "base", "counts"])
@pytest.mark.parametrize("d,pt", [(128, 16), (64, 16), (24, 4)])
def test_accepted_path_moves_behind_the_committed_tokens(d, pt, alias):
    lib = _abi.load()
    rng = np.random.default_rng(d)
    t, lens = 40, np.array([100, 0, 37, 31], np.int32)
    c = Cache(rng, lens, 100 + t, 3, d, pt, poison=False).upload(lens)
    keep = np.full((4, 1, t), -1, np.int32)
    counts = np.array([9, 40, 0, 1], np.int32)
    for b in range(4):
        keep[b, 0, : counts[b]] = np.sort(rng.permutation(t)[: counts[b]])
    base, cd = dev(lens), dev(counts)
    new = {"none": torch.zeros(4, dtype=torch.int32, device="cuda"), "base": base, "counts": cd}[alias]
    compact(lib, c, c.kd, c.vd, base, dev(keep), cd, new)
    k, v = c.logical(c.kd, c.vd)
    for b in range(4):
        at, m = lens[b], counts[b]
        for got, was in ((k, c.k), (v, c.v)):
            np.testing.assert_array_equal(got[b, :, at: at + m], was[b][:, at + keep[b, 0, :m]])
            np.testing.assert_array_equal(got[b, :, :at], was[b, :, :at])
            np.testing.assert_array_equal(got[b, :, at + m:], was[b, :, at + m:])
    np.testing.assert_array_equal(host(new), lens + counts)


def test_compaction_skips_what_names_no_token():
    """Entries below their index, past the capacity or negative, pages outside the pool, counts and bases
    out of range: nothing is moved for them and nothing outside is touched."""
    lib = _abi.load()
    rng = np.random.default_rng(3)
    for d, pt in ((128, 16), (20, 4)):
        c = Cache(rng, (64, 64, 64), 64, 2, d, pt, poison=False).upload((64, 64, 64))
        table = c.table.copy()
        table[1, 0], table[1, 2] = -3, c.pages + 4
        c.td = dev(table)
        keep = np.tile(np.array([0, 9, 1, 64, -1, 1 << 30, 8, 7, 40, 63], np.int32), (3, 1, 1))
        counts, base = dev(np.array([99, 10, -4], np.int32)), dev(np.array([0, 0, 1 << 30], np.int32))
        new = torch.zeros(3, dtype=torch.int32, device="cuda")
        compact(lib, c, c.kd, c.vd, base, dev(keep), counts, new)
        k, v = c.logical(c.kd, c.vd)
        ref_k, ref_v = c.k.copy(), c.v.copy()
        ok = (table >= 0) & (table < c.pages)
        for b in range(2):
            for i, s in enumerate(keep[b, 0]):
                if s > i and s < 64 and ok[b, s // pt] and ok[b, i // pt]:
                    ref_k[b, :, i], ref_v[b, :, i] = c.k[b, :, s], c.v[b, :, s]
        np.testing.assert_array_equal(k, ref_k)
        np.testing.assert_array_equal(v, ref_v)
        np.testing.assert_array_equal(host(new), [10, 10, c.per * pt])


def bounds_reference(c, lens, fresh, before):
    out = before.copy()
    for n in range(c.b):
        for p in range(-(-int(lens[n]) // c.pt)):
            end = min((p + 1) * c.pt, int(lens[n]))
            if (p + 1) * c.pt <= lens[n] - fresh:
                continue
            t = c.k[n, :, p * c.pt: end]
            out[c.table[n, p], :, 0], out[c.table[n, p], :, 1] = t.min(1), t.max(1)
    return out


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d,pt", [(128, 16), (64, 16), (80, 16), (33, 5), (256, 3)])
def test_page_bounds(d, pt, dtype):
    lib = _abi.load()
    rng = np.random.default_rng(d)
    lens = np.array([200, 0, 1, 16, 17, 199], np.int32)
    c = Cache(rng, lens, 200, 3, d, pt, dtype).upload(lens)
    tdt = torch.bfloat16 if dtype == "bf16" else torch.float32
    for fresh in (1, 2, 16, 17, 40, 200, 10 ** 6):
        before = oracle.round_bf16(rng.standard_normal((c.pages, 3, 2, d)).astype(np.float32))
        bd = torch.from_numpy(before).to(tdt).cuda()
        _abi.check(lib.sfg_hip_kv_page_bounds_v1(c.kd.data_ptr(), BF16 if dtype == "bf16" else F32, c.td.data_ptr(),
                                                 c.ld.data_ptr(), 200, fresh, bd.data_ptr(), c.b, 3, d, pt, c.per, c.pages,
                                                 stream()))
        np.testing.assert_array_equal(value(bd), bounds_reference(c, lens, fresh, before), err_msg=str(fresh))


# (q heads, kv heads, D, page tokens, rows, lengths, top, sink, recent, splits)
SPARSE = [
    (8, 2, 128, 16, 1, (900, 0, 1, 16, 17, 130), 8, 1, 1, 0),
    (4, 4, 64, 16, 1, (1300, 333), 3, 0, 0, 0),
    (16, 4, 128, 16, 3, (700, 3, 2, 65), 5, 2, 2, 2),
    (34, 2, 64, 16, 2, (400, 90), 4, 0, 1, 0),
    (6, 3, 80, 16, 1, (500, 129), 6, 1, 1, 0),
    (2, 1, 33, 5, 2, (123, 64), 7, 1, 3, 9),
    (4, 2, 128, 16, 1, (300, 20), 64, 1, 2, 0),      # more than there are
    (4, 2, 128, 8, 1, (461, 8), 1, 0, 1, 0),
    (4, 1, 128, 16, 1, (40000, 17000), 40, 1, 2, 0),  # more pages than a workgroup has threads
]


@pytest.mark.parametrize("types", ["bf16/bf16/bf16", "f32/bf16/f32", "f32/f32/f32"])
@pytest.mark.parametrize("hq,hkv,d,pt,rows,lens,top,sink,recent,splits", SPARSE)
def test_sparse_attention(hq, hkv, d, pt, rows, lens, top, sink, recent, splits, types):
    lib = _abi.load()
    qt, kt, ot = types.split("/")
    rng = np.random.default_rng(hq + d + top)
    longest = max(lens)
    c = Cache(rng, lens, longest, hkv, d, pt, kt).upload(lens)
    tdt = torch.bfloat16 if kt == "bf16" else torch.float32
    bd = torch.zeros((c.pages, hkv, 2, d), dtype=tdt, device="cuda")
    _abi.check(lib.sfg_hip_kv_page_bounds_v1(c.kd.data_ptr(), BF16 if kt == "bf16" else F32, c.td.data_ptr(), c.ld.data_ptr(),
                                             longest, longest, bd.data_ptr(), c.b, hkv, d, pt, c.per, c.pages, stream()))
    bounds = value(bd).astype(np.float64)
    q, qd, qdt = queries(rng, c.b, hq, rows, d, qt)
    out, odt = output(q.shape, ot)
    sel = torch.full((c.b, rows, hkv, top), 77, dtype=torch.int32, device="cuda")
    a = c.args(qd, out, qdt, odt, longest, splits)
    ws = workspace(lib.sfg_hip_attn_sparse_workspace_v1(ctypes.byref(a), top))
    _abi.check(lib.sfg_hip_attn_sparse_v1(ctypes.byref(a), bd.data_ptr(), top, sink, recent, sel.data_ptr(), ws.data_ptr(),
                                          ws.numel(), stream()))
    got_sel, g = host(sel), hq // hkv
    want = np.full((c.b, rows, hkv, top), -1)
    for n in range(c.b):
        for i in range(rows):
            pages = -(-max(int(c.lens[n]) - rows + i + 1, 0) // pt)
            for h in range(hkv):
                bd_n = bounds[c.table[n, :pages], h]
                qg = q[n, h * g: (h + 1) * g, i].astype(np.float64)
                score = np.zeros(pages)
                for x in qg:
                    score += np.maximum(x * bd_n[:, 0], x * bd_n[:, 1]).sum(1)
                first = set(range(min(sink, pages))) | set(range(max(0, pages - recent), pages))
                rest = [p for p in np.lexsort((np.arange(pages), -score)) if p not in first]
                take = sorted(first | set(rest[: top - len(first)]))
                want[n, i, h, : len(take)] = take
    np.testing.assert_array_equal(got_sel, want)

    def see(n, h, i):
        end = int(c.lens[n]) - rows + i + 1
        s = np.zeros(c.per * pt, bool)
        for p in want[n, i, h // g]:
            if p >= 0:
                s[p * pt: min((p + 1) * pt, end)] = True
        return s
    ref, _, err, _ = ref_rows(c, q, see, types == "bf16/bf16/bf16", ot == "bf16")
    close(value(out), ref, err, "sparse")


def test_equal_scores_take_the_lower_pages():
    """Every page holds the same keys: ties everywhere, behind the forced pages."""
    lib = _abi.load()
    rng = np.random.default_rng(8)
    c = Cache(rng, (640,), 640, 2, 64, 16)
    c.k[:] = np.tile(c.k[:, :, :16], (1, 1, 40, 1))
    c.upload((640,))
    bd = torch.zeros((c.pages, 2, 2, 64), dtype=torch.bfloat16, device="cuda")
    _abi.check(lib.sfg_hip_kv_page_bounds_v1(c.kd.data_ptr(), BF16, c.td.data_ptr(), None, 640, 640, bd.data_ptr(), 1, 2, 64, 16,
                                             c.per, c.pages, stream()))
    q, qd, qdt = queries(rng, 1, 4, 1, 64, "bf16")
    out, odt = output(q.shape, "bf16")
    sel = torch.zeros((1, 1, 2, 9), dtype=torch.int32, device="cuda")
    a = c.args(qd, out, qdt, odt, 640, lens=False)
    ws = workspace(lib.sfg_hip_attn_sparse_workspace_v1(ctypes.byref(a), 9))
    _abi.check(lib.sfg_hip_attn_sparse_v1(ctypes.byref(a), bd.data_ptr(), 9, 0, 2, sel.data_ptr(), ws.data_ptr(), ws.numel(), stream()))
    np.testing.assert_array_equal(host(sel), np.tile([0, 1, 2, 3, 4, 5, 6, 38, 39], (1, 1, 2, 1)))


def test_captured_calls_replay_like_eager_ones():
    """Every operator captured into one graph, replayed with eager work between: the same bits each time."""
    lib = _abi.load()
    rng = np.random.default_rng(21)
    b, hq, hkv, d, longest, t, top, budget = 3, 8, 2, 128, 500, 6, 7, 200
    c = Cache(rng, (500, 44, 333), longest + t, hkv, d).upload((506, 50, 339))
    q, qd, qdt = queries(rng, b, hq, t, d, "bf16")
    q1, q1d, _ = queries(rng, b, hq, 1, d, "bf16")
    mask = dev(words(ancestors(random_tree(rng, b, t))))
    wd = dev(rng.uniform(0, 1, (b, hkv, longest)).astype(np.float32))
    w0 = wd.clone()
    bd = torch.zeros((c.pages, hkv, 2, d), dtype=torch.bfloat16, device="cuda")
    keep = torch.zeros((b, hkv, budget), dtype=torch.int32, device="cuda")
    counts, kept = torch.zeros(b, dtype=torch.int32, device="cuda"), torch.zeros_like(wd)
    new = torch.zeros(b, dtype=torch.int32, device="cuda")
    sel = torch.zeros((b, 1, hkv, top), dtype=torch.int32, device="cuda")
    k0, v0 = c.kd.clone(), c.vd.clone()
    outs = [output(q.shape, "bf16")[0], output(q1.shape, "bf16")[0], output(q1.shape, "bf16")[0]]
    args = [c.args(qd, outs[0], BF16, BF16, longest), c.args(q1d, outs[1], BF16, BF16, longest), c.args(q1d, outs[2], BF16, BF16, longest)]
    ws = [workspace(lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(args[0]))),
          workspace(lib.sfg_hip_attn_weights_workspace_v1(ctypes.byref(args[1]))),
          workspace(lib.sfg_hip_attn_sparse_workspace_v1(ctypes.byref(args[2]), top))]

    def all_calls():
        s = stream()
        c.kd.copy_(k0)
        c.vd.copy_(v0)
        wd.copy_(w0)
        _abi.check(lib.sfg_hip_attn_tree_v1(ctypes.byref(args[0]), mask.data_ptr(), t, ws[0].data_ptr(), ws[0].numel(), s))
        _abi.check(lib.sfg_hip_attn_weights_v1(ctypes.byref(args[1]), wd.data_ptr(), longest, ws[1].data_ptr(), ws[1].numel(), s))
        _abi.check(lib.sfg_hip_kv_page_bounds_v1(c.kd.data_ptr(), BF16, c.td.data_ptr(), c.ld.data_ptr(), longest, longest,
                                                 bd.data_ptr(), b, hkv, d, 16, c.per, c.pages, s))
        _abi.check(lib.sfg_hip_attn_sparse_v1(ctypes.byref(args[2]), bd.data_ptr(), top, 1, 1, sel.data_ptr(), ws[2].data_ptr(),
                                              ws[2].numel(), s))
        _abi.check(lib.sfg_hip_kv_select_v1(wd.data_ptr(), longest, c.ld.data_ptr(), longest, budget, 9, keep.data_ptr(),
                                            counts.data_ptr(), kept.data_ptr(), b, hkv, s))
        _abi.check(lib.sfg_hip_kv_compact_v1(c.kd.data_ptr(), c.vd.data_ptr(), BF16, c.td.data_ptr(), None, keep.data_ptr(), hkv,
                                             budget, counts.data_ptr(), new.data_ptr(), budget, b, hkv, d, 16, c.per, c.pages, s))

    state = [c.kd, c.vd, wd, bd, keep, counts, kept, new, sel, *outs]
    all_calls()
    torch.cuda.synchronize()
    want = [x.clone() for x in state]
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            all_calls()
    for _ in range(4):
        for x in state:
            x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for x, y in zip(state, want):
            assert torch.equal(x.view(torch.int16) if x.dtype == torch.bfloat16 else x,
                               y.view(torch.int16) if y.dtype == torch.bfloat16 else y)
        all_calls()  # eager between
        torch.cuda.synchronize()
        assert torch.equal(outs[0].view(torch.int16), want[-3].view(torch.int16))


def test_two_streams_with_workspaces_of_their_own():
    lib = _abi.load()
    rng = np.random.default_rng(22)
    c = Cache(rng, (900, 500), 920, 2, 128).upload((910, 510))
    mask = dev(words(ancestors(random_tree(rng, 2, 10))))
    q, qd, qdt = queries(rng, 2, 8, 10, 128, "bf16")
    q2, q2d, _ = queries(rng, 2, 8, 10, 128, "bf16")
    alone = []
    for x in (qd, q2d):
        out, odt = output(q.shape, "bf16")
        run_tree(lib, c, x, qdt, mask, 10, out, odt, 900)
        alone.append(out)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [output(q.shape, "bf16")[0] for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, x, o in zip(streams, (qd, q2d), outs):
            with torch.cuda.stream(s):
                run_tree(lib, c, x, qdt, mask, 10, o, BF16, 900)
    torch.cuda.synchronize()
    for o, w in zip(outs, alone):
        assert torch.equal(o.view(torch.int16), w.view(torch.int16))


@pytest.mark.parametrize("src", ["bf16", "f32"])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("d", [128, 24])
def test_several_tokens_appended_by_pages(d, dtype, src):
    """Runs of tokens that start and end inside pages, at lengths of their own (a negative and a full one
    among them); slots that the call does not cover and tokens past the capacity are not written."""
    lib = _abi.load()
    rng = np.random.default_rng(d)
    for tokens in (2, 15, 16, 17, 40):
        starts = np.array([0, 5, 16, 31, 64, 80, -3, 79], np.int32)
        c = Cache(rng, starts, 80, 3, d, 16, dtype, poison=False).upload(starts)
        table = c.table.copy()
        table[1, 1] = -1
        c.td = dev(table)
        k, v = (rng.standard_normal((8, 3, tokens, d)).astype(np.float32) for _ in range(2))
        if src == "bf16":
            k, v = oracle.round_bf16(k), oracle.round_bf16(v)
        to = (lambda x: dev(oracle.to_bf16_bits(x).view(np.int16))) if src == "bf16" else dev
        _abi.check(lib.sfg_hip_kv_append_pool_v1(
            to(k).data_ptr(), to(v).data_ptr(), BF16 if src == "bf16" else F32, c.kd.data_ptr(), c.vd.data_ptr(),
            BF16 if dtype == "bf16" else F32, c.td.data_ptr(), c.ld.data_ptr(), 0, 0, 8, 3, tokens, d, 16, c.per, c.pages, stream()))
        for got, was, new in zip(c.logical(c.kd, c.vd), (c.k, c.v), (k, v)):
            want = was.copy()
            for n in range(8):
                for t in range(tokens):
                    at = starts[n] + t
                    if 0 <= at < 80 and table[n, at // 16] >= 0:
                        want[n, :, at] = c.round(new[n, :, t])
            np.testing.assert_array_equal(got, want)


# (q heads, kv heads, D, nodes, lengths, splits): more than 32 columns in bf16
TILES = [(16, 4, 128, 24, (1500, 0, 64, 63, 65, 130), 0), (8, 2, 64, 30, (1000, 1, 700), 0), (8, 2, 128, 70, (900, 40, 0), 0),
         (12, 2, 128, 9, (300, 2000, 128), 3), (16, 4, 64, 100, (600, 33), 7), (8, 1, 128, 5, (4096, 17), 0),
         (4, 4, 128, 200, (190, 0, 500), 0), (64, 1, 64, 3, (250,), 1), (4, 2, 128, 64, tuple(range(0, 700, 10)), 0)]


@pytest.mark.parametrize("hq,hkv,d,t,lens,splits", TILES)
def test_trees_of_many_columns(hq, hkv, d, t, lens, splits):
    """The tile kernel: every number of columns a wave and a workgroup, runs that begin and end anywhere in a
    sequence, masks of up to seven words, poison where nothing may look, twice over the same workspace."""
    lib = _abi.load()
    rng = np.random.default_rng(hq + d + t)
    longest = max(lens)
    c = Cache(rng, lens, longest + t, hkv, d)
    c.upload(c.lens + t)
    for _ in range(2):
        bits = ancestors(random_tree(rng, c.b, t))
        q, qd, qdt = queries(rng, c.b, hq, t, d, "bf16")
        out, odt = output(q.shape, "bf16")
        run_tree(lib, c, qd, qdt, dev(words(bits)), t * -(-t // 32), out, odt, longest, splits)
        got = value(out)
        pick = rng.permutation(c.b * hq * t)[:400]  # (every column is computed; some are compared)
        for x in pick:
            n, h, i = x // (hq * t), x // t % hq, x % t
            s = np.arange(c.per * 16) < c.lens[n]
            s[c.lens[n]: c.lens[n] + t] = bits[n, i]
            ref, _, err, _ = attend(q[n, h, i], c.k[n, h // (hq // hkv)], c.v[n, h // (hq // hkv)], s, True, True)
            close(got[n, h, i], ref, err, f"column {n} {h} {i}")


@pytest.mark.parametrize("longest", [70, 3000])
def test_visible_infinities_in_trees_of_many_columns(longest):
    """Infinite drafted values reach the rows that see them, and no others; infinite committed values reach all:
    where one workgroup walks a sequence, and where several do."""
    lib = _abi.load()
    rng = np.random.default_rng(longest)
    t = 20
    c = Cache(rng, (longest, 60), longest + t, 2, 128)
    at = longest + 11
    c.v[0, 1, at, 5], c.v[0, 1, at, 100] = np.inf, np.nan
    c.v[0, 0, 33, 7] = -np.inf
    c.upload(c.lens + t)
    bits = ancestors(random_tree(rng, 2, t))
    q, qd, qdt = queries(rng, 2, 8, t, 128, "bf16")
    out, odt = output(q.shape, "bf16")
    run_tree(lib, c, qd, qdt, dev(words(bits)), t, out, odt, longest)
    got = value(out)
    for i in range(t):
        sees = bits[0, i, 11]
        assert ((got[0, 4:, i, 5] == np.inf) == sees).all() and (np.isnan(got[0, 4:, i, 100]) == sees).all()
    assert (got[0, :4, :, 7] == -np.inf).all()
    got[0, 4:, :, 5] = got[0, 4:, :, 100] = got[0, :4, :, 7] = 0.0
    assert np.isfinite(got).all()


@pytest.mark.parametrize("t,d", [(64, 128), (12, 64), (24, 128)])
def test_captured_trees_of_many_columns(t, d):
    """Replays with other lengths, masks and queries in the same buffers: nothing of a capture is kept but its
    addresses; an output off an 8-byte boundary gives what an aligned one gives, within rounding."""
    lib = _abi.load()
    rng = np.random.default_rng(t)
    b, hq, hkv, longest = 3, 8, 2, 6000
    c = Cache(rng, (6000, 17, 2500), longest + t, hkv, d, poison=False).upload((0, 0, 0))
    q, qd, qdt = queries(rng, b, hq, t, d, "bf16")
    mask = dev(words(ancestors(random_tree(rng, b, t))))
    out, odt = output(q.shape, "bf16")
    off, _ = output((q.size + 1,), "bf16")
    a = c.args(qd, out, qdt, odt, longest)
    ws = workspace(lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(a)))
    run_tree(lib, c, qd, qdt, mask, t * -(-t // 32), out, odt, longest, ws=ws)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            run_tree(lib, c, qd, qdt, mask, t * -(-t // 32), out, odt, longest, ws=ws)
    torch.cuda.synchronize()
    for lens in ((6000, 17, 2500), (1, 5999, 64), (0, 0, 0)):
        c.ld.copy_(torch.tensor(lens, dtype=torch.int32))
        qd.copy_(torch.from_numpy(rng.standard_normal(q.shape).astype(np.float32)))
        mask.copy_(torch.from_numpy(words(ancestors(random_tree(rng, b, t)))))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        run_tree(lib, c, qd, qdt, mask, t * -(-t // 32), out, odt, longest)
        view = off[1:].view(q.shape)
        run_tree(lib, c, qd, qdt, mask, t * -(-t // 32), view, odt, longest)
        torch.cuda.synchronize()
        assert torch.equal(replayed.view(torch.int16), out.view(torch.int16))
        # both within 2^-7 of the values they round, whose size the values' bound gives
        assert (view.float() - out.float()).abs().max() <= 2.0 ** -6 * np.abs(c.v).max()
