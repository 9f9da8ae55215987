"""bf16 queries, pools and output (GPU only): softmax weights keep 16 bits, so that an output is as far from the formula
as its own rounding takes it, and infinities among the visible keys and values give what the formula gives, whatever
the types."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from schedforge_amd import _abi
from schedforge_amd._abi import BF16, F32

from _helpers import dev, host, stream
from _paged_chosen import Cache, ancestors, close, output, queries, random_tree, value, words, workspace
from _tree_tiles import attend16, formula, sees

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def tree(lib, c, qd, qdt, bits, out, odt, splits=0):
    t = bits.shape[1]
    a = c.args(qd, out, qdt, odt, int(c.lens.max()), splits)
    ws = workspace(lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(a)))
    mask = dev(words(bits))
    _abi.check(lib.sfg_hip_attn_tree_v1(ctypes.byref(a), mask.data_ptr(), t * -(-t // 32), ws.data_ptr(), ws.numel(), stream()))


def weights(lib, c, qd, qdt, out, odt, wd, splits=0):
    a = c.args(qd, out, qdt, odt, int(c.lens.max()), splits)
    ws = workspace(lib.sfg_hip_attn_weights_workspace_v1(ctypes.byref(a)))
    _abi.check(lib.sfg_hip_attn_weights_v1(ctypes.byref(a), wd.data_ptr(), wd.shape[2], ws.data_ptr(), ws.numel(), stream()))


def sparse(lib, c, qd, qdt, out, odt, top):
    longest, dt = int(c.lens.max()), BF16 if c.dtype == "bf16" else F32
    bd = torch.zeros((c.pages, c.hkv, 2, c.d), dtype=torch.bfloat16 if c.dtype == "bf16" else torch.float32, device="cuda")
    _abi.check(lib.sfg_hip_kv_page_bounds_v1(c.kd.data_ptr(), dt, c.td.data_ptr(), c.ld.data_ptr(), longest, longest, bd.data_ptr(),
                                             c.b, c.hkv, c.d, c.pt, c.per, c.pages, stream()))
    sel = torch.full((c.b, qd.shape[2], c.hkv, top), 77, dtype=torch.int32, device="cuda")
    a = c.args(qd, out, qdt, odt, longest)
    ws = workspace(lib.sfg_hip_attn_sparse_workspace_v1(ctypes.byref(a), top))
    _abi.check(lib.sfg_hip_attn_sparse_v1(ctypes.byref(a), bd.data_ptr(), top, 1, 1, sel.data_ptr(), ws.data_ptr(), ws.numel(), stream()))
    return host(sel)


# (q heads, kv heads, D, rows, lengths, splits)
CALLS = [(8, 2, 128, 1, (900, 1, 17, 300), 0), (8, 2, 64, 4, (333, 40), 0), (34, 2, 128, 2, (500, 64), 3), (4, 4, 64, 1, (1300,), 0),
         (16, 4, 128, 3, (257, 260), 1)]


@pytest.mark.parametrize("std", [0.5, 2.5])
@pytest.mark.parametrize("hq,hkv,d,rows,lens,splits", CALLS)
def test_outputs_are_off_by_their_own_rounding(hq, hkv, d, rows, lens, splits, std):
    lib = _abi.load()
    rng = np.random.default_rng(hq + d)
    g = hq // hkv
    c = Cache(rng, lens, max(lens) + rows, hkv, d)
    c.upload(c.lens + rows)
    q, qd, qdt = queries(rng, c.b, hq, rows, d, "bf16", std=std)
    bits = ancestors(random_tree(rng, c.b, rows))
    out, odt = output(q.shape, "bf16")
    capacity = c.per * 16

    def compare(see, what):
        got = value(out)
        for n in range(c.b):
            for h in range(hq):
                for i in range(rows):
                    s = see(n, h, i)
                    if s.any():
                        ref, err = attend16(q[n, h, i], c.k[n, h // g], c.v[n, h // g], s)
                        close(got[n, h, i], ref, err, f"{what} {n} {h} {i}")
    tree(lib, c, qd, qdt, bits, out, odt, splits)
    compare(lambda n, h, i: sees(capacity, c.lens[n], bits[n, i]), "tree")
    weights(lib, c, qd, qdt, out, odt, torch.zeros((c.b, hkv, capacity), device="cuda"), splits)
    compare(lambda n, h, i: np.arange(capacity) < c.lens[n] - rows + i + 1, "weights")
    sel = sparse(lib, c, qd, qdt, out, odt, 6)
    compare(lambda n, h, i: (np.arange(capacity) < c.lens[n] - rows + i + 1) & np.isin(np.arange(capacity) // 16, sel[n, i, h // g]), "sparse")


@pytest.mark.parametrize("types", ["bf16/bf16/bf16", "bf16/bf16/f32", "f32/bf16/f32", "f32/f32/f32", "bf16/f32/bf16"])
@pytest.mark.parametrize("d", [128, 64, 80])
def test_visible_infinite_keys_and_values(d, types):
    """An infinite key element makes a row's scores of that token +inf (the row is NaN) or -inf (the token has no
    weight); infinite values make that dim infinite, or NaN where both signs meet."""
    lib = _abi.load()
    qt, kt, ot = types.split("/")
    rng = np.random.default_rng(d)
    hq, hkv, t, lens = 8, 2, 5, (70, 130)
    c = Cache(rng, lens, 160, hkv, d, 16, kt)
    c.k[0, 0, 20, 3], c.k[0, 1, 72, 9] = np.inf, -np.inf     # the second in a draft
    c.v[1, 0, 33, 5], c.v[1, 0, 40, 9] = np.inf, -np.inf
    c.v[1, 1, 3, 7], c.v[1, 1, 131, 7] = np.inf, -np.inf     # the second in a draft
    c.upload(c.lens + t)
    bits = ancestors(random_tree(rng, 2, t))
    q, qd, qdt = queries(rng, 2, hq, t, d, qt)
    out, odt = output(q.shape, ot)

    def compare(see):
        got = value(out)
        for n in range(2):
            for h in range(hq):
                for i in range(t):
                    want, _ = formula(q[n, h, i], c.k[n, h // 4], c.v[n, h // 4], see(n, h, i))
                    line = got[n, h, i]
                    np.testing.assert_array_equal(np.isnan(line), np.isnan(want), err_msg=f"{n} {h} {i}")
                    np.testing.assert_array_equal(np.isinf(line) * np.sign(line), np.isinf(want) * np.sign(want))
    tree(lib, c, qd, qdt, bits, out, odt)
    compare(lambda n, h, i: sees(c.per * 16, c.lens[n], bits[n, i]))
    weights(lib, c, qd, qdt, out, odt, torch.zeros((2, hkv, 160), device="cuda"))
    compare(lambda n, h, i: np.arange(c.per * 16) < c.lens[n] - t + i + 1)


@pytest.mark.parametrize("types", ["bf16/bf16/bf16", "f32/bf16/f32", "f32/f32/f32"])
@pytest.mark.parametrize("d,pt", [(128, 16), (64, 16), (80, 16), (33, 5)])
def test_accumulated_weights_of_infinite_scores(d, pt, types):
    """A token whose score is -inf draws nothing beside others, and NaN where every score that the row sees is -inf
    (as its output); a row with a score of +inf draws NaN; a row that sees nothing, its length past its place or
    its pages outside the pool, adds nothing."""
    lib = _abi.load()
    qt, kt, ot = types.split("/")
    rng = np.random.default_rng(d)
    hq, hkv, rows, lens = 4, 2, 2, (1, 40, 40, 33, 40)
    c = Cache(rng, lens, 40, hkv, d, pt, kt)
    c.k[0, 0, 0, 3] = -np.inf        # its only token
    c.k[1, 1, :, 3] = -np.inf        # every token
    c.k[2, 0, 7, 3] = -np.inf        # one of many
    c.k[2, 1, 39, 3] = np.inf        # the newest: only the second row sees it
    c.upload(c.lens)
    table = c.table.copy()
    table[4] = -1
    c.td = dev(table)
    q, qd, qdt = queries(rng, c.b, hq, rows, d, qt)
    q[..., 3] = np.abs(q[..., 3])
    qd.copy_(torch.from_numpy(q))
    out, odt = output(q.shape, ot)
    wd = torch.ones((c.b, hkv, 43), device="cuda")
    weights(lib, c, qd, qdt, out, odt, wd, 2)
    got, res = host(wd).astype(np.float64), value(out)
    for n in range(c.b):
        for h in range(hkv):
            want = np.ones(43)
            for head in (2 * h, 2 * h + 1):
                for i in range(rows):
                    s = np.arange(c.per * pt) < lens[n] - rows + i + 1
                    if not s.any() or n == 4:
                        assert np.isnan(res[n, head, i]).all()
                        continue
                    o, p = formula(q[n, head, i], c.k[n, h], c.v[n, h], s)
                    np.testing.assert_array_equal(np.isnan(res[n, head, i]), np.isnan(o))
                    want[: p.size] += p
            np.testing.assert_array_equal(np.isnan(got[n, h]), np.isnan(want))
            # four weights, each off by 2 (D + 4) 2^-24 times c sum |q k| (under 20 here) of itself: 1.3e-3 in all
            assert np.abs(got[n, h] - want)[~np.isnan(want)].max(initial=0.0) < 2.0 ** -9
