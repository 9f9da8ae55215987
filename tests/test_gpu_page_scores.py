"""Page scores where keys or queries are infinite or NaN (GPU only): the pages taken are those of the largest
sum of max(q lo, q hi), whatever the signs of a group's queries, and NaN scores come last."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from schedforge_amd import _abi
from schedforge_amd._abi import BF16, F32

from _helpers import host, stream
from _paged_chosen import Cache, output, queries, value, workspace

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def select(lib, c, q, qd, qdt, top, sink, recent):
    longest, dt = int(c.lens.max()), BF16 if c.dtype == "bf16" else F32
    bd = torch.zeros((c.pages, c.hkv, 2, c.d), dtype=torch.bfloat16 if c.dtype == "bf16" else torch.float32, device="cuda")
    _abi.check(lib.sfg_hip_kv_page_bounds_v1(c.kd.data_ptr(), dt, c.td.data_ptr(), c.ld.data_ptr(), longest, longest, bd.data_ptr(),
                                             c.b, c.hkv, c.d, c.pt, c.per, c.pages, stream()))
    sel = torch.full((c.b, q.shape[2], c.hkv, top), 77, dtype=torch.int32, device="cuda")
    out, odt = output(q.shape, "f32")
    a = c.args(qd, out, qdt, odt, longest)
    ws = workspace(lib.sfg_hip_attn_sparse_workspace_v1(ctypes.byref(a), top))
    _abi.check(lib.sfg_hip_attn_sparse_v1(ctypes.byref(a), bd.data_ptr(), top, sink, recent, sel.data_ptr(), ws.data_ptr(), ws.numel(),
                                          stream()))
    return host(sel), value(bd)


def bounds(k):
    """[pages][pt][D] -> lowest and highest [pages][D], NaN keys passed over."""
    none = np.isnan(k).all(1)
    lo = np.where(none, np.nan, np.where(np.isnan(k), np.inf, k).min(1))
    hi = np.where(none, np.nan, np.where(np.isnan(k), -np.inf, k).max(1))
    return lo, hi


def scores(q, lo, hi):
    """q [G][D]: the definition in 64 bits."""
    with np.errstate(invalid="ignore"):
        q = q.astype(np.float64)[:, None]
        return np.maximum(q * lo, q * hi).sum((0, 2))  # (maximum hands NaN on)


def taken(score, top, sink, recent):
    n = score.size
    first = set(range(min(sink, n))) | set(range(max(0, n - recent), n))
    rest = [p for p in np.lexsort((np.arange(n), -np.where(np.isnan(score), 0.0, score), np.isnan(score))) if p not in first]
    return sorted(first | set(rest[: max(0, top - len(first))]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("hq,hkv,d,pt,rows,sink,recent", [(8, 2, 128, 16, 1, 0, 1), (8, 2, 64, 16, 3, 1, 1), (2, 2, 64, 16, 1, 0, 0),
                                                          (6, 3, 80, 16, 2, 0, 1), (4, 2, 33, 5, 1, 1, 2)])
def test_infinite_and_nan_bounds(hq, hkv, d, pt, rows, sink, recent, dtype):
    lib = _abi.load()
    rng = np.random.default_rng(d + hq)
    lens, g = (60 * pt - 3, 20 * pt, 9), hq // hkv
    c = Cache(rng, lens, 60 * pt, hkv, d, pt, dtype)
    q, qd, qdt = queries(rng, 3, hq, rows, d, "bf16")
    q[..., 0:4], q[..., 4:8] = np.abs(q[..., 0:4]), -np.abs(q[..., 4:8])  # dims of one sign in every group
    q[..., 8] = 0.0
    q[2, :, :, 9] = np.nan
    qd.copy_(torch.from_numpy(q))
    for n, pages in ((0, 60), (1, 20)):
        for h in range(hkv):
            spots = rng.permutation(pages)
            for x, (dim, v) in enumerate(((0, -np.inf), (1, np.inf), (4, np.inf), (5, -np.inf), (8, np.inf), (20, np.inf), (21, -np.inf))):
                for p in spots[2 * x: 2 * x + 2]:
                    c.k[n, h, p * pt + 1, dim] = v  # (a page holds more tokens than that)
            c.k[n, h, spots[14] * pt: (spots[14] + 1) * pt, 12] = np.nan
            c.k[n, h, spots[15] * pt + 1, 13] = np.nan
            c.k[n, h, spots[16] * pt: (spots[16] + 1) * pt, 2] = -np.inf
            c.k[n, h, spots[17] * pt, 3], c.k[n, h, spots[17] * pt, 6] = -np.inf, np.inf
    c.upload(lens)
    for top in (2, 7, 30, 45):
        if top < sink + recent:
            continue
        sel, bd = select(lib, c, q, qd, qdt, top, sink, recent)
        for n in range(3):
            for h in range(hkv):
                for i in range(rows):
                    end = max(lens[n] - rows + i + 1, 0)
                    pages, held = -(-end // pt), -(-lens[n] // pt)
                    k = np.where((np.arange(held * pt) < lens[n])[:, None], c.k[n, h, : held * pt], np.nan).reshape(held, pt, d)
                    lo, hi = bounds(k)
                    np.testing.assert_array_equal(bd[c.table[n, :held], h], np.stack((lo, hi), 1).astype(np.float32))
                    want = taken(scores(q[n, h * g: (h + 1) * g, i], lo[:pages], hi[:pages]), top, sink, recent)
                    np.testing.assert_array_equal(sel[n, i, h, : len(want)], want, err_msg=f"{top} {n} {h} {i}")
                    assert (sel[n, i, h, len(want):] == -1).all()
