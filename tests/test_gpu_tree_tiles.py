"""Trees of many columns through the tile kernel (GPU only): every number of columns a wave and a workgroup, at both
head dims, as the call plans itself and with as many ranges as asked for.  tests/test_tree_tiles_plan.py checks on the
CPU that these calls are the tile kernel's."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from schedforge_amd import _abi
from schedforge_amd._abi import BF16

from _helpers import dev, stream
from _paged_chosen import Cache, ancestors, close, output, queries, random_tree, value, words, workspace
from _tree_tiles import TILES, attend16, formula, sees

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def run(lib, c, qd, bits, out, longest, splits, ws=None):
    t = bits.shape[1]
    a = c.args(qd, out, BF16, BF16, longest, splits)
    ws = workspace(lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(a))) if ws is None else ws
    mask = dev(words(bits))
    _abi.check(lib.sfg_hip_attn_tree_v1(ctypes.byref(a), mask.data_ptr(), t * -(-t // 32), ws.data_ptr(), ws.numel(), stream()))
    return ws


@pytest.mark.parametrize("hq,hkv,d,t,lens,splits", TILES)
def test_tiles_against_64_bits(hq, hkv, d, t, lens, splits):
    """Columns of every sequence and kv head; poison where nothing may look, twice over the same workspace."""
    lib = _abi.load()
    rng = np.random.default_rng(hq + d + t + splits)
    longest, g = max(lens), hq // hkv
    c = Cache(rng, lens, longest + t, hkv, d)
    c.upload(c.lens + t)
    ws = None
    for _ in range(2):
        bits = ancestors(random_tree(rng, c.b, t))
        q, qd, _ = queries(rng, c.b, hq, t, d, "bf16", std=2.5)
        out, _ = output(q.shape, "bf16")
        ws = run(lib, c, qd, bits, out, longest, splits, ws)
        got = value(out)
        assert np.isfinite(got).all()
        for n in range(c.b):
            for h in range(hkv):
                for x in rng.permutation(t * g)[:6]:
                    i, head = x // g, h * g + x % g
                    ref, err = attend16(q[n, head, i], c.k[n, h], c.v[n, h], sees(c.per * 16, c.lens[n], bits[n, i]))
                    close(got[n, head, i], ref, err, f"column {n} {head} {i}")


# infinities: (q heads, kv heads, D, nodes, lengths, splits); one range a (sequence, kv head), and several
INFINITE = [(8, 2, 128, 8, (130, 130), 1), (8, 2, 128, 30, (130, 130), 1), (8, 2, 64, 64, (130, 130), 1), (8, 2, 128, 64, (130, 130), 1),
            (8, 2, 64, 12, (900, 40), 4), (8, 2, 128, 25, (700, 63), 3), (8, 2, 64, 50, (640, 65), 5), (8, 2, 128, 70, (300, 500), 2),
            (16, 4, 128, 64, (2600, 64, 1311), 0)]


@pytest.mark.parametrize("hq,hkv,d,t,lens,splits", INFINITE)
def test_infinities_and_nan_reach_who_sees_them(hq, hkv, d, t, lens, splits):
    """Infinite and NaN values, and infinite keys, among the committed tokens and the drafts: every output is what
    the formula gives, and rows that see none of them are finite."""
    lib = _abi.load()
    rng = np.random.default_rng(d + t)
    longest, g = max(lens), hq // hkv
    c = Cache(rng, lens, longest + t, hkv, d)
    a, b = int(c.lens[0]), int(c.lens[1])
    c.v[0, 0, 33, 7], c.v[0, 0, 34, 7] = -np.inf, -np.inf
    c.v[0, 1, 17, 3], c.v[0, 1, a - 1, 3] = np.inf, -np.inf       # both: NaN
    c.v[0, 1, a + t // 2, 5], c.v[0, 1, a + t // 2, d - 1] = np.inf, np.nan
    c.k[1, 0, b + t // 3, 11] = np.inf                            # scores of both signs
    c.k[1, 1, 20, 2] = -np.inf
    c.upload(c.lens + t)
    bits = ancestors(random_tree(rng, c.b, t))
    q, qd, _ = queries(rng, c.b, hq, t, d, "bf16")
    out, _ = output(q.shape, "bf16")
    run(lib, c, qd, bits, out, longest, splits)
    got = value(out)
    plain = odd = 0
    for n in range(2):
        for head in range(hq):
            for i in range(t):
                s = sees(c.per * 16, c.lens[n], bits[n, i])
                want, _ = formula(q[n, head, i], c.k[n, head // g], c.v[n, head // g], s)
                line = got[n, head, i]
                np.testing.assert_array_equal(np.isnan(line), np.isnan(want))
                np.testing.assert_array_equal(np.isinf(line) * np.sign(line), np.isinf(want) * np.sign(want))
                finite = np.isfinite(want).all()
                plain, odd = plain + finite, odd + (not finite)
    assert odd > 0 and plain > 0


def test_captured_tiles_replay_with_other_inputs():
    """One capture over long sequences, replayed with other lengths, masks and queries: columns against 64 bits."""
    lib = _abi.load()
    rng = np.random.default_rng(77)
    hq, hkv, d, t, longest = 32, 8, 128, 64, 3000
    c = Cache(rng, (3000, 17, 2500), longest + t, hkv, d, poison=False).upload((0, 0, 0))
    q, qd, _ = queries(rng, 3, hq, t, d, "bf16")
    mask = dev(words(ancestors(random_tree(rng, 3, t))))
    out, _ = output(q.shape, "bf16")
    a = c.args(qd, out, BF16, BF16, longest)
    ws = workspace(lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(a)))

    def go():
        _abi.check(lib.sfg_hip_attn_tree_v1(ctypes.byref(a), mask.data_ptr(), t * 2, ws.data_ptr(), ws.numel(), stream()))
    go()
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        with torch.cuda.graph(graph, stream=side):
            go()
    for lens in ((3000, 17, 2500), (64, 2999, 1), (0, 0, 1500)):
        bits = ancestors(random_tree(rng, 3, t))
        x = value(torch.from_numpy(rng.standard_normal(q.shape).astype(np.float32)).to(torch.bfloat16))
        c.ld.copy_(torch.tensor(lens, dtype=torch.int32))
        qd.copy_(torch.from_numpy(x))
        mask.copy_(torch.from_numpy(words(bits)))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = value(out)
        for n in range(3):
            for _ in range(40):
                head, i = int(rng.integers(hq)), int(rng.integers(t))
                ref, err = attend16(x[n, head, i], c.k[n, head // 4], c.v[n, head // 4], sees(c.per * 16, lens[n], bits[n, i]))
                close(got[n, head, i], ref, err, f"column {n} {head} {i}")
        torch.matmul(torch.ones(64, 64, device="cuda"), torch.ones(64, 64, device="cuda"))  # eager work between
        go()
        torch.cuda.synchronize()
        assert torch.equal(torch.from_numpy(got), out.float().cpu())
