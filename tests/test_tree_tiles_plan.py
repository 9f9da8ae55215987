"""Which trees the tile kernel takes, by the workspace it asks for (no GPU needed): only bf16 calls with a bf16 output
do, so that the same call with an fp32 output asks for the ordinary kernels' workspace, which is smaller."""
from __future__ import annotations

import ctypes

import pytest

from schedforge_amd import _abi

from _tree_tiles import TILES


def query(lib, hq, hkv, d, t, batch, longest, splits, out):
    a = _abi.PagedAttnArgs()
    a.q_dtype, a.kv_dtype, a.out_dtype = _abi.BF16, _abi.BF16, out
    a.batch, a.q_heads, a.kv_heads, a.rows, a.head_dim = batch, hq, hkv, t, d
    a.page_tokens, a.pages_per_seq, a.num_pages = 16, -(-(longest + t) // 16), 1
    a.max_context, a.kv_splits = longest, splits
    return lib.sfg_hip_attn_tree_workspace_v1(ctypes.byref(a))


@pytest.mark.parametrize("hq,hkv,d,t,lens,splits", TILES + [(32, 8, 128, 64, (3000, 17, 2500), 0)])
def test_these_calls_take_the_tile_kernel(hq, hkv, d, t, lens, splits):
    lib = _abi.load()
    tiles, ordinary = (query(lib, hq, hkv, d, t, len(lens), max(lens), splits, out) for out in (_abi.BF16, _abi.F32))
    assert tiles > ordinary


def test_every_kernel_of_the_tiles_is_among_them():
    kinds = {(d, (cols > 64) + (cols > 128) + (cols > 256), splits > 0)
             for hq, hkv, d, t, _, splits in TILES for cols in (t * hq // hkv,)}
    assert kinds == {(d, c, s) for d in (64, 128) for c in range(4) for s in (False, True)}


def test_small_trees_do_not():
    lib = _abi.load()
    for hq, hkv, d, t, longest in ((32, 8, 128, 8, 900), (16, 4, 64, 1, 8000), (8, 8, 128, 7, 8000)):
        assert query(lib, hq, hkv, d, t, 1, longest, 0, _abi.BF16) == query(lib, hq, hkv, d, t, 1, longest, 0, _abi.F32)
