"""Refusals of the operators that choose what a paged cache keeps and reads: invalid arguments come back from
the host with the documented code and a message, before anything is launched (no GPU needed: the pointers are
never followed), and the Python layer refuses what it can see."""
from __future__ import annotations

import ctypes

import numpy as np
import pytest

from schedforge_amd import _abi

CONFIG, SHAPE, GUARD, UNSUPPORTED, WORKSPACE = (_abi.ERR_INVALID_CONFIG, _abi.ERR_SHAPE, _abi.ERR_GUARD,
                                                _abi.ERR_UNSUPPORTED, _abi.ERR_WORKSPACE)


@pytest.fixture(scope="module")
def lib():
    return _abi.load()


def args(**kw):
    a = _abi.PagedAttnArgs()
    base = dict(q=64, q_dtype=_abi.BF16, k_pool=64, v_pool=64, kv_dtype=_abi.BF16, page_table=64, seq_lens=None, out=64,
                out_dtype=_abi.BF16, batch=2, q_heads=8, kv_heads=2, rows=4, head_dim=128, page_tokens=16, pages_per_seq=8,
                num_pages=16, max_context=100, kv_splits=0, scale=0.0)
    base.update(kw)
    for k, v in base.items():
        setattr(a, k, v)
    return a


def calls(lib, a):
    """The three attentions of one argument block, with no workspace."""
    r = ctypes.byref(a)
    yield lib.sfg_hip_attn_tree_v1(r, 64, 4, None, 0, None)
    yield lib.sfg_hip_attn_weights_v1(r, 64, 128, None, 0, None)
    yield lib.sfg_hip_attn_sparse_v1(r, 64, 4, 1, 1, 64, None, 0, None)


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), CONFIG), (dict(k_pool=None), CONFIG), (dict(v_pool=None), CONFIG), (dict(page_table=None), CONFIG),
    (dict(out=None), CONFIG), (dict(batch=0), CONFIG), (dict(q_heads=7), CONFIG), (dict(q_heads=0), CONFIG),
    (dict(kv_heads=0), CONFIG), (dict(rows=0), CONFIG), (dict(head_dim=0), CONFIG), (dict(page_tokens=0), CONFIG),
    (dict(pages_per_seq=0), CONFIG), (dict(num_pages=0), CONFIG), (dict(max_context=-1), CONFIG),
    (dict(head_dim=257), UNSUPPORTED), (dict(kv_dtype=_abi.I8), UNSUPPORTED), (dict(q_dtype=_abi.I32), UNSUPPORTED),
    (dict(out_dtype=_abi.I8), UNSUPPORTED), (dict(max_context=129), GUARD),
    (dict(pages_per_seq=1 << 40), UNSUPPORTED), (dict(num_pages=1 << 31), UNSUPPORTED), (dict(batch=1 << 24), UNSUPPORTED),
    (dict(rows=1 << 30, pages_per_seq=1 << 26), UNSUPPORTED), (dict(q_heads=1 << 40), UNSUPPORTED)])
def test_attention_arguments(lib, bad, code):
    for rc in calls(lib, args(**bad)):
        assert rc == code, (bad, rc, lib.sfg_hip_last_error())
        assert lib.sfg_hip_last_error()


def test_attention_specifics(lib):
    a = args()
    r = ctypes.byref(a)
    assert lib.sfg_hip_attn_tree_v1(None, 64, 4, None, 0, None) == SHAPE
    assert lib.sfg_hip_attn_tree_v1(r, None, 4, None, 0, None) == SHAPE
    assert lib.sfg_hip_attn_tree_v1(r, 64, 3, None, 0, None) == SHAPE               # masks of 4 words overlap
    assert lib.sfg_hip_attn_tree_v1(r, 64, -4, None, 0, None) == SHAPE
    assert lib.sfg_hip_attn_tree_v1(ctypes.byref(args(max_context=125)), 64, 4, None, 0, None) == GUARD  # no room for 4 drafts
    assert lib.sfg_hip_attn_weights_v1(r, None, 128, None, 0, None) == SHAPE
    assert lib.sfg_hip_attn_weights_v1(r, 64, 99, None, 0, None) == SHAPE
    assert lib.sfg_hip_attn_weights_v1(ctypes.byref(args(max_context=3)), 64, 128, None, 0, None) == CONFIG  # 4 rows of 3 tokens
    assert lib.sfg_hip_attn_weights_v1(ctypes.byref(args(max_context=0)), 64, 128, None, 0, None) == CONFIG
    assert lib.sfg_hip_attn_weights_v1(r, 64, 128, None, 0, None) == WORKSPACE
    for top, sink, recent in ((0, 0, 0), (4, -1, 0), (4, 0, -1), (4, 3, 2), (4, 5, 0), (1 << 32, 1, 1)):
        assert lib.sfg_hip_attn_sparse_v1(r, 64, top, sink, recent, 64, None, 0, None) == SHAPE, (top, sink, recent)
    assert lib.sfg_hip_attn_sparse_v1(r, None, 4, 1, 1, 64, None, 0, None) == SHAPE
    assert lib.sfg_hip_attn_sparse_v1(r, 64, 4, 1, 1, None, None, 0, None) == SHAPE
    n = lib.sfg_hip_attn_sparse_workspace_v1(r, 4)
    assert n > 0
    assert lib.sfg_hip_attn_sparse_v1(r, 64, 4, 1, 1, 64, 64, n - 1, None) == WORKSPACE
    assert lib.sfg_hip_attn_sparse_v1(r, 64, 4, 1, 1, 64, 72, n, None) == WORKSPACE  # off a 16-byte boundary
    with pytest.raises(RuntimeError, match="workspace"):
        _abi.check(lib.sfg_hip_attn_sparse_v1(r, 64, 4, 1, 1, 64, None, 0, None))


def test_workspace_queries_of_bad_sizes_are_zero(lib):
    for bad in (dict(batch=0), dict(q_heads=7), dict(rows=0), dict(head_dim=300), dict(page_tokens=0), dict(max_context=-2)):
        r = ctypes.byref(args(**bad))
        assert lib.sfg_hip_attn_tree_workspace_v1(r) == 0
        assert lib.sfg_hip_attn_weights_workspace_v1(r) == 0
        assert lib.sfg_hip_attn_sparse_workspace_v1(r, 4) == 0
    assert lib.sfg_hip_attn_tree_workspace_v1(None) == 0
    assert lib.sfg_hip_attn_sparse_workspace_v1(ctypes.byref(args()), 0) == 0


def test_sizes_past_counting(lib):
    """Sizes whose products or sums leave 64 bits: queries say 0, calls refuse."""
    far = (1 << 63) - 1
    for bad in (dict(batch=1 << 32, kv_heads=1 << 32, q_heads=1 << 32), dict(rows=1 << 62), dict(q_heads=1 << 40), dict(page_tokens=far),
                dict(batch=1 << 12, rows=1 << 10)):
        r = ctypes.byref(args(**bad))
        assert lib.sfg_hip_attn_tree_workspace_v1(r) == 0, bad
        assert lib.sfg_hip_attn_weights_workspace_v1(r) == 0, bad
        assert lib.sfg_hip_attn_sparse_workspace_v1(r, 4) == 0, bad
    for longest in (far, far - 3, 1 << 31):
        r = ctypes.byref(args(max_context=longest))
        assert lib.sfg_hip_attn_tree_workspace_v1(r) == lib.sfg_hip_attn_sparse_workspace_v1(r, 4) == 0
        for rc in calls(lib, args(max_context=longest)):
            assert rc == GUARD, longest
    wide = args(batch=1 << 20, q_heads=2, kv_heads=2, rows=1)
    for rc in calls(lib, wide):
        assert rc == UNSUPPORTED


def test_token_selection(lib):
    def call(weights=64, ld=100, lens=None, longest=100, budget=10, recent=2, keep=64, counts=128, kept=None, b=2, h=2):
        return lib.sfg_hip_kv_select_v1(weights, ld, lens, longest, budget, recent, keep, counts, kept, b, h, None)
    for bad in (dict(weights=None), dict(keep=None), dict(counts=None), dict(ld=99), dict(longest=0), dict(b=0), dict(h=0),
                dict(lens=128)):
        assert call(**bad) == SHAPE, bad
    for bad in (dict(budget=0), dict(recent=-1), dict(recent=11)):
        assert call(**bad) == CONFIG, bad
    for bad in (dict(b=1 << 22), dict(longest=1 << 31, ld=1 << 31), dict(budget=1 << 31)):
        assert call(**bad) == UNSUPPORTED, bad


def test_compaction_and_bounds(lib):
    def compact(k=64, v=64, dt=_abi.BF16, table=64, keep=64, heads=2, ld=10, counts=64, new=64, most=10, b=2, h=2, d=128, pt=16,
                per=8, pages=16):
        return lib.sfg_hip_kv_compact_v1(k, v, dt, table, None, keep, heads, ld, counts, new, most, b, h, d, pt, per, pages, None)
    for bad in (dict(k=None), dict(v=None), dict(keep=None), dict(counts=None), dict(new=None), dict(heads=3), dict(heads=0),
                dict(ld=9), dict(most=0)):
        assert compact(**bad) == SHAPE, bad
    for bad in (dict(table=None), dict(b=0), dict(h=0), dict(d=0), dict(pt=0), dict(per=0), dict(pages=0)):
        assert compact(**bad) == CONFIG, bad
    assert compact(dt=_abi.I8) == UNSUPPORTED and compact(d=300) == UNSUPPORTED
    assert compact(most=129, ld=200) == GUARD

    def bounds(k=64, dt=_abi.BF16, table=64, longest=100, fresh=1, out=64, b=2, h=2, d=128, pt=16, per=8, pages=16):
        return lib.sfg_hip_kv_page_bounds_v1(k, dt, table, None, longest, fresh, out, b, h, d, pt, per, pages, None)
    for bad in (dict(k=None), dict(out=None), dict(longest=0), dict(fresh=0)):
        assert bounds(**bad) == SHAPE, bad
    assert bounds(table=None) == CONFIG and bounds(longest=129) == GUARD and bounds(dt=_abi.I32) == UNSUPPORTED


def test_python_layer():
    torch = pytest.importorskip("torch")
    from schedforge_amd import paged_ops as po
    mask = po.tree_mask([[-1, 0, 0, 1], [-1, -1, 1, 2]], device="cpu")
    assert mask.shape == (2, 4, 1) and mask[..., 0].tolist() == [[1, 3, 5, 11], [1, 2, 6, 14]]
    wide = po.tree_mask([list(range(-1, 39))], device="cpu")  # a chain: every earlier node
    assert wide.shape == (1, 40, 2) and wide[0, 39].numpy().view(np.uint32).tolist() == [0xFFFFFFFF, 0xFF]
    for bad in ([[0]], [[-1, 1]], [[-2]], [-1], np.zeros((1, 0))):
        with pytest.raises(ValueError):
            po.tree_mask(bad, device="cpu")

    class Host:  # the fields that argument checks look at
        from schedforge_amd.kvcache import PagedKVConfig
        config, device, length = PagedKVConfig(2, 2, 64, 64, 16, 64), torch.device("cpu"), 40
    q = torch.zeros(2, 4, 3, 64)
    po._tensor(Host, q, "query", (torch.float32,), (2, 4, 3, 64))
    for bad in (q.double(), q[..., ::2], q[:1], q.numpy(), torch.zeros(2, 4, 64, 3).transpose(2, 3)):
        with pytest.raises(ValueError, match="query"):
            po._tensor(Host, bad, "query", (torch.float32,), (2, 4, 3, 64))
    with pytest.raises(ValueError, match="seq_lens"):
        po._lens(Host, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(ValueError, match="capacity"):
        po.accept_drafts(Host, torch.zeros((2, 30), dtype=torch.int32), torch.zeros(2, dtype=torch.int32),
                         torch.zeros(2, dtype=torch.int32))
    with pytest.raises(ValueError, match="budget"):
        po.evict_paged_kv(Host, torch.zeros(2, 2, 64), 10, 11)
