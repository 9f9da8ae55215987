"""The Python layer over the paged operators on the host (no GPU needed): what it hands to the C ABI, what it refuses
and what it leaves unchanged when it does.  The pools are CPU tensors and the library records the calls."""
from __future__ import annotations

import contextlib

import pytest

from schedforge_amd._abi import BF16
from schedforge_amd.kvcache import PageAllocator, PagedKVConfig

torch = pytest.importorskip("torch")

from schedforge_amd import paged_ops as po  # noqa: E402


class Library:
    def __init__(self):
        self.calls = []

    def __getattr__(self, name):
        def call(*args):
            self.calls.append((name, args))
            return 0
        return call


class Cache:
    """A PagedKVCache without a device."""
    device, pool_dtype = torch.device("cpu"), BF16
    length = property(lambda self: self.alloc.length)
    page_table = property(lambda self: self.alloc.page_table)

    def __init__(self, length=40, batch=2, kv_heads=2, d=64, capacity=128):
        self.config = PagedKVConfig(batch, kv_heads, d, d, 16, capacity)
        self.alloc, self.lib, self.uploads = PageAllocator(self.config), Library(), 0
        n = self.config.num_pages
        self.k_pool = self.v_pool = torch.zeros((n, kv_heads, 16, d), dtype=torch.int16)
        self.table = torch.zeros((batch, self.config.pages_per_seq), dtype=torch.int32)
        self.alloc.reserve(length)
        self.alloc.length = length

    def _sync_table(self, *_):
        self.uploads += 1


real_on = po._on


@pytest.fixture(autouse=True)
def host(monkeypatch):
    @contextlib.contextmanager
    def on(cache, stream):
        yield 0
    monkeypatch.setattr(po, "_on", on)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def drafts(t, b=2, h=2, d=64):
    return torch.zeros((b, h, t, d), dtype=torch.bfloat16)


def test_accepted_counts_are_cut_to_the_longest():
    """The kernel takes the host's bound on the counts, so that no length passes cache.length."""
    cache = Cache()
    po.append_drafts(cache, drafts(6), drafts(6), ints(2))
    po.accept_drafts(cache, ints(2, 6), ints(2), ints(2), longest=3)
    name, args = cache.lib.calls[-1]
    assert name == "sfg_hip_kv_compact_v1" and args[7] == 6 and args[10] == 3
    assert cache.length == 43
    po.accept_drafts(cache, ints(2, 5), ints(2), ints(2))
    assert cache.lib.calls[-1][1][10] == 5 and cache.length == 48


def test_nothing_accepted_launches_nothing():
    cache = Cache()
    po.append_drafts(cache, drafts(6), drafts(6), ints(2))
    calls = len(cache.lib.calls)
    po.accept_drafts(cache, ints(2, 6), ints(2), ints(2), longest=0)
    assert len(cache.lib.calls) == calls and cache.length == 40


def test_counts_beyond_the_path_or_the_capacity_are_refused():
    cache = Cache()
    for n, longest in ((30, -1), (30, 31), (100, 89)):
        with pytest.raises(ValueError):
            po.accept_drafts(cache, ints(2, n), ints(2), ints(2), longest=longest)
    assert cache.length == 40 and not cache.lib.calls


def test_calls_that_change_the_tables_are_not_captured(monkeypatch):
    """A capture is refused before anything is changed where pages change hands, and let through where none do."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    cache = Cache()  # 40 tokens in three pages
    po.append_drafts(cache, drafts(8), drafts(8), ints(2))
    with pytest.raises(RuntimeError, match="captured"):
        po.append_drafts(cache, drafts(9), drafts(9), ints(2))
    weights = torch.zeros((2, 2, 128))
    with pytest.raises(RuntimeError, match="captured"):
        po.evict_paged_kv(cache, weights, 39, 3)
    po.evict_paged_kv(cache, weights, 40, 3)  # nothing to evict
    assert cache.uploads == 0 and cache.length == 40 and [len(p) for p in cache.page_table] == [3, 3]
    assert [name for name, _ in cache.lib.calls] == ["sfg_hip_kv_append_pool_v1", "sfg_hip_kv_select_v1"]


def test_tensors_and_streams_of_another_device_are_refused(monkeypatch):
    cache = Cache()
    cache.device = torch.device("cuda", 1)
    with pytest.raises(ValueError, match="cuda:1"):
        po.append_drafts(cache, drafts(3), drafts(3))
    with pytest.raises(ValueError, match="cuda:1"):
        po._tensor(cache, torch.empty(2, device="meta"), "query", torch.float32, (2,))

    class Stream:
        def __init__(self, index):
            self.device = torch.device("cuda", index)
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    for stream in (Stream(0), 12345, "side"):
        with pytest.raises(ValueError, match="stream"):
            with real_on(cache, stream):
                pass


def test_arguments_that_are_no_tensors_are_refused():
    cache, q = Cache(), torch.zeros((2, 4, 3, 64))
    mask, weights, bounds = ints(2, 3, 1), torch.zeros((2, 2, 128)), torch.zeros((cache.config.num_pages, 2, 2, 64), dtype=torch.bfloat16)
    calls = [("query", dict(query=None)), ("query", dict(query=q.numpy())), ("query", dict(query=q[0])), ("query", dict(query=q[..., ::2])),
             ("out", dict(out=q.numpy())), ("out", dict(out=q[:, :2])), ("workspace", dict(workspace=bytes(8))), ("workspace", dict(workspace=64)),
             ("workspace", dict(workspace=torch.zeros(8)))]
    for name, bad in calls:
        a = dict(query=q, **bad) if name != "query" else bad
        for call in (lambda: po.tree_attention(cache, mask=mask, **a), lambda: po.weighted_decode_attention(cache, weights=weights, **a),
                     lambda: po.sparse_decode_attention(cache, bounds=bounds, top_pages=4, **a)):
            with pytest.raises(ValueError, match=name):
                call()
    assert not any("workspace" not in name for name, _ in cache.lib.calls)
