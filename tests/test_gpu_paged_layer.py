"""The Python layer over the paged operators on the device (GPU only): lengths, waits and devices."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from schedforge_amd import paged_ops as po
from schedforge_amd.kvcache import PagedKVConfig, append_paged_kv, make_paged_kv_cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def bf16(rng, *shape):
    return torch.from_numpy(oracle.round_bf16(rng.standard_normal(shape).astype(np.float32))).to(torch.bfloat16).cuda()


def filled(rng, batch=2, tokens=40, capacity=400, d=64):
    cache = make_paged_kv_cache(PagedKVConfig(batch, 2, d, d, 16, capacity))
    k = oracle.round_bf16(rng.standard_normal((batch, 2, tokens, d)).astype(np.float32))
    append_paged_kv(cache, k, k, tokens)
    return cache


def test_no_length_passes_the_bound_that_the_host_gave():
    cache = filled(np.random.default_rng(1))
    lens = torch.tensor([40, 33], dtype=torch.int32, device="cuda")
    x = bf16(np.random.default_rng(2), 2, 2, 9, 64)
    po.append_drafts(cache, x, x, lens)
    path = torch.arange(9, dtype=torch.int32, device="cuda").repeat(2, 1)
    po.accept_drafts(cache, path, torch.tensor([9, 2], dtype=torch.int32, device="cuda"), lens, longest=4)
    assert lens.tolist() == [44, 35] and cache.length == 44
    po.accept_drafts(cache, path, torch.tensor([9, 2], dtype=torch.int32, device="cuda"), lens, longest=0)
    assert lens.tolist() == [44, 35] and cache.length == 44


def test_calls_that_change_the_tables_do_not_wait():
    """Work that takes a while is queued, then drafts are appended into new pages and tokens evicted: both calls come
    back while the work still runs, and the tables arrive in order."""
    rng = np.random.default_rng(3)
    warm, cache = filled(rng), filled(rng)
    x = bf16(rng, 2, 2, 60, 64)
    weights = po.attention_weights(cache)
    weights.uniform_(0.0, 1.0)
    for c in (warm, cache):
        w = weights.clone()
        a = torch.ones((4096, 4096), device="cuda")
        torch.cuda.synchronize()
        if c is cache:
            for _ in range(200):
                a = a @ a  # (infinite soon, and as slow)
        busy = torch.cuda.Event()
        busy.record()
        po.append_drafts(c, x, x)
        appended = busy.query()
        table = c.table.clone()
        want_appended = c.alloc.table_array()
        po.evict_paged_kv(c, w, 20, 4)
        evicted = busy.query()
        torch.cuda.synchronize()
        np.testing.assert_array_equal(table.cpu().numpy(), want_appended)
        np.testing.assert_array_equal(c.table.cpu().numpy(), c.alloc.table_array())
        if c is cache:
            assert not appended and not evicted


def test_a_cache_knows_its_device():
    """The device's index is the pools', also where the cache was made on "cuda"; streams are torch's, of that device."""
    cache = filled(np.random.default_rng(5))
    assert cache.device == cache.k_pool.device and cache.device.index is not None
    x = bf16(np.random.default_rng(6), 2, 2, 3, 64)
    po.append_drafts(cache, x, x, stream=torch.cuda.Stream())
    for stream in (torch.cuda.current_stream().cuda_stream, "side"):
        with pytest.raises(ValueError, match="stream"):
            po.append_drafts(cache, x, x, stream=stream)
    torch.cuda.synchronize()
