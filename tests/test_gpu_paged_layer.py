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
