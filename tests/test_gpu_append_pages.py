"""Appends of several tokens (GPU only): calls large enough to go by pages, and calls with more (sequence, head)s than
such a launch holds, write what the call covers and nothing else."""
from __future__ import annotations

import numpy as np
import pytest

import oracle
from schedforge_amd import _abi
from schedforge_amd._abi import BF16, F32

from _helpers import dev, host, stream
from _paged_chosen import Cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# (kv heads, D, tokens): rows of 8 sequences from 2048 on (moved as they are) and from 16384 on (converted)
@pytest.mark.parametrize("src,dtype,h,d,tokens", [
    ("bf16", "bf16", 64, 128, 4), ("bf16", "bf16", 20, 24, 15), ("f32", "f32", 16, 128, 17), ("bf16", "bf16", 8, 64, 40),
    ("bf16", "bf16", 256, 20, 8), ("f32", "f32", 70, 33, 40), ("f32", "bf16", 130, 128, 16), ("bf16", "f32", 60, 24, 40),
    ("f32", "bf16", 256, 33, 9)])
def test_appends_by_pages(src, dtype, h, d, tokens):
    lib = _abi.load()
    rng = np.random.default_rng(h + d)
    starts = np.array([0, 5, 16, 31, 64, 80, -3, 79], np.int32)
    c = Cache(rng, starts, 80, h, d, 16, dtype, poison=False).upload(starts)
    table = c.table.copy()
    table[1, 1] = -1
    c.td = dev(table)
    k, v = (rng.standard_normal((8, h, tokens, d)).astype(np.float32) for _ in range(2))
    if src == "bf16":
        k, v = oracle.round_bf16(k), oracle.round_bf16(v)
    to = (lambda x: dev(oracle.to_bf16_bits(x).view(np.int16))) if src == "bf16" else dev
    kd, vd = to(k), to(v)
    _abi.check(lib.sfg_hip_kv_append_pool_v1(
        kd.data_ptr(), vd.data_ptr(), BF16 if src == "bf16" else F32, c.kd.data_ptr(), c.vd.data_ptr(),
        BF16 if dtype == "bf16" else F32, c.td.data_ptr(), c.ld.data_ptr(), 0, 0, 8, h, tokens, d, 16, c.per, c.pages, stream()))
    for got, was, new in zip(c.logical(c.kd, c.vd), (c.k, c.v), (k, v)):
        want = was.copy()
        for n in range(8):
            for t in range(tokens):
                at = starts[n] + t
                if 0 <= at < 80 and table[n, at // 16] >= 0:
                    want[n, :, at] = c.round(new[n, :, t])
        np.testing.assert_array_equal(got, want)


def test_more_heads_than_a_launch_by_pages_holds():
    lib = _abi.load()
    b, h, t = 257, 65535, 8  # 2^24 (sequence, head)s and more
    k = torch.zeros((b, h, t, 1), dtype=torch.int16, device="cuda")
    k[-1] = torch.arange(h * t, device="cuda").remainder(30000).to(torch.int16).view(h, t, 1)
    v = k + 1
    kp, vp = (torch.full((1, h, 16), -1, dtype=torch.int16, device="cuda") for _ in range(2))
    table = torch.full((b, 1), -1, dtype=torch.int32, device="cuda")
    table[-1] = 0
    _abi.check(lib.sfg_hip_kv_append_pool_v1(k.data_ptr(), v.data_ptr(), BF16, kp.data_ptr(), vp.data_ptr(), BF16, table.data_ptr(),
                                             None, 5, 0, b, h, t, 1, 16, 1, 1, stream()))
    for got, new in ((kp, k), (vp, v)):
        want = np.full((h, 16), -1, np.int16)
        want[:, 5:13] = host(new[-1])[..., 0]
        np.testing.assert_array_equal(host(got)[0], want)
