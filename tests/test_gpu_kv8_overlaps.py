"""Outputs between the rows of inputs, and outputs over them, in a step over an 8-bit cache (GPU only)."""
from __future__ import annotations

import numpy as np
import pytest

from schedforge_amd import quantized_kv as qk

from test_gpu_kv8 import dev, random_cache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
BF16, F32 = torch.bfloat16, torch.float32
T, HQ, D = 9, 4, 64
W = HQ * D


def buffer(dtype):
    x = torch.from_numpy(np.random.default_rng(2).standard_normal((T, 6 * W)).astype(np.float32)).to(dtype).cuda()
    q = x[:, :W].view(T, HQ, D)
    beside = x[:, 2 * W: 3 * W].view(T, HQ, D)                        # the same rows, other columns
    # two rows of the buffer apart, four of them
    skipping = x.view(-1)[4 * W:].as_strided((4, HQ, D), (12 * W, D, 1))
    return x, q, beside, skipping


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotate(dtype):
    x, q, beside, skipping = buffer(dtype)
    a, pos = qk.RotaryAngles(D), torch.arange(T, dtype=torch.int32, device="cuda")
    want, _ = qk.rotate(a, pos, q)
    before = x.clone()
    qk.rotate(a, pos, q, q_out=beside)
    assert torch.equal(beside, want)
    before[:, 2 * W: 3 * W] = want.view(T, W)
    assert torch.equal(x, before)
    qk.rotate(a, pos[:4], q[:4], q_out=skipping)
    assert torch.equal(skipping, want[:4])
    for bad in (x[:, D: W + D].view(T, HQ, D), x[:, W // 2: W // 2 + W].view(T, HQ, D)):
        with pytest.raises(ValueError, match="overlap"):
            qk.rotate(a, pos, q, q_out=bad)
    with pytest.raises(ValueError, match="overlap"):
        qk.rotate(a, pos, q, beside, q_out=beside)
    with pytest.raises(ValueError, match="overlap"):
        qk.rotate(a, pos, q, beside, q_out=q, k_out=q)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_attention(dtype):
    x, q, beside, skipping = buffer(dtype)
    cache, _, _ = random_cache(np.random.default_rng(3), [300, 40], 2, D, 16, "int8")
    starts = dev([0, 5, T], torch.int32)
    want = qk.quantized_attention(cache, q, starts)
    qk.quantized_attention(cache, q, starts, out=beside)
    assert torch.equal(beside, want)
    want = qk.quantized_attention(cache, q[:4], starts)
    qk.quantized_attention(cache, q[:4], starts, out=skipping)
    assert torch.equal(skipping, want)
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    over = ws[: 2 * T * W * x.element_size()].view(dtype)[: T * W].view(T, HQ, D)
    for more in (dict(out=x[:, D: W + D].view(T, HQ, D)), dict(out=over, workspace=ws, kv_splits=3)):
        with pytest.raises(ValueError, match="overlap"):
            qk.quantized_attention(cache, q, starts, **more)
