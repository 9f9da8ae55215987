"""What schedforge_amd.quantized_kv answers and refuses before anything runs (no GPU needed: tensors and caches of the host)."""
from __future__ import annotations

import pytest

from schedforge_amd import quantized_kv as qk

torch = pytest.importorskip("torch")
BF16, F32 = torch.bfloat16, torch.float32


def cache(heads=2, d=64):
    return qk.QuantizedKVCache(qk.QuantizedKVConfig(4, heads, d, 16, 4096, 32), device="cpu")


def test_gradients_are_refused():
    """The outputs carry none, so rows that ask for them are not taken silently."""
    q, k = torch.ones(4, 4, 64, requires_grad=True), torch.ones(4, 2, 64)
    a, pos = qk.RotaryAngles(64, device="cpu"), torch.zeros(4, dtype=torch.int32)
    for call in (lambda: qk.rotate(a, pos, q), lambda: qk.rotate(a, pos, k, q), lambda: qk.rotate(a, pos, k=q * 2.0),
                 lambda: qk.rotate(a, pos, k, q_out=torch.ones(4, 2, 64, requires_grad=True)),
                 lambda: qk.quantized_attention(cache(), q), lambda: qk.quantized_attention(cache(), q.detach(), out=torch.ones(4, 4, 64, requires_grad=True))):
        with pytest.raises(ValueError, match="gradient"):
            call()


def test_gradients_that_nobody_asks_for():
    """Under no_grad, and detached, the same rows get as far as the device."""
    q = torch.ones(4, 4, 64, requires_grad=True)
    a, pos = qk.RotaryAngles(64, device="cpu"), torch.zeros(4, dtype=torch.int32)
    calls = (lambda x: qk.rotate(a, pos, x), lambda x: qk.quantized_attention(cache(), x))
    for call in calls:
        for grad, x in ((False, q), (True, q.detach())):
            with torch.set_grad_enabled(grad), pytest.raises(Exception) as e:
                call(x)                                               # (a device of the host cannot run it)
            assert "gradient" not in str(e.value)


def test_workspace_of_another_output_type():
    """bf16 queries with an fp32 output run on other kernels, whose workspace is larger at some sizes."""
    c = cache(2, 128)
    same, other = (qk.attention_workspace(c, 64, 16, BF16, max_rows=16, out_dtype=t) for t in (BF16, F32))
    assert qk.attention_workspace(c, 64, 16, BF16, max_rows=16) == same != other
    assert qk.attention_workspace(c, 64, 16, F32, max_rows=16) == other == qk.attention_workspace(c, 64, 16, F32, max_rows=16, out_dtype=BF16)


def test_workspace_refusals():
    c = cache()
    for more in (dict(dtype=torch.float16), dict(dtype="bf16"), dict(dtype=BF16, out_dtype=torch.int8), dict(dtype=BF16, starts=None, tokens=7),
                 dict(dtype=BF16, q_heads=3)):
        with pytest.raises(ValueError):
            qk.attention_workspace(c, **{"tokens": 8, "q_heads": 4, **more})
