"""Rotary positions of one head so small that a row is a single unit of work: queries alone, keys alone (GPU only)."""
from __future__ import annotations

import numpy as np
import pytest

from schedforge_amd import quantized_kv as qk

import _kv8 as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
BF16, F32 = torch.bfloat16, torch.float32

SMALL = [  # type, heads, head dim, rotary dim, layout
    (BF16, 1, 16, 16, "half"), (BF16, 1, 8, 8, "interleaved"), (F32, 1, 8, 8, "half"), (F32, 1, 4, 4, "interleaved"),
    (BF16, 1, 2, 2, "half"), (F32, 1, 2, 2, "half"), (BF16, 1, 2, 2, "interleaved"), (F32, 1, 2, 2, "interleaved"),
    # two units a row: two heads, or a copied part beside the paired one
    (BF16, 2, 16, 16, "half"), (F32, 2, 2, 2, "half"), (BF16, 1, 24, 16, "half"), (F32, 1, 3, 2, "interleaved")]


@pytest.mark.parametrize("t", [1, 2, 100, 1025, 5000])
@pytest.mark.parametrize("dtype,heads,d,rotary,layout", SMALL)
def test_rows_of_one_unit(dtype, heads, d, rotary, layout, t):
    rng = np.random.default_rng(t + d)
    x = torch.from_numpy(rng.standard_normal((t, heads, d)).astype(np.float32)).to(dtype).cuda()
    pos = rng.integers(0, 1 << 20, t)
    if t > 3:
        pos[[1, t - 2]] = -1
    at = torch.from_numpy(pos).to(torch.int32).cuda()
    a = qk.RotaryAngles(rotary, 10000.0)
    live = pos >= 0
    want, size = plain.rotate64(x.double().cpu().numpy()[live], pos[live], a.inv_freq, 1.0, layout == "interleaved")
    # the angle in turns to 2^-25 (fp32 of 1/2) and 2^-33 (its fixed point), sine and cosine to 4 ulp, two products and a sum
    off = size * (2 * np.pi * (2.0 ** -25 + 2.0 ** -32) + 4 * 2.0 ** -23 + 4 * 2.0 ** -24)
    for name in ("q", "k"):
        out = torch.full_like(x, 7.0)
        qk.rotate(a, at, layout=layout, **{name: x, name + "_out": out})
        got = out.double().cpu().numpy()
        plain.close(got[live], want, off, plain.HALF[dtype])
        assert (got[~live] == 7.0).all()
        y = x.clone()
        qk.rotate(a, at, layout=layout, **{name: y, name + "_out": y})
        assert torch.equal(y[at >= 0], out[at >= 0]) and torch.equal(y[at < 0], x[at < 0])
