"""Attention over an 8-bit cache: prompts of many blocks of columns, and each decode kernel under the bounds that choose it, held to
the float64 bounds (GPU only)."""
from __future__ import annotations

import numpy as np
import pytest

from schedforge_amd import quantized_kv as qk

import _kv8 as plain
from test_gpu_kv8 import check_attention, dev, random_cache, rounded

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
BF16, F32 = torch.bfloat16, torch.float32


# q heads, kv heads, head dim, page tokens, type, codes, lengths, rows: the first sequence's blocks are 69, 132, 66 and 129,
# dealt across workgroups; the last two cases have more rows than partial results are kept for, beside a long sequence of one row
PROMPTS = [
    (32, 8, 64, 16, BF16, "fp8", [2200, 1, 700], [2200, 1, 9]),
    (32, 8, 64, 16, BF16, "int8", [4200, 3000], [4200, 1]),
    (32, 8, 64, 32, F32, "fp8", [1300, 900], [1050, 1]),
    (32, 8, 128, 16, BF16, "fp8", [4300, 40], [4100, 3]),
    (64, 8, 128, 16, BF16, "int8", [3300, 9000, 1], [3300, 1, 1]),
    (16, 8, 128, 16, F32, "int8", [7000, 9000], [6600, 1])]


@pytest.mark.parametrize("hq,hkv,d,pt,dtype,kind,lens,rows", PROMPTS)
def test_prompts_of_many_blocks(hq, hkv, d, pt, dtype, kind, lens, rows):
    """Rows on both sides of block borders, among them the 64th and 128th block's, and every other sequence's."""
    rng = np.random.default_rng(sum(lens) + hq)
    cache, model, table = random_cache(rng, lens, hkv, d, pt, kind)
    starts = np.concatenate(([0], np.cumsum(rows)))
    total = int(starts[-1])
    q = rounded(rng, (total, hq, d), dtype, 1.3)
    out = torch.full((total + 2, hq, d), 9.0, dtype=dtype, device="cuda")
    qd = torch.zeros((total + 2, hq, d), dtype=dtype, device="cuda")
    qd[:total] = dev(q, dtype)
    qk.quantized_attention(cache, qd, dev(starts, torch.int32), max_rows=max(rows), out=out)
    got = out.double().cpu().numpy()
    assert not np.isnan(got).any() and (got[total:] == 9.0).all()
    a_block = (128 if dtype == BF16 else 64) * hkv // hq                 # rows
    for b, (n, r) in enumerate(zip(lens, rows)):
        k, v = model.tokens(table[b], n)
        borders = [x * a_block for x in (0, 1, 2, 31, 63, 64, 65, 127, 128, 129)] + [r]
        picked = sorted({(max(x - 2, 0), min(x + 2, r)) for x in borders if x - 2 < r})
        for i, j in picked:
            seen = n - r + j                                             # tokens that row j - 1 sees
            want, off = plain.attend64(q[starts[b] + i: starts[b] + j].astype(np.float64), k[:, :seen], v[:, :seen], seen, d ** -0.5, dtype == F32)
            plain.close(got[starts[b] + i: starts[b] + j], want, off, plain.HALF[dtype])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,pt", [(8, 2, 128, 16), (4, 1, 64, 16), (3, 3, 128, 64), (16, 1, 64, 32), (24, 1, 128, 16), (32, 8, 128, 32)])
def test_decode_under_a_bound_of_one_row(hq, hkv, d, pt, dtype, kind):
    """max_rows of 1: sixteen columns a wave where the heads of a group fit."""
    rng = np.random.default_rng(hq * 5 + d + pt)
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 130, 301, 700, 1500, 12]
    cache, model, table = random_cache(rng, lens, hkv, d, pt, kind)
    for context in (None, 1500):
        check_attention(cache, model, table, lens, [1] * 12 + [0], hq, dtype, rng, max_rows=1, max_context=context)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,pt,rows,context", [(8, 2, 16, 1, 500), (8, 2, 48, 1, 512), (16, 4, 64, 4, 257), (4, 4, 16, 1, 320), (16, 1, 32, 1, 450)])
def test_short_contexts_by_eight_waves(hq, hkv, pt, rows, context, d, kind):
    """Bounds of five to eight tiles and at most 16 columns: a tile a wave, nothing split."""
    rng = np.random.default_rng(context + d)
    lens = [context, 1, 0, 63, 64, 65, 128, 200, min(321, context), context - 1]
    cache, model, table = random_cache(rng, lens, hkv, d, pt, kind)
    own = [min(rows, 1 + b % rows) for b in range(len(lens))]
    check_attention(cache, model, table, lens, own, hq, BF16, rng, max_rows=rows, max_context=context)
    assert qk.attention_workspace(cache, sum(own) + 2, hq, BF16, max_rows=rows, max_context=64) == 0


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("d,pt", [(64, 16), (128, 16), (128, 32)])
def test_many_short_sequences_by_four_heads(d, pt, kind):
    """So many tiles that a workgroup's waves take four heads, beside sequences of no token and of one."""
    rng = np.random.default_rng(d + pt)
    lens = [int(n) for n in rng.integers(0, 2500, 64)] + [0, 1, 64, 2500]
    cache, model, table = random_cache(rng, lens, 8, d, pt, kind)
    check_attention(cache, model, table, lens, [1] * len(lens), 32, BF16, rng, max_rows=1)
