"""Attention over an 8-bit cache under bounds much larger than the step (GPU only)."""
from __future__ import annotations

import numpy as np
import pytest

from schedforge_amd import quantized_kv as qk

import _kv8 as plain

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
BF16, F32 = torch.bfloat16, torch.float32


def dev(a, dtype):
    return torch.from_numpy(np.ascontiguousarray(a)).to(dtype).cuda()


def bounded(rng, lens, heads, d, pt, kind, capacity, spare=3):
    """A cache of a capacity far over its sequences' lengths, codes and scales drawn as they are."""
    need = [-(-n // pt) for n in lens]
    cache = qk.QuantizedKVCache(qk.QuantizedKVConfig(len(lens), heads, d, pt, capacity, sum(need) + spare, kind))
    model = plain.Cache(cache.num_pages, heads, pt, d, kind)
    model.codes[:] = rng.integers(0, 256, model.codes.shape)
    model.codes[model.codes & 0x7F == 0x7F] = 3                       # (e4m3's NaN)
    model.scales[:] = np.exp(rng.standard_normal(model.scales.shape)) * (0.02 if kind == "int8" else 0.01)
    ids, at = rng.permutation(cache.num_pages), 0
    tables = []
    for b, n in enumerate(need):
        tables.append(ids[at: at + n])
        cache.page_table[b, :n] = dev(tables[-1], torch.int32)
        at += n
    model.upload(cache)
    cache.seq_lens.copy_(dev(lens, torch.int32))
    return cache, model, tables


def queries(rng, rows, hq, d, dtype):
    """Rows of the type, on the device and (the step's own) in float64."""
    q = torch.zeros((rows, hq, d), dtype=dtype, device="cuda")
    q[:64] = dev(rng.standard_normal((64, hq, d)).astype(np.float32), dtype)
    return q, q[:64].double().cpu().numpy()


# rows of the bound, capacity: the costs of a sequence at both bounds pass what 32-bit sums hold, or just do not
LONG_BOUNDS = [(BF16, 32, 8, 128, 16, 8192, 1 << 20), (BF16, 64, 8, 64, 16, 32768, 1 << 17), (F32, 8, 2, 64, 32, 8192, 1 << 20),
               (BF16, 32, 8, 128, 16, 8000, 1 << 20)]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,hq,hkv,d,pt,rows,capacity", LONG_BOUNDS)
def test_long_bounds_stay_on_the_matrix_cores(dtype, hq, hkv, d, pt, rows, capacity, kind):
    """Lengths of thousands under bounds that a captured call may have: right, and where nothing is split the same bits as
    under bounds of the lengths' size, so from the same kernel."""
    rng = np.random.default_rng(rows + d)
    lens, own = [1500, 7, 0, 640], [1, 5, 0, 33]
    cache, model, tables = bounded(rng, lens, hkv, d, pt, kind, capacity)
    q, q64 = queries(rng, rows, hq, d, dtype)
    starts = np.concatenate(([0], np.cumsum(own)))
    at = dev(starts, torch.int32)
    out = torch.full_like(q, 9.0)
    qk.quantized_attention(cache, q, at, out=out)
    got = out[: starts[-1]].double().cpu().numpy()
    assert (out[starts[-1]:] == 9.0).all()
    for b, n in enumerate(lens):
        if own[b]:
            k, v = model.tokens(tables[b], n)
            t = slice(starts[b], starts[b + 1])
            want, off = plain.attend64(q64[t], k, v, n, d ** -0.5, dtype == F32)
            plain.close(got[t], want, off, plain.HALF[dtype])
    whole = qk.quantized_attention(cache, q, at, kv_splits=1)
    near = qk.quantized_attention(cache, q, at, kv_splits=1, max_context=2048)
    assert torch.equal(whole[: starts[-1]], near[: starts[-1]])


@pytest.mark.parametrize("dtype,d,pt", [(BF16, 128, 16), (F32, 64, 32), (BF16, 80, 16)])
def test_one_workspace_for_all_steps(dtype, d, pt):
    """A workspace of the largest step and the capacity serves every smaller call, with the bits that its own gives."""
    rng = np.random.default_rng(d)
    hq, hkv, most = 16, 4, 6000
    lens = [3000, 900, 64, 1, 2049]
    cache, _, _ = bounded(rng, lens, hkv, d, pt, "int8", 8192)
    q = torch.from_numpy(rng.standard_normal((most, hq, d)).astype(np.float32)).to(dtype).cuda()
    ws = torch.empty(qk.attention_workspace(cache, most, hq, dtype), dtype=torch.uint8, device="cuda")
    for own, rows, context in (([1] * 5, 1, None), ([1] * 5, 1, 3000), ([1] * 5, 1, 500), ([1] * 5, 5, None), ([3, 1, 9, 0, 4], 9, None),
                               ([600, 3, 1, 1, 70], 600, None), ([2500, 800, 1, 1, 2000], 2500, None), ([1, 2, 0, 0, 3], 4096, None)):
        starts = dev(np.concatenate(([0], np.cumsum(own))), torch.int32)
        for total in sorted({max(sum(own), rows), most}):
            more = dict(max_rows=rows, max_context=context)
            got = qk.quantized_attention(cache, q[:total], starts, workspace=ws, **more)
            need = qk.attention_workspace(cache, total, hq, dtype, **more)
            assert need <= ws.numel()
            want = qk.quantized_attention(cache, q[:total], starts, **more)
            assert torch.equal(torch.nan_to_num(got[: sum(own)].float(), 7.0), torch.nan_to_num(want[: sum(own)].float(), 7.0))
