"""The workspace of attention over an 8-bit cache, by the host's query: what serves a call's bounds serves every shorter one
(no GPU needed)."""
from __future__ import annotations

import ctypes
import itertools
import random

import pytest

from schedforge_amd import _abi

MIB = 1 << 20


def workspace(lib, model, types, batch, tokens, max_rows, context, page=16, splits=0):
    hq, hkv, d = model
    a = _abi.Kv8AttnArgs()
    a.q_dtype, a.out_dtype = types
    a.pool_dtype, a.batch, a.tokens, a.max_rows = _abi.I8, batch, tokens, max_rows
    a.q_heads, a.kv_heads, a.head_dim, a.page_tokens = hq, hkv, d, page
    a.pages_per_seq, a.num_pages, a.max_context, a.kv_splits = max(1, -(-context // page)), 1 << 20, context, splits
    return lib.sfg_hip_attn_kv8_workspace_v1(ctypes.byref(a))


MODELS = [(32, 8, 128), (16, 4, 64), (64, 8, 128), (64, 64, 64), (4, 1, 64), (128, 4, 128), (32, 8, 80), (3, 1, 33), (24, 8, 256)]
TYPES = [(_abi.BF16, _abi.BF16), (_abi.BF16, _abi.F32), (_abi.F32, _abi.F32)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("model", MODELS)
@pytest.mark.parametrize("splits", [0, 1, 2, 7, 1000])
def test_shorter_bounds_need_no_more(model, types, splits):
    lib = _abi.load()
    rng = random.Random(str((model, types, splits)))
    contexts = [0, 1, 64, 100, 256, 500, 512, 513, 1000, 2000, 8192, 40000, 131072, 1 << 20]
    for batch in (1, 3, 16, 64, 300):
        most = min(1 << 16, ((1 << 22) - 1) // model[0])
        rows = sorted({1, 2, 4, 5, 8, 9, 16, 17, 64, 500, 2048, 4096, 8192, 32768, most} & set(range(1, most + 1)))
        for _ in range(60):
            r, r2 = (rng.choice(rows) for _ in range(2))
            t, t2 = (min(most, max(batch, x) + rng.choice((0, 1, 63, 64 * rng.randrange(1, 100)))) for x in (r, r2))
            big = (max(t, t2), max(r, r2), rng.choice(contexts))
            small = (min(t, t2), min(r, r2, min(t, t2)), rng.choice([c for c in contexts if c <= big[2]]))
            need = [workspace(lib, model, types, batch, *x, splits=splits) for x in (big, small)]
            assert need[1] <= need[0], (batch, big, small, need)


def test_steps_of_one_capacity():
    """The workspace of the largest step serves the decode step and the chunks of the same cache."""
    lib = _abi.load()
    steps = [(64, 1), (64, 64), (519, 512), (2048, 2048), (3900, 3900), (4096, 4096), (4096, 1), (8192, 8192), (65536, 65536)]
    for context in (8192, 131072, 1 << 20):
        need = {s: workspace(lib, (32, 8, 128), TYPES[0], 64, *s, context) for s in steps}
        for a, b in itertools.product(steps, steps):
            if a[0] <= b[0] and a[1] <= b[1]:
                assert need[a] <= need[b], (a, b, need)
        assert need[65536, 65536] <= 128 * MIB               # and it is bounded, unless kv_splits asks for more


def test_calls_that_split_nothing_need_none():
    lib = _abi.load()
    assert workspace(lib, (32, 8, 128), TYPES[0], 4, 4, 1, 128) == 0          # two tiles
    assert workspace(lib, (32, 8, 128), TYPES[0], 4, 400, 100, 8192, splits=1) == 0
    assert workspace(lib, (32, 8, 80), TYPES[0], 4, 4, 1, 192) == 0
    assert workspace(lib, (32, 8, 80), TYPES[0], 4, 4, 1, 1 << 20, splits=1) == 0
