"""Outputs that overlap what a call reads or writes besides are refused on the host; rows that lie between each other without
meeting are not (no GPU needed: the pointers are never followed)."""
from __future__ import annotations

import random

import pytest

from schedforge_amd import _abi

from test_kv8_refusals import ATTN, ROPE, SHAPE, filled

MIB = 1 << 20
# 3 rows of 4 and 2 heads of 128 in bf16, positions, turns
APART = dict(ROPE, q=1 * MIB, k=2 * MIB, q_out=3 * MIB, k_out=4 * MIB, positions=5 * MIB, turns=6 * MIB)
# 6 rows of 4 heads of 128 in bf16; 16 pages of 2 heads, 16 tokens of 128
STEP = dict(ATTN, q=1 * MIB, out=2 * MIB, k_pool=3 * MIB, v_pool=4 * MIB, scales=5 * MIB, page_table=6 * MIB, seq_lens=7 * MIB, starts=8 * MIB)


@pytest.fixture(scope="module")
def lib():
    return _abi.load()


@pytest.mark.parametrize("bad", [
    dict(q_out=2 * MIB), dict(k_out=1 * MIB), dict(q_out=1 * MIB + 2), dict(q_out=1 * MIB + 1024), dict(q_out=1 * MIB - 1024 * 2),
    dict(q_out=4 * MIB), dict(k_out=3 * MIB + 1024 + 1022), dict(q_out=5 * MIB - 3072 + 2), dict(k_out=5 * MIB + 8), dict(k_out=6 * MIB + 508),
    dict(q_out=1 * MIB, k_out=1 * MIB + 1024),                        # in place, but the keys over the queries
    dict(q_out=1 * MIB, k=1 * MIB + 1022), dict(q_out=1 * MIB + 512, q_out_stride=1024), dict(k=None, k_out=None, kv_heads=0, q_out=1 * MIB + 1022)])
def test_rope(lib, bad):
    assert lib.sfg_hip_rope_v1(filled(_abi.RopeArgs, APART, bad), None) == SHAPE
    assert b"overlap" in lib.sfg_hip_last_error()


@pytest.mark.parametrize("bad", [
    dict(out=1 * MIB + 16), dict(out=1 * MIB - 5 * 1024), dict(out=3 * MIB + 16 * 2 * 16 * 128 - 2), dict(out=4 * MIB), dict(out=5 * MIB - 6 * 1024 + 2),
    dict(out=5 * MIB + 16 * 2 * 8 - 2), dict(out=6 * MIB + 4 * 8 * 2 - 2), dict(out=7 * MIB + 4), dict(out=8 * MIB + 8), dict(out=1 * MIB + 1022, out_stride=1024, q_stride=1024),
    dict(out=1 * MIB + 1026, out_stride=4096, out_dtype=_abi.F32), dict(tokens=1, max_rows=1, starts=None, seq_lens=None, batch=1, out=1 * MIB + 1022)])
def test_attention(lib, bad):
    assert lib.sfg_hip_attn_kv8_v1(filled(_abi.Kv8AttnArgs, STEP, bad), None, 0, None) == SHAPE
    assert b"overlap" in lib.sfg_hip_last_error()


def test_workspace(lib):
    more = dict(max_context=128 * 16, pages_per_seq=128, kv_splits=4)
    need = lib.sfg_hip_attn_kv8_workspace_v1(filled(_abi.Kv8AttnArgs, STEP, more))
    assert need > 0
    for at in (2 * MIB - need + 16, 2 * MIB, 1 * MIB + 5120, 3 * MIB, 4 * MIB, 5 * MIB, 6 * MIB, 7 * MIB, 8 * MIB):
        assert lib.sfg_hip_attn_kv8_v1(filled(_abi.Kv8AttnArgs, STEP, more), at // 16 * 16, need, None) == SHAPE, at
        assert b"overlap" in lib.sfg_hip_last_error()


def meet(a, b):
    """Rows (start, stride, bytes, count) one by one."""
    for i in range(a[3]):
        for j in range(b[3]):
            x, y = a[0] + i * a[1], b[0] + j * b[1]
            if x < y + b[2] and y < x + a[2]:
                return True
    return False


def test_rows_by_rows(lib):
    """Random rows of queries and outputs, side by side or not, against all pairs of rows."""
    torch = pytest.importorskip("torch")
    if torch.cuda.is_available():
        pytest.skip("calls that are taken would run")
    rng = random.Random(4)
    seen = {True: 0, False: 0}
    for _ in range(3000):
        tokens, heads, d = rng.randrange(1, 7), rng.randrange(1, 3), 2 * rng.randrange(1, 3)
        w = heads * d
        strides = [rng.randrange(w, 6 * w + 1) for _ in range(2)]
        if rng.random() < 0.4:
            strides[1] = strides[0]
        es = rng.choice((2, 4))
        at = [64 * 1024 + es * rng.randrange(0, 60) for _ in range(2)]
        if at[0] == at[1]:
            continue
        rows = [(at[i], strides[i] * es, w * es, tokens) for i in (0, 1)]
        want = meet(*rows)
        a = filled(_abi.RopeArgs, ROPE, dict(q=at[0], q_out=at[1], q_stride=strides[0], q_out_stride=strides[1], k=None, k_out=None, kv_heads=0,
                                            dtype=_abi.BF16 if es == 2 else _abi.F32, tokens=tokens, q_heads=heads, head_dim=d,
                                            rotary_dim=2, positions=1 << 20, turns=1 << 21))
        rc = lib.sfg_hip_rope_v1(a, None)
        assert (rc == SHAPE and b"overlap" in lib.sfg_hip_last_error()) == want, rows
        seen[want] += 1
    assert min(seen.values()) > 200, seen
