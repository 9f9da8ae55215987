"""Refusals of the operators of a step over an 8-bit paged cache: invalid arguments come back from the host with the
documented code and a message, before anything is launched (no GPU needed: the pointers are never followed).  The
host's rotary angles against their formulas."""
from __future__ import annotations

import ctypes
import math
from fractions import Fraction

import numpy as np
import pytest

from schedforge_amd import _abi

CONFIG, SHAPE, GUARD, UNSUPPORTED, WORKSPACE = (_abi.ERR_INVALID_CONFIG, _abi.ERR_SHAPE, _abi.ERR_GUARD,
                                                _abi.ERR_UNSUPPORTED, _abi.ERR_WORKSPACE)


@pytest.fixture(scope="module")
def lib():
    return _abi.load()


def filled(struct, base, more):
    a = struct()
    for k, v in {**base, **more}.items():
        setattr(a, k, v)
    return ctypes.byref(a)


PLAN = dict(keep=None, counts=1 << 12, seq_lens=2 << 12, page_table=3 << 12, free_pages=4 << 12, free_count=5 << 12,
            starts=6 << 12, positions=7 << 12, slots=8 << 12, batch=4, pages_per_seq=8, num_pages=32, page_tokens=16, max_tokens=64)
ROPE = dict(q=64, k=1 << 20, q_out=2 << 20, k_out=3 << 20, dtype=_abi.BF16, q_stride=512, k_stride=256, q_out_stride=512, k_out_stride=256,
            positions=64, turns=64, magnitude=1.0, layout=_abi.ROPE_HALF, tokens=3, q_heads=4, kv_heads=2, head_dim=128, rotary_dim=128)
APPEND = dict(keys=64, values=64, dtype=_abi.BF16, key_stride=256, value_stride=256, k_pool=64, v_pool=64, pool_dtype=_abi.I8,
              scales=64, slots=64, tokens=3, kv_heads=2, head_dim=128, page_tokens=16, num_pages=8)
ATTN = dict(q=64, q_dtype=_abi.BF16, q_stride=512, out=128, out_dtype=_abi.BF16, out_stride=512, k_pool=64, v_pool=64,
            pool_dtype=_abi.FP8, scales=64, page_table=64, seq_lens=None, starts=64, batch=2, tokens=6, max_rows=4, q_heads=4,
            kv_heads=2, head_dim=128, page_tokens=16, pages_per_seq=8, num_pages=16, max_context=100, kv_splits=0, scale=0.0)


@pytest.mark.parametrize("bad,code", [
    (dict(counts=None), CONFIG), (dict(seq_lens=None), CONFIG), (dict(page_table=None), CONFIG), (dict(free_pages=None), CONFIG),
    (dict(free_count=None), CONFIG), (dict(starts=None), CONFIG), (dict(positions=None), CONFIG), (dict(slots=None), CONFIG),
    (dict(batch=0), CONFIG), (dict(pages_per_seq=0), CONFIG), (dict(num_pages=0), CONFIG), (dict(page_tokens=0), CONFIG),
    (dict(max_tokens=0), CONFIG), (dict(max_tokens=-1), CONFIG), (dict(page_tokens=1 << 30), UNSUPPORTED),
    (dict(pages_per_seq=1 << 27), UNSUPPORTED), (dict(num_pages=1 << 31), UNSUPPORTED), (dict(batch=1 << 21), UNSUPPORTED),
    (dict(batch=1 << 19, pages_per_seq=1 << 13), UNSUPPORTED), (dict(max_tokens=1 << 22), UNSUPPORTED),
    (dict(starts=2 << 12), SHAPE), (dict(keep=3 << 12), SHAPE), (dict(counts=(6 << 12) + 16), SHAPE),
    (dict(keep=(2 << 12) + 4), SHAPE), (dict(free_count=(4 << 12) + 124), SHAPE)])
def test_plan(lib, bad, code):
    assert lib.sfg_hip_kv_plan_v1(filled(_abi.KvPlanArgs, PLAN, bad), None) == code, lib.sfg_hip_last_error()
    assert lib.sfg_hip_last_error()


@pytest.mark.parametrize("bad,code", [
    (dict(positions=None), CONFIG), (dict(turns=None), CONFIG), (dict(tokens=0), CONFIG), (dict(q_heads=-1), CONFIG),
    (dict(q_heads=0, kv_heads=0), CONFIG), (dict(head_dim=0), CONFIG), (dict(rotary_dim=0), CONFIG), (dict(rotary_dim=63), CONFIG),
    (dict(rotary_dim=130), CONFIG), (dict(magnitude=math.nan), CONFIG), (dict(magnitude=math.inf), CONFIG), (dict(dtype=_abi.I8), UNSUPPORTED),
    (dict(dtype=_abi.FP8), UNSUPPORTED), (dict(layout=2), UNSUPPORTED), (dict(tokens=1 << 22), UNSUPPORTED),
    (dict(q_heads=1 << 16), UNSUPPORTED), (dict(head_dim=1026), UNSUPPORTED),
    (dict(q=None), SHAPE), (dict(k_out=None), SHAPE), (dict(q_heads=0), SHAPE), (dict(q_stride=511), SHAPE),
    (dict(k_out_stride=255), SHAPE), (dict(q_stride=1 << 31), SHAPE), (dict(q_out=64, q_out_stride=1024), SHAPE)])
def test_rope(lib, bad, code):
    assert lib.sfg_hip_rope_v1(filled(_abi.RopeArgs, ROPE, bad), None) == code, lib.sfg_hip_last_error()


@pytest.mark.parametrize("bad,code", [
    *[({n: None}, CONFIG) for n in ("keys", "values", "k_pool", "v_pool", "scales", "slots")],
    *[({n: 0}, CONFIG) for n in ("tokens", "kv_heads", "head_dim", "page_tokens", "num_pages")],
    (dict(dtype=_abi.I8), UNSUPPORTED), (dict(pool_dtype=_abi.BF16), UNSUPPORTED), (dict(pool_dtype=_abi.I32), UNSUPPORTED),
    (dict(head_dim=257), UNSUPPORTED), (dict(tokens=1 << 22), UNSUPPORTED), (dict(kv_heads=1 << 16), UNSUPPORTED),
    (dict(page_tokens=1 << 23), UNSUPPORTED), (dict(num_pages=1 << 31), UNSUPPORTED), (dict(key_stride=255), SHAPE),
    (dict(value_stride=255), SHAPE), (dict(value_stride=1 << 31), SHAPE)])
def test_append(lib, bad, code):
    assert lib.sfg_hip_kv8_append_v1(filled(_abi.Kv8AppendArgs, APPEND, bad), None) == code, lib.sfg_hip_last_error()


@pytest.mark.parametrize("bad,code", [
    *[({n: None}, CONFIG) for n in ("q", "out", "k_pool", "v_pool", "scales", "page_table")],
    *[({n: 0}, CONFIG) for n in ("batch", "tokens", "max_rows", "q_heads", "kv_heads", "head_dim", "page_tokens", "pages_per_seq", "num_pages")],
    (dict(q_heads=3), CONFIG), (dict(max_context=-1), CONFIG), (dict(q_dtype=_abi.I8), UNSUPPORTED), (dict(out_dtype=_abi.FP8), UNSUPPORTED),
    (dict(pool_dtype=_abi.BF16), UNSUPPORTED), (dict(head_dim=257), UNSUPPORTED), (dict(page_tokens=1 << 23), UNSUPPORTED),
    (dict(pages_per_seq=1 << 40), UNSUPPORTED), (dict(num_pages=1 << 31), UNSUPPORTED), (dict(batch=1 << 21), UNSUPPORTED),
    (dict(tokens=1 << 20), UNSUPPORTED), (dict(max_rows=7), SHAPE), (dict(starts=None), SHAPE), (dict(starts=None, max_rows=6), SHAPE),
    (dict(q_stride=511), SHAPE), (dict(out_stride=511), SHAPE), (dict(out=64), SHAPE), (dict(max_context=129), GUARD)])
def test_attention(lib, bad, code):
    a = filled(_abi.Kv8AttnArgs, ATTN, bad)
    assert lib.sfg_hip_attn_kv8_v1(a, None, 0, None) == code, lib.sfg_hip_last_error()


def test_attention_workspace(lib):
    """A workspace that is too small or off its boundary is refused; sizes that cannot run need none."""
    a = filled(_abi.Kv8AttnArgs, ATTN, dict(max_context=128 * 16, pages_per_seq=128, kv_splits=4))
    need = lib.sfg_hip_attn_kv8_workspace_v1(a)
    assert lib.sfg_hip_attn_kv8_workspace_v1(None) == 0
    assert lib.sfg_hip_attn_kv8_workspace_v1(filled(_abi.Kv8AttnArgs, ATTN, dict(q_heads=3))) == 0
    if need:
        assert lib.sfg_hip_attn_kv8_v1(a, None, 0, None) == WORKSPACE
        assert lib.sfg_hip_attn_kv8_v1(a, 16, need - 1, None) == WORKSPACE
        assert lib.sfg_hip_attn_kv8_v1(a, 24, need, None) == WORKSPACE


def test_null_arguments(lib):
    assert lib.sfg_hip_kv_plan_v1(None, None) == SHAPE
    assert lib.sfg_hip_rope_v1(None, None) == SHAPE
    assert lib.sfg_hip_kv8_append_v1(None, None) == SHAPE
    assert lib.sfg_hip_attn_kv8_v1(None, None, 0, None) == SHAPE


# ---------------------------------------------------------------- rotary angles
def angles(lib, rotary, **kw):
    w, f = np.empty(rotary // 2), ctypes.c_float()
    how = _abi.RopeScaling(**kw)
    rc = lib.sfg_hip_rope_inv_freq_host_v1(w.ctypes.data, ctypes.byref(f), rotary, ctypes.byref(how))
    assert rc == 0, lib.sfg_hip_last_error()
    return w, f.value


def test_angles_follow_their_formulas(lib):
    r, theta, s, ctx = 64, 10000.0, 4.0, 2048.0
    w = np.array([theta ** (-2.0 * i / r) for i in range(r // 2)])
    near = lambda a, b: np.testing.assert_allclose(a, b, rtol=1e-14)  # noqa: E731
    near(angles(lib, r, kind=_abi.ROPE_PLAIN, theta=theta)[0], w)
    near(angles(lib, r, kind=_abi.ROPE_LINEAR, theta=theta, factor=s)[0], w / s)
    base = theta * s ** (r / (r - 2.0))
    got, f = angles(lib, r, kind=_abi.ROPE_BASE, theta=theta, factor=s)
    near(got, [base ** (-2.0 * i / r) for i in range(r // 2)])
    near(got[-1], w[-1] / s)                       # the slowest pair turns s times slower, the fastest as before
    assert f == 1.0 and got[0] == 1.0
    got, _ = angles(lib, r, kind=_abi.ROPE_BANDS, theta=theta, factor=s, context=ctx, low=1.0, high=4.0)
    for i in range(r // 2):
        turns = ctx * w[i] / (2 * math.pi)
        t = (turns - 1.0) / 3.0
        want = w[i] if turns >= 4 else w[i] / s if turns <= 1 else w[i] * (t + (1 - t) / s)
        near(got[i], want)
    got, f = angles(lib, r, kind=_abi.ROPE_RAMP, theta=theta, factor=s, context=ctx, low=1.0, high=32.0)
    pair = lambda x: r * math.log(ctx / (2 * math.pi * x)) / (2 * math.log(theta))  # noqa: E731
    a, b = math.floor(pair(32.0)), math.ceil(pair(1.0))
    assert 0 < a < b < r // 2
    near(got, [w[i] * (1 - min(max((i - a) / (b - a), 0), 1) * (1 - 1 / s)) for i in range(r // 2)])
    assert f == np.float32(0.1 * math.log(s) + 1)


@pytest.mark.parametrize("bad,code", [
    (dict(kind=5), UNSUPPORTED), (dict(kind=-1), UNSUPPORTED), (dict(theta=1.0), CONFIG), (dict(theta=math.nan), CONFIG),
    (dict(factor=0.5), CONFIG), (dict(factor=math.inf), CONFIG), (dict(context=0.0), CONFIG), (dict(low=0.0), CONFIG),
    (dict(high=1.0), CONFIG)])
def test_angle_refusals(lib, bad, code):
    how = _abi.RopeScaling(**{**dict(kind=_abi.ROPE_RAMP, theta=1e4, factor=4.0, context=2048.0, low=1.0, high=32.0), **bad})
    w, f = np.empty(32), ctypes.c_float()
    assert lib.sfg_hip_rope_inv_freq_host_v1(w.ctypes.data, ctypes.byref(f), 64, ctypes.byref(how)) == code
    ok = _abi.RopeScaling(_abi.ROPE_PLAIN, 1e4)
    assert lib.sfg_hip_rope_inv_freq_host_v1(w.ctypes.data, ctypes.byref(f), 63, ctypes.byref(ok)) == SHAPE
    assert lib.sfg_hip_rope_inv_freq_host_v1(None, ctypes.byref(f), 64, ctypes.byref(ok)) == SHAPE


def test_turns_are_exact_to_the_last_bit(lib):
    """round(w 2^64 / 2 pi) modulo 2^64, against pi to 60 digits (Fraction); off by at most one."""
    pi = Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)
    w = np.array([1.0, 0.5, 10000.0 ** -0.3, 1e-7, 6.283185307179586, 7.5, -0.25, 0.0, 123456.789])
    turns = np.empty(len(w), np.uint64)
    assert lib.sfg_hip_rope_turns_host_v1(turns.ctypes.data, w.ctypes.data, len(w)) == 0
    for x, t in zip(w, turns):
        want = round(Fraction(float(x)) / (2 * pi) * 2 ** 64) % 2 ** 64
        off = (int(t) - want) % 2 ** 64
        slack = max(1, int(abs(x)))   # (the quotient's whole turns take bits of a 64-bit fraction)
        assert min(off, 2 ** 64 - off) <= slack, (x, int(t), want)
    bad = np.array([1.0, np.nan])
    assert lib.sfg_hip_rope_turns_host_v1(turns.ctypes.data, bad.ctypes.data, 2) == CONFIG
    assert lib.sfg_hip_rope_turns_host_v1(turns.ctypes.data, w.ctypes.data, 0) == SHAPE
