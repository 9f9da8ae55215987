"""A step over an 8-bit paged cache, operator by operator and together, through schedforge_amd.quantized_kv (GPU only).
Pages, slots, codes and scales are exact; rotary positions and attention are held to bounds that follow from fp32
arithmetic (_kv8.py) plus half a step of the output's type."""
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


def rounded(rng, shape, dtype, std=1.0):
    """Values of the type, as fp32."""
    return torch.from_numpy((std * rng.standard_normal(shape)).astype(np.float32)).to(dtype).float().numpy()


def make(batch, heads, d, pt, capacity, kind, pages=None):
    return qk.QuantizedKVCache(qk.QuantizedKVConfig(batch, heads, d, pt, capacity, pages, kind))


# ---------------------------------------------------------------- pages and slots
def check_plan(cache, model, counts, room, keep=None, out=None):
    want = model.step(counts, room, keep)
    got = qk.plan_step(cache, dev(counts, torch.int32), room, None if keep is None else dev(keep, torch.int32), out)
    for name, w, g in zip(("starts", "positions", "slots"), want, (got.starts, got.positions, got.slots)):
        assert g.cpu().tolist() == w, name
    assert cache.seq_lens.cpu().tolist() == model.lens
    assert cache.page_table.cpu().tolist() == model.table
    assert int(cache.free_count) == model.count
    assert cache.free_pages.cpu().tolist()[: model.count] == model.stack[: model.count]
    return got


@pytest.mark.parametrize("batch,pt,capacity,pages,room", [
    (1, 16, 100, 7, 64), (5, 16, 64, 12, 100), (64, 16, 200, 500, 64), (300, 4, 40, 1500, 3000), (1500, 3, 20, 6000, 9000),
    (1025, 1, 6, 3000, 2000), (7, 128, 3000, 40, 20000)])
def test_plans_follow_the_model(batch, pt, capacity, pages, room):
    """Steps that grow, shrink and end sequences, that run into the capacity, the rows and the free pages."""
    rng = np.random.default_rng(batch * 7 + pt)
    cache = make(batch, 1, 1, pt, capacity, "int8", pages)
    model = plain.Pages(batch, cache.config.pages_per_seq, pages, pt)
    for step in range(8):
        counts = rng.integers(-1, 2 if step % 2 else max(2, 2 * capacity // 3), batch)
        keep = None if step in (0, 3) else np.where(rng.random(batch) < 0.3, rng.integers(-2, capacity + 5, batch), 1 << 30)
        if step == 5:
            keep = np.zeros(batch, np.int64)             # all end, and begin again
        check_plan(cache, model, counts, room, keep)


def test_plan_refuses_in_order():
    """A sequence that does not fit stops the later ones that need what it waited for, and no others."""
    cache, model = make(5, 1, 1, 4, 16, "int8", 5), plain.Pages(5, 4, 5, 4)
    check_plan(cache, model, [3, 4, 0, 1, 1], 32)                     # 1 + 1 + 0 + 1 + 1 pages
    got = check_plan(cache, model, [1, 9, 4, 1, 17], 32)              # 0 fits, 1 needs 3, 2 needs 1, 3 stays on its page
    assert np.diff(got.starts.cpu().numpy()).tolist() == [1, 0, 0, 1, 0]
    got = check_plan(cache, model, [0, 0, 4, 2, 2], 5)                # rows: 4 + 2 are over 5, and so is the rest
    assert np.diff(got.starts.cpu().numpy()).tolist() == [0, 0, 4, 0, 0]


def test_plan_of_nothing_and_of_padding():
    cache, model = make(3, 1, 1, 16, 64, "int8"), plain.Pages(3, 4, 12, 16)
    got = check_plan(cache, model, [0, 0, 0], 9)
    assert (got.slots == -1).all() and (got.positions == -1).all()
    again = check_plan(cache, model, [5, 0, 1], 9, out=got)
    assert again is got and got.slots.cpu().tolist()[6:] == [-1] * 3


def test_plan_counts_beyond_32_bit_sums():
    """Requests whose sum passes 2^31, past the capacity and past the rows."""
    cache, model = make(6, 1, 1, 16, 1 << 20, "int8", 8), plain.Pages(6, (1 << 20) // 16, 8, 16)
    check_plan(cache, model, [7, 2 ** 31 - 1, 1 << 20, 1 << 20, 2 ** 31 - 1, 3], 100)


def test_plan_takes_lists_that_hold_anything():
    """Lengths, counts and free counts outside their ranges, ids outside the pool: nothing is followed."""
    cache = make(4, 1, 1, 16, 64, "int8", 6)
    cache.seq_lens.copy_(dev([-5, 1 << 30, 3, 0], torch.int32))
    cache.free_count.fill_(1 << 30)
    cache.free_pages.copy_(dev([0, 1, 2, -7, 99, 5], torch.int32))
    got = qk.plan_step(cache, dev([16, 1, 20, 16], torch.int32), 60)
    assert cache.seq_lens.cpu().tolist() == [16, 64, 23, 16]
    table = cache.page_table.cpu().tolist()
    assert table[0][0] == 5 and table[2][1] == 99 and table[3][0] == -7
    slots = got.slots.cpu().tolist()
    assert slots[:16] == list(range(80, 96)) and slots[16:] == [-1] * 44


# ---------------------------------------------------------------- rotary positions
ROPES = [  # tokens, q heads, kv heads, head dim, rotary dim
    (1, 32, 8, 128, 128), (1, 1, 1, 2, 2), (7, 4, 2, 64, 64), (130, 16, 4, 64, 16), (33, 3, 1, 80, 40), (5, 2, 2, 33, 30),
    (3, 5, 5, 256, 128), (64, 8, 8, 128, 96), (9, 1, 1, 1024, 1024), (2000, 4, 1, 128, 128), (257, 6, 3, 96, 96), (1700, 32, 8, 128, 128)]  # (the last one writes over 16 MB)


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("t,hq,hkv,d,rotary", ROPES)
def test_rotate(t, hq, hkv, d, rotary, dtype, layout):
    """Parts of wider rows, positions from 0 to 2^31 - 1, padding rows that stay as they were."""
    rng = np.random.default_rng(t + d)
    wide = rounded(rng, (t, (hq + hkv) * d + 24), dtype)
    x = dev(wide, dtype)
    q, k = x[:, 8: 8 + hq * d].view(t, hq, d), x[:, 8 + hq * d: 8 + (hq + hkv) * d].view(t, hkv, d)
    pos = rng.integers(0, 2 ** 31, t) >> rng.integers(0, 31, t)
    pos[0] = 2 ** 31 - 1 if t > 1 else 4095
    pos[t // 2] = 0 if t > 2 else pos[t // 2]
    if t > 4:
        pos[[1, t - 1]] = -1, -5
    a = qk.RotaryAngles(rotary, 500000.0, "ramp", factor=8.0, context=8192.0)
    qo, ko = torch.full((t, hq, d), 7.0, dtype=dtype, device="cuda"), torch.full((t, hkv + 1, d), 7.0, dtype=dtype, device="cuda")[:, :hkv]
    assert qk.rotate(a, dev(pos, torch.int32), q, k, layout, qo, ko) == (qo, ko)
    for src, got in ((q, qo), (k, ko)):
        src, got = src.double().cpu().numpy(), got.double().cpu().numpy()
        live = pos >= 0
        want, size = plain.rotate64(src[live], pos[live], a.inv_freq, a.magnitude, layout == "interleaved")
        # the angle in turns to 2^-25 (fp32 of 1/2) and 2^-33 (its fixed point), sine and cosine to 4 ulp, two
        # products and a sum, the magnitude
        off = size * (2 * np.pi * (2.0 ** -25 + 2.0 ** -32) + 4 * 2.0 ** -23 + 4 * 2.0 ** -24)
        plain.close(got[live], want, off, plain.HALF[dtype])
        assert (got[~live] == 7.0).all()
        assert np.array_equal(got[live][..., rotary:], src[live][..., rotary:])
    assert torch.equal(x, dev(wide, dtype))                       # the inputs stay


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("d,rotary,layout", [(128, 128, "half"), (128, 64, "interleaved"), (80, 40, "half"), (64, 64, "interleaved")])
def test_rotate_in_place_alone_and_back(dtype, d, rotary, layout):
    """Inputs as outputs give the same bits; keys alone; turning back by the negated angles."""
    rng = np.random.default_rng(d)
    x = dev(rounded(rng, (50, 6, d), dtype), dtype)
    pos = dev(rng.integers(0, 1 << 20, 50), torch.int32)
    a = qk.RotaryAngles(rotary)
    want, none = qk.rotate(a, pos, x, layout=layout)
    assert none is None
    y = x.clone()
    qk.rotate(a, pos, k=y, layout=layout, k_out=y)
    assert torch.equal(y, want)
    back, _ = qk.rotate(qk.RotaryAngles(rotary, inv_freq=-a.inv_freq), pos, y, layout=layout)
    # two turns, each rounded: sqrt(2) in the pair's size each
    size = x.double().abs().max() * 2
    assert float((back.double() - x.double()).abs().max()) <= float(size) * (2 * plain.HALF[dtype] + 2.0 ** -20)


def test_rotate_keeps_what_is_not_finite_in_its_pair():
    x = torch.ones(3, 2, 64, device="cuda", dtype=BF16)
    x[0, 0, 3], x[1, 1, 40], x[2, 0, 5] = float("nan"), float("inf"), float("-inf")
    x.view(torch.int16)[0, 1, 9] = 0x7FFF                            # a NaN of all ones
    y, _ = qk.rotate(qk.RotaryAngles(64), dev([5, 6, 7], torch.int32), x)
    bad = ~torch.isfinite(y)
    want = torch.zeros_like(bad)
    for t, h, i in ((0, 0, 3), (1, 1, 8), (2, 0, 5), (0, 1, 9)):
        want[t, h, i] = want[t, h, i + 32] = True
    assert torch.equal(bad, want)


# ---------------------------------------------------------------- appends
APPENDS = [  # heads, head dim, page tokens
    (8, 128, 16), (4, 64, 16), (2, 128, 64), (3, 64, 32), (2, 256, 16), (2, 80, 16), (1, 33, 5), (2, 128, 1), (5, 1, 7), (1, 128, 100), (1, 96, 24)]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads,d,pt", APPENDS)
def test_appends_are_exact(heads, d, pt, dtype, kind):
    """Steps of one token and of many into ragged sequences: each code and scale, and what lies around them."""
    rng = np.random.default_rng(d * 100 + pt)
    batch, capacity = 5, 7 * pt + 3
    cache = make(batch, heads, d, pt, capacity, kind)
    model = plain.Cache(cache.num_pages, heads, pt, d, kind)
    model.codes[:] = rng.integers(0, 127, model.codes.shape)         # stale codes and scales
    model.scales[:] = rng.random(model.scales.shape)
    model.upload(cache)
    for step in range(6):
        many = step in (0, 3)
        counts = rng.integers(0, 2 * pt + 3, batch) if many else rng.integers(0, 3, batch)
        room = int(counts.sum()) + 3
        plan = qk.plan_step(cache, dev(counts, torch.int32), room)
        # values that grow, whole ones among them (their quotients fall on ties), rows of zeros
        std = 4.0 ** (step - 2)
        wide = rounded(rng, (room, 3 * heads * d), dtype, std)
        keys, values = wide[:, : heads * d].reshape(room, heads, d), wide[:, 2 * heads * d:].reshape(room, heads, d)
        if step % 2:
            keys, values = np.rint(keys * 3).astype(np.float32), values * np.float32(0 if step == 1 else 1)
        x = dev(np.concatenate((keys.reshape(room, -1), values.reshape(room, -1)), 1), dtype)
        keys, values = (x[:, i * heads * d: (i + 1) * heads * d].view(room, heads, d) for i in (0, 1))
        qk.append_quantized_kv(cache, keys, values, plan.slots)
        model.append(keys.float().cpu().numpy(), values.float().cpu().numpy(), plan.slots.cpu().numpy())
        codes, scales = plain.download(cache)
        np.testing.assert_array_equal(scales, model.scales)
        np.testing.assert_array_equal(codes, model.codes)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("d", [128, 80])
def test_appends_of_extremes(d, kind):
    """Ties, the largest and smallest floats, signed zeros, a scale that underflows; NaN and infinities poison their
    page and head until its first token comes again."""
    heads, pt = 3, 16
    cache = make(1, heads, d, pt, 64, kind)
    model = plain.Cache(cache.num_pages, heads, pt, d, kind)
    rng = np.random.default_rng(3)
    big = np.float32(3.4e38)
    rows = np.zeros((6, heads, d), np.float32)
    rows[0] = (np.arange(d) - d // 2) / 2                             # halves under a scale of 1: ties
    rows[0, :, 0] = plain.MOST[kind]
    rows[1, 0], rows[1, 1], rows[1, 2] = big, -big, np.float32(1e-40)
    rows[2] = -0.0
    rows[3] = np.float32(1e-45)
    rows[4] = rng.standard_normal((heads, d))
    rows[4, 1, 7], rows[4, 2, 5] = np.nan, -np.inf
    rows[5] = 1.0

    def put(i, slot):
        x = dev(rows[i: i + 1], F32)
        y = dev(-rows[i: i + 1], F32)
        qk.append_quantized_kv(cache, x, y, dev([slot], torch.int64))
        model.append(rows[i: i + 1], -rows[i: i + 1], [slot])
        codes, scales = plain.download(cache)
        np.testing.assert_array_equal(scales, model.scales)
        np.testing.assert_array_equal(codes, model.codes)
    for page, order in enumerate(((0, 1, 2, 3), (3, 2, 0, 5), (4, 0), (2, 5, 4, 5))):
        for off, i in enumerate(order):
            put(i, page * pt + off)
    assert np.isnan(model.scales[2, 1:]).all() and not np.isnan(model.scales[2, 0]).any()
    put(5, 2 * pt)                                                   # begins the page anew
    assert not np.isnan(model.scales[2]).any()


def test_append_skips_slots_outside_the_pool():
    cache = make(1, 2, 64, 16, 64, "int8", 4)
    x = torch.ones(6, 2, 64, device="cuda")
    qk.append_quantized_kv(cache, x, x, dev([-1, 4 * 16, 2 ** 40, -2 ** 40, 63, 2 ** 63 - 1], torch.int64))
    codes, scales = plain.download(cache)
    assert (codes[3, :, :, 15] == 127).all() and (scales[3] > 0).all()
    codes[3, :, :, 15] = 0
    assert not codes.any() and not scales[:3].any()


# ---------------------------------------------------------------- attention
def filled(rng, lens, heads, d, pt, kind, spare=3):
    """A cache whose sequences hold random tokens, page ids shuffled; pages of no sequence hold NaN."""
    batch, capacity = len(lens), max(max(lens), 1) + pt
    per = -(-capacity // pt)
    need = [-(-n // pt) for n in lens]
    cache = make(batch, heads, d, pt, capacity, kind, sum(need) + spare)
    model = plain.Cache(cache.num_pages, heads, pt, d, kind)
    model.codes[:] = 0x7F                                            # e4m3: NaN
    model.scales[:] = np.nan
    ids = rng.permutation(cache.num_pages)
    table = np.full((batch, per), -1)
    at = 0
    for b, n in enumerate(lens):
        table[b, : need[b]] = ids[at: at + need[b]]
        at += need[b]
        shift = rng.standard_normal((1, heads, d)) * 0.7
        k = (rng.standard_normal((n, heads, d)) + shift) * np.exp(rng.standard_normal((n, 1, 1)) * 0.3)
        pos = np.arange(n)
        model.append(k.astype(np.float32), rng.standard_normal((n, heads, d)).astype(np.float32), table[b, pos // pt] * pt + pos % pt)
    model.upload(cache)
    cache.page_table.copy_(dev(table, torch.int32))
    cache.seq_lens.copy_(dev(lens, torch.int32))
    return cache, model, table


def check_attention(cache, model, table, lens, rows, hq, dtype, rng, out_dtype=None, scale=0.0, pad=2, std=1.3, **more):
    d = model.d
    starts = np.concatenate(([0], np.cumsum(rows)))
    total = int(starts[-1]) + pad
    q = rounded(rng, (total, hq, d), dtype, std)
    wide = torch.full((total, hq * d + 16), 5.0, dtype=dtype, device="cuda")
    wide[:, 8: 8 + hq * d] = dev(q, dtype).view(total, -1)
    out = torch.full((total, hq + 1, d), 9.0, dtype=out_dtype or dtype, device="cuda")[:, :hq]
    got = qk.quantized_attention(cache, wide[:, 8: 8 + hq * d].view(total, hq, d), dev(starts, torch.int32), out=out, scale=scale, **more)
    assert got is out
    got = got.double().cpu().numpy()
    most = more.get("max_rows") or total
    for b, n in enumerate(lens):
        t0, r = starts[b], int(rows[b])
        if not r:
            continue
        k, v = model.tokens(table[b], n)
        want, off = plain.attend64(q[t0: t0 + r].astype(np.float64), k, v, n, scale or d ** -0.5, dtype == F32 or out_dtype == F32)
        plain.close(got[t0: t0 + min(r, most)], want[:most], off[:most], plain.HALF[out_dtype or dtype])
        assert (got[t0 + min(r, most): t0 + r] == 9.0).all()
    assert (got[starts[-1]:] == 9.0).all()
    return got


SHAPES = [  # q heads, kv heads, head dim, page tokens
    (8, 2, 128, 16), (4, 1, 64, 16), (3, 3, 128, 64), (16, 1, 64, 32), (24, 1, 128, 16), (10, 2, 64, 48), (2, 1, 80, 16), (3, 1, 33, 5),
    (4, 4, 256, 16), (2, 2, 1, 1), (4, 2, 128, 8), (6, 2, 128, 20)]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,pt", SHAPES)
def test_decode_rows(hq, hkv, d, pt, dtype, kind):
    """One row a sequence, from a length of one to several hundred, page borders and odd ones; one sequence has no
    row, one has no token."""
    rng = np.random.default_rng(hq + d + pt)
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 130, 301, 500, 12]
    cache, model, table = filled(rng, lens, hkv, d, pt, kind)
    check_attention(cache, model, table, lens, [1] * 11 + [0], hq, dtype, rng)


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype,out_dtype", [(BF16, None), (F32, None), (BF16, F32), (F32, BF16)])
@pytest.mark.parametrize("hq,hkv,d,pt", SHAPES[:8])
def test_ragged_rows(hq, hkv, d, pt, dtype, out_dtype, kind):
    """Chunks of a prompt, drafts and single tokens in one call; rows that come before the first token see nothing."""
    rng = np.random.default_rng(hq * 3 + d + pt)
    lens, rows = [200, 70, 3, 40, 129, 1, 0], [37, 1, 5, 40, 0, 1, 2]
    cache, model, table = filled(rng, lens, hkv, d, pt, kind)
    got = check_attention(cache, model, table, lens, rows, hq, dtype, rng, out_dtype, scale=0.11)
    assert np.isnan(got[38:40]).all() and not np.isnan(got[40:83]).any()   # sequence 2: two rows before its 3 tokens


@pytest.mark.parametrize("splits", [1, 2, 3, 7, 64, 1000])
@pytest.mark.parametrize("hq,hkv,d,pt,rows", [(8, 2, 128, 16, 1), (4, 1, 64, 64, 9), (4, 2, 80, 16, 2)])
def test_splits(hq, hkv, d, pt, rows, splits):
    """Any number of splits, over lengths from less than one to many times a split's tokens."""
    rng = np.random.default_rng(splits)
    lens = [900, 64, 9, 333]
    cache, model, table = filled(rng, lens, hkv, d, pt, "int8")
    check_attention(cache, model, table, lens, [rows] * 4, hq, BF16, rng, kv_splits=splits, max_rows=rows, max_context=900)


def random_cache(rng, lens, heads, d, pt, kind, spare=5):
    """As `filled`, with codes and scales drawn as they are."""
    batch, capacity = len(lens), max(lens) + pt
    need = [-(-n // pt) for n in lens]
    cache = make(batch, heads, d, pt, capacity, kind, sum(need) + spare)
    model = plain.Cache(cache.num_pages, heads, pt, d, kind)
    model.codes[:] = rng.integers(0, 256, model.codes.shape)
    model.codes[model.codes & 0x7F == 0x7F] = 3                       # (e4m3's NaN)
    model.scales[:] = np.exp(rng.standard_normal(model.scales.shape)) * (0.02 if kind == "int8" else 0.01)
    ids = rng.permutation(cache.num_pages)
    table = np.full((batch, cache.config.pages_per_seq), -1)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at: at + n]
        at += n
    model.upload(cache)
    cache.page_table.copy_(dev(table, torch.int32))
    cache.seq_lens.copy_(dev(lens, torch.int32))
    return cache, model, table


LONG = [  # q heads, kv heads, head dim, page tokens, lengths, rows
    (4, 2, 128, 16, [2500, 1, 700], [1, 1, 1]),
    (4, 2, 64, 32, [3000] + [90] * 69 + [1100], [1] * 35 + [0] + [1] * 35),
    (6, 2, 128, 16, [1500, 2000, 64], [40, 3, 1]),
    (20, 2, 64, 16, [1300, 1100], [2, 2]),
    # more than 16 tiles for each of the 512 / 64 workgroups of a head: dealt across sequences
    (64, 64, 64, 16, [4000, 3, 64, 0, 2111, 900, 1537], [1, 1, 1, 0, 1, 1, 1]),
    (64, 64, 64, 64, [130] * 66 + [1000, 129], [1] * 3 + [0] * 2 + [1] * 63),
    (64, 64, 128, 16, [2900, 5000, 1200], [4, 40, 1]),
    (128, 64, 64, 16, [3000, 2000, 4100], [1, 17, 9])]


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,pt,lens,rows", LONG)
def test_long_sequences(hq, hkv, d, pt, lens, rows, dtype, kind):
    """Sequences in pieces, and workgroups that cross from one to the next; the bounds a captured call would have."""
    rng = np.random.default_rng(len(lens) + d)
    cache, model, table = random_cache(rng, lens, hkv, d, pt, kind)
    got = check_attention(cache, model, table, lens, rows, hq, dtype, rng, max_rows=max(rows))
    rng = np.random.default_rng(len(lens) + d + 1)
    again = check_attention(cache, model, table, lens, rows, hq, dtype, rng)
    assert got.shape == again.shape


# more than 16 tiles for each of a head's workgroups, of sequences whose rows fill several blocks of 64 or 128 columns
PROMPTS = [
    (64, 64, 64, 16, [1100], [1100]),                               # a whole prompt: blocks see 1, 3, 5 ... tiles
    (64, 64, 128, 16, [1100, 3, 640, 1000, 0], [500, 1, 130, 300, 2]),
    (128, 64, 64, 32, [900, 77, 1300], [300, 0, 400]),
    (192, 64, 64, 16, [700, 1500], [300, 100]),                     # no whole number of rows a block
    (256, 32, 64, 48, [1000, 50, 900], [257, 180, 100])]            # 130 rows before the first token


@pytest.mark.parametrize("dtype,kind", [(BF16, "fp8"), (F32, "int8")])
@pytest.mark.parametrize("hq,hkv,d,pt,lens,rows", PROMPTS)
def test_prompts_in_shares(hq, hkv, d, pt, lens, rows, dtype, kind):
    """Workgroups whose shares begin and end inside blocks that see different numbers of tokens."""
    rng = np.random.default_rng(sum(lens) + hq)
    cache, model, table = random_cache(rng, lens, hkv, d, pt, kind)
    check_attention(cache, model, table, lens, rows, hq, dtype, rng, max_rows=max(rows))


def test_the_same_call_gives_the_same_bits():
    rng = np.random.default_rng(3)
    lens = [4000, 100, 900, 2000]
    cache, model, table = random_cache(rng, lens, 4, 128, 16, "int8")
    q = dev(rounded(rng, (40, 16, 128), BF16), BF16)
    starts = dev([0, 1, 2, 30, 40], torch.int32)
    want = qk.quantized_attention(cache, q, starts)
    for _ in range(5):
        assert torch.equal(qk.quantized_attention(cache, q, starts), want)


def test_rows_past_max_rows_stay():
    rng = np.random.default_rng(5)
    cache, model, table = filled(rng, [100, 50], 2, 128, 16, "int8")
    check_attention(cache, model, table, [100, 50], [7, 2], 4, BF16, rng, max_rows=4)


@pytest.mark.parametrize("hq,hkv,d,pt", [(8, 2, 128, 16), (4, 2, 64, 32), (4, 2, 40, 16)])
def test_starts_in_disorder_are_not_followed(hq, hkv, d, pt):
    """Overlapping, falling and far starts: rows in range are computed for some sequence, others are not touched."""
    rng = np.random.default_rng(4)
    lens = [100, 50, 70, 20]
    cache, model, table = filled(rng, lens, hkv, d, pt, "int8")
    q = rounded(rng, (6, hq, d), BF16)
    out = torch.full((6, hq, d), 9.0, dtype=BF16, device="cuda")
    for splits in (0, 3):
        qk.quantized_attention(cache, dev(q, BF16), dev([0, 2, 1, 2 ** 31 - 1, -7], torch.int32), out=out, kv_splits=splits)
        torch.cuda.synchronize()
        k, v = model.tokens(table[0], 100)
        want, off = plain.attend64(q[:2].astype(np.float64), k, v, 100, d ** -0.5, False)
        plain.close(out[:1].double().cpu().numpy(), want[:1], off[:1], 2.0 ** -8)   # row 1 is two sequences'


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 2, 64), (4, 2, 48)])
def test_rows_and_pools_off_their_borders(hq, hkv, d, dtype):
    """Queries, outputs, keys, values and pools that begin anywhere; common lengths without a list of them: the C calls
    that take what the Python layer does not make."""
    import ctypes

    from schedforge_amd import _abi
    rng = np.random.default_rng(d)
    lens, pt, lib = [70, 70], 16, _abi.load()
    cache, model, table = filled(rng, lens, hkv, d, pt, "int8")
    dt = _abi.F32 if dtype == F32 else _abi.BF16
    odd = lambda n, kind: torch.full((n + 7,), 3, dtype=kind, device="cuda")[3:]  # noqa: E731
    keys, values, q = (rounded(rng, (2, h, d), dtype) for h in (hkv, hkv, hq))
    slots = np.array([table[b, 69 // pt] * pt + 69 % pt for b in range(2)], np.int64)
    model.append(keys, values, slots)
    kp, vp = odd(cache.k_pool.numel(), torch.uint8), odd(cache.k_pool.numel(), torch.uint8)
    kp[: cache.k_pool.numel()] = cache.k_pool.view(torch.uint8).flatten()
    vp[: cache.k_pool.numel()] = cache.v_pool.view(torch.uint8).flatten()
    stride = hq * d + 1
    rows = {n: odd(2 * stride, dtype) for n in ("k", "v", "q", "out")}
    for n, x in (("k", keys), ("v", values), ("q", q)):
        for t in range(2):
            rows[n][t * stride: t * stride + x[t].size] = dev(x[t].ravel(), dtype)
    begun = cache.scales.clone()
    for kpool, vpool in ((cache.k_pool, cache.v_pool), (kp, vp)):
        cache.scales.copy_(begun)                                     # the scales that these codes were stored under
        a = _abi.Kv8AppendArgs()
        a.keys, a.values, a.dtype, a.key_stride, a.value_stride = rows["k"].data_ptr(), rows["v"].data_ptr(), dt, stride, stride
        a.k_pool, a.v_pool, a.pool_dtype, a.scales = kpool.data_ptr(), vpool.data_ptr(), _abi.I8, cache.scales.data_ptr()
        at = dev(slots, torch.int64)
        a.slots, a.tokens, a.kv_heads, a.head_dim, a.page_tokens, a.num_pages = at.data_ptr(), 2, hkv, d, pt, cache.num_pages
        _abi.check(lib.sfg_hip_kv8_append_v1(ctypes.byref(a), None))
        a = _abi.Kv8AttnArgs()
        a.q, a.q_dtype, a.q_stride, a.out, a.out_dtype, a.out_stride = rows["q"].data_ptr(), dt, stride, rows["out"].data_ptr(), dt, stride
        a.k_pool, a.v_pool, a.pool_dtype, a.scales = kpool.data_ptr(), vpool.data_ptr(), _abi.I8, cache.scales.data_ptr()
        a.page_table, a.batch, a.tokens, a.max_rows, a.q_heads, a.kv_heads, a.head_dim = cache.page_table.data_ptr(), 2, 2, 1, hq, hkv, d
        a.page_tokens, a.pages_per_seq, a.num_pages, a.max_context = pt, cache.config.pages_per_seq, cache.num_pages, 70
        ws = torch.empty(max(1, lib.sfg_hip_attn_kv8_workspace_v1(ctypes.byref(a))), dtype=torch.uint8, device="cuda")
        _abi.check(lib.sfg_hip_attn_kv8_v1(ctypes.byref(a), ws.data_ptr(), ws.numel(), None))
        for b in range(2):
            k, v = model.tokens(table[b], 70)
            want, off = plain.attend64(q[b: b + 1].astype(np.float64), k, v, 70, d ** -0.5, dtype == F32)
            got = rows["out"][b * stride: b * stride + hq * d].view(1, hq, d).double().cpu().numpy()
            plain.close(got, want, off, plain.HALF[dtype])
        assert float(rows["out"][hq * d]) == 3.0 and float(rows["out"][stride + hq * d]) == 3.0
    codes, scales = plain.download(cache)
    np.testing.assert_array_equal(codes, model.codes)
    np.testing.assert_array_equal(scales, model.scales)
    n = cache.k_pool.numel()
    assert torch.equal(kp[:n], cache.k_pool.view(torch.uint8).flatten()) and torch.equal(vp[:n], cache.v_pool.view(torch.uint8).flatten())
    assert (kp[n:] == 3).all() and (vp[n:] == 3).all()


def test_no_context_at_all():
    cache = make(2, 2, 64, 16, 32, "int8")
    for d in (64, 40):
        cache = make(2, 2, d, 16, 32, "int8")
        assert torch.isnan(qk.quantized_attention(cache, torch.ones(4, 2, d, dtype=BF16, device="cuda"), max_context=0)).all()


def test_lengths_are_cut_to_max_context():
    rng = np.random.default_rng(6)
    cache, model, table = filled(rng, [100, 50], 2, 64, 16, "fp8")
    cache.seq_lens.copy_(dev([5000, -3], torch.int32))
    check_attention(cache, model, table, [90, 0], [1, 1], 4, BF16, rng, max_context=90)


@pytest.mark.parametrize("hq,hkv,d,pt", [(8, 2, 128, 16), (4, 2, 64, 32), (4, 2, 40, 16)])
def test_uniform_rows_without_starts(hq, hkv, d, pt):
    rng = np.random.default_rng(7)
    lens = [60, 333]
    cache, model, table = filled(rng, lens, hkv, d, pt, "int8")
    q = dev(rounded(rng, (6, hq, d), BF16), BF16)
    starts = dev([0, 3, 6], torch.int32)
    assert torch.equal(qk.quantized_attention(cache, q), qk.quantized_attention(cache, q, starts, max_rows=3))


@pytest.mark.parametrize("hq,hkv,d,pt", [(8, 2, 128, 16), (4, 2, 64, 32), (4, 2, 40, 16)])
def test_pages_outside_the_pool_are_not_seen(hq, hkv, d, pt):
    """A page id outside the pool hides its tokens: as if the sequence held the other pages alone."""
    rng = np.random.default_rng(8)
    n = 9 * pt + 5
    cache, model, table = filled(rng, [n, n], hkv, d, pt, "int8")
    broken = table.copy()
    broken[0, [1, 4, 5]] = -1, 10 ** 6, -2 ** 31
    broken[1, :10] = -1
    cache.page_table.copy_(dev(broken, torch.int32))
    q = rounded(rng, (2, hq, d), BF16)
    got = qk.quantized_attention(cache, dev(q, BF16)).double().cpu().numpy()
    k, v = model.tokens(table[0], n)
    live = np.isin(np.arange(n) // pt, [1, 4, 5], invert=True)
    want, off = plain.attend64(q[:1].astype(np.float64), k[:, live], v[:, live], int(live.sum()), d ** -0.5, False)
    plain.close(got[:1], want, off, 2.0 ** -8)
    assert np.isnan(got[1]).all()


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("hq,hkv,d,pt", [(8, 2, 128, 16), (4, 2, 64, 32), (4, 2, 40, 16)])
def test_poisoned_pages_reach_the_rows_that_see_them(hq, hkv, d, pt, kind):
    """A NaN scale makes NaN of the rows and heads that see its page, and of no others; NaN codes behind the cached
    tokens of a page are not seen."""
    rng = np.random.default_rng(9)
    n = 5 * pt
    cache, model, table = filled(rng, [n, n - 3], hkv, d, pt, kind)
    page = int(table[0, 4])
    cache.scales[page, 0, 1] = float("nan")                           # V's of kv head 0, the last page
    cache.scales[int(table[1, 2]), 1, 0] = float("nan")               # K's of kv head 1, a page that all see
    rows = pt + 3                                                     # the first 3 rows come before the last page
    q = dev(rounded(rng, (2 * rows, hq, d), BF16), BF16)
    nan = torch.isnan(qk.quantized_attention(cache, q).float()).cpu().numpy()
    group = hq // hkv
    want = np.zeros((2, rows, hq, d), bool)
    want[0, 3:, :group] = True
    want[1, :, group:] = True
    assert np.array_equal(nan.reshape(2, rows, hq, d), want)


def test_queries_that_are_not_finite_stay_in_their_rows():
    rng = np.random.default_rng(10)
    cache, model, table = filled(rng, [100, 50], 2, 128, 16, "int8")
    q = dev(rounded(rng, (2, 8, 128), BF16), BF16)
    want = qk.quantized_attention(cache, q)
    q[0, 3, 5], q[1, 6, 0] = float("nan"), float("inf")
    got = qk.quantized_attention(cache, q)
    bad = torch.zeros(2, 8, dtype=torch.bool, device="cuda")
    bad[0, 3] = bad[1, 6] = True
    assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
def test_scores_far_apart(kind):
    """Queries whose scores span thousands: the softmax is one token's, whichever split it lies in."""
    rng = np.random.default_rng(11)
    cache, model, table = filled(rng, [700, 700], 2, 128, 16, kind)
    check_attention(cache, model, table, [700, 700], [1, 4], 8, BF16, rng, std=60.0, kv_splits=5)
    check_attention(cache, model, table, [700, 700], [1, 4], 8, F32, rng, std=1e-6)


# ---------------------------------------------------------------- together
@pytest.mark.parametrize("kind,dtype,d,pt", [("int8", BF16, 128, 16), ("fp8", BF16, 64, 32), ("int8", F32, 64, 16), ("fp8", BF16, 80, 16)])
def test_a_captured_step_serves_requests(kind, dtype, d, pt):
    """The four calls of a step, captured once and replayed with other counts: requests of several lengths come, grow
    token by token, give drafts back, end and make room.  Plans, codes and scales are exact each time."""
    rng = np.random.default_rng(d)
    batch, hq, hkv, room, capacity, pages = 4, 8, 2, 40, 160, 3 * 160 // pt
    cache = make(batch, hkv, d, pt, capacity, kind, pages)
    model, store = plain.Pages(batch, cache.config.pages_per_seq, pages, pt), plain.Cache(pages, hkv, pt, d, kind)
    angles = qk.RotaryAngles(d // 2, 10000.0, "bands", factor=4.0, context=64.0, low=1.0, high=4.0)
    counts, keep = (torch.zeros(batch, dtype=torch.int32, device="cuda") for _ in range(2))
    qkv = torch.zeros(room, (hq + 2 * hkv) * d, dtype=dtype, device="cuda")
    q, k, v = (qkv[:, a * d: (a + n) * d].view(room, n, d) for a, n in ((0, hq), (hq, hkv), (hq + hkv, hkv)))
    ws = torch.empty(max(1, qk.attention_workspace(cache, room, hq, dtype)), dtype=torch.uint8, device="cuda")

    def step():
        plan = qk.plan_step(cache, counts, room, keep)
        qr, kr = qk.rotate(angles, plan.positions, q, k, "interleaved")
        qk.append_quantized_kv(cache, kr, v, plan.slots)
        return plan, qr, kr, qk.quantized_attention(cache, qr, plan.starts, workspace=ws)
    step()                                                            # (loads the kernels; no tokens)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan, qr, kr, out = step()
    script = [([30, 5, 0, 1], None), ([1, 1, 20, 1], None), ([1, 6, 1, 1], None), ([1, 2, 1, 1], (1, 8)), ([1, 1, 1, 39], (3, 0)),
              ([1, 1, 1, 30], (3, 0)), ([1] * 4, None), ([40, 0, 0, 0], (0, 0))]
    for asked, cut in script:
        lens = list(model.lens)
        kept = [lens[b] if cut is None or cut[0] != b else cut[1] for b in range(batch)]
        qkv.copy_(dev(rounded(rng, qkv.shape, dtype), dtype))
        counts.copy_(dev(asked, torch.int32))
        keep.copy_(dev(kept, torch.int32))
        graph.replay()
        starts, positions, slots = model.step(asked, room, kept)
        assert plan.starts.cpu().tolist() == starts and plan.positions.cpu().tolist() == positions
        assert plan.slots.cpu().tolist() == slots and cache.page_table.cpu().tolist() == model.table
        total = starts[-1]
        want, size = plain.rotate64(k[:total].double().cpu().numpy(), positions[:total], angles.inv_freq, angles.magnitude, True)
        plain.close(kr[:total].double().cpu().numpy(), want, size * 2.0 ** -20, plain.HALF[dtype])
        store.append(kr.float().cpu().numpy(), v.float().cpu().numpy(), slots)
        codes, scales = plain.download(cache)
        np.testing.assert_array_equal(scales, store.scales)
        np.testing.assert_array_equal(codes, store.codes)
        for b in range(batch):
            t0, t1, n = starts[b], starts[b + 1], model.lens[b]
            if t1 > t0:
                kk, vv = store.tokens(np.array(model.table[b]), n)
                want, off = plain.attend64(qr[t0:t1].double().cpu().numpy(), kk, vv, n, d ** -0.5, dtype == F32)
                plain.close(out[t0:t1].double().cpu().numpy(), want, off, plain.HALF[dtype])


@pytest.mark.parametrize("kind", ["int8", "fp8"])
@pytest.mark.parametrize("d", [128, 80])
def test_pages_beyond_32_bit_offsets(d, kind):
    """The same step in a pool of a few pages and, from the highest ids down, in one whose codes pass 2^31 bytes."""
    rng = np.random.default_rng(d)
    k, v = (dev(rounded(rng, (93, 8, d), BF16), BF16) for _ in range(2))
    q = dev(rounded(rng, (93, 16, d), BF16), BF16)
    found = []
    for pages in (8, (1 << 31) // (8 * 16 * d) + 9):
        cache = make(2, 8, d, 16, 100, kind, pages)
        step = qk.plan_step(cache, dev([90, 3], torch.int32), 93)
        assert int(cache.page_table.max()) == pages - 1
        qk.append_quantized_kv(cache, k, v, step.slots)
        found.append((qk.quantized_attention(cache, q, step.starts), cache.k_pool[pages - 7:].view(torch.int8),
                      cache.v_pool[pages - 7:].view(torch.int8), cache.scales[pages - 7:]))
        assert pages < 9 or cache.k_pool[: pages - 7].view(torch.int8).count_nonzero() == 0
    for small, large in zip(*found):
        assert torch.equal(small, large)
    assert not found[1][0].isnan().any()


def test_rows_beyond_32_bit_offsets():
    """Queries, keys and values as columns of rows so wide that the last ones lie past 2^31 elements."""
    rng = np.random.default_rng(8)
    rows, wide, d = 2100, 1 << 20, 128
    block = torch.zeros((rows, wide), dtype=BF16, device="cuda")
    near = dev(rounded(rng, (rows, 4 * d), BF16), BF16)
    block[:, wide - 4 * d:] = near
    far = block[:, wide - 4 * d:]
    found = []
    for x in (near, far):
        cache = make(1, 1, d, 16, rows, "int8")
        step = qk.plan_step(cache, dev([rows], torch.int32), rows)
        q, k, v = x[:, : 2 * d].view(rows, 2, d), x[:, 2 * d: 3 * d].view(rows, 1, d), x[:, 3 * d:].view(rows, 1, d)
        q_out, k_out = qk.rotate(qk.RotaryAngles(d), step.positions, q, k, q_out=q, k_out=k)
        qk.append_quantized_kv(cache, k_out, v, step.slots)
        found.append((qk.quantized_attention(cache, q_out, step.starts, out=q_out.clone()), cache.k_pool, cache.v_pool, cache.scales))
        found[-1] += (qk.quantized_attention(cache, q_out, step.starts, out=q_out.new_zeros((rows, 3, d))[:, :2]),)
    for a, b in zip(*found):
        assert torch.equal(a, b)
    assert torch.equal(found[0][0], found[0][4])


def test_on_a_stream_of_its_own():
    """The calls run on the stream they are given, behind what it holds, while another one is current."""
    rng = np.random.default_rng(12)
    cache = make(2, 2, 64, 16, 256, "int8")
    model = plain.Cache(cache.num_pages, 2, 16, 64, "int8")
    side = torch.cuda.Stream()
    x = rounded(rng, (200, 2, 64), BF16)
    with torch.cuda.stream(side):
        keys = torch.zeros(200, 2, 64, dtype=BF16, device="cuda")
        a = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):
            a = a @ a * 1e-3                                         # keeps the stream busy
        keys.copy_(dev(x, BF16))
    plan = qk.plan_step(cache, dev([120, 80], torch.int32), 200, stream=side)
    side.wait_stream(torch.cuda.current_stream())
    qk.append_quantized_kv(cache, keys, keys, plan.slots, stream=side)
    q = torch.ones(2, 4, 64, dtype=BF16, device="cuda")
    side.wait_stream(torch.cuda.current_stream())
    out = qk.quantized_attention(cache, q, stream=side)
    side.synchronize()
    model.append(x, x, plan.slots.cpu().numpy())
    codes, scales = plain.download(cache)
    np.testing.assert_array_equal(codes, model.codes)
    for b, n in enumerate((120, 80)):
        k, v = model.tokens(cache.page_table[b].cpu().numpy(), n)
        want, off = plain.attend64(np.ones((1, 4, 64)), k, v, n, 0.125, False)
        plain.close(out[b: b + 1].double().cpu().numpy(), want, off, 2.0 ** -8)


# ---------------------------------------------------------------- what Python refuses
def test_refusals():
    cache = make(2, 2, 64, 16, 256, "int8")
    q = torch.ones(2, 4, 64, dtype=BF16, device="cuda")
    slots, counts = torch.zeros(2, dtype=torch.int64, device="cuda"), torch.ones(2, dtype=torch.int32, device="cuda")
    k = torch.ones(2, 2, 64, dtype=BF16, device="cuda")
    a, pos = qk.RotaryAngles(64), torch.zeros(2, dtype=torch.int32, device="cuda")
    bad = [
        lambda: qk.QuantizedKVCache(qk.QuantizedKVConfig(2, 2, 64, 16, 256, pool_dtype="int4")),
        lambda: qk.QuantizedKVCache(qk.QuantizedKVConfig(2, 2, 64, 16, 0)),
        lambda: qk.plan_step(cache, counts.long(), 4), lambda: qk.plan_step(cache, counts[:1], 4),
        lambda: qk.plan_step(cache, counts, 0), lambda: qk.plan_step(cache, counts.cpu(), 4),
        lambda: qk.plan_step(cache, counts, 4, keep=[1, 2]), lambda: qk.plan_step(cache, counts, 4, stream=0),
        lambda: qk.plan_step(cache, counts, 4, out=qk.plan_step(cache, torch.zeros_like(counts), 5)),
        lambda: qk.RotaryAngles(63), lambda: qk.RotaryAngles(64, scaling="other"), lambda: qk.RotaryAngles(64, inv_freq=np.ones(31)),
        lambda: qk.RotaryAngles(64, scaling="linear", factor=0.5), lambda: qk.RotaryAngles(64, scaling="bands", factor=2.0),
        lambda: qk.rotate(a, pos), lambda: qk.rotate(a, pos, q.half()), lambda: qk.rotate(a, pos[:1], q),
        lambda: qk.rotate(a, pos, q, k.float()), lambda: qk.rotate(a, pos, q, layout="other"), lambda: qk.rotate(a, pos, q[:, :, :32]),
        lambda: qk.rotate(a, pos, q.transpose(0, 1)), lambda: qk.rotate(a, pos, q, k_out=k), lambda: qk.rotate(a, pos, q[:0]),
        lambda: qk.rotate(a, pos, q, q_out=q[:1]), lambda: qk.rotate(a, pos, q[:1].expand(2, 4, 64)),
        lambda: qk.append_quantized_kv(cache, k, k, slots.int()), lambda: qk.append_quantized_kv(cache, k, k.float(), slots),
        lambda: qk.append_quantized_kv(cache, k[:, :1], k[:, :1], slots), lambda: qk.append_quantized_kv(cache, k, k, slots[:1]),
        lambda: qk.append_quantized_kv(cache, k.cpu(), k, slots), lambda: qk.append_quantized_kv(cache, k.int(), k.int(), slots),
        lambda: qk.quantized_attention(cache, q[0]), lambda: qk.quantized_attention(cache, q[:, :3]),
        lambda: qk.quantized_attention(cache, q[:1]), lambda: qk.quantized_attention(cache, q, counts),
        lambda: qk.quantized_attention(cache, q, max_rows=2), lambda: qk.quantized_attention(cache, q, max_context=257),
        lambda: qk.quantized_attention(cache, q, out=q), lambda: qk.quantized_attention(cache, q[:, :, :32]),
        lambda: qk.quantized_attention(cache, q, out=torch.empty(2, 4, 64, device="cuda", dtype=torch.float16)),
        lambda: qk.quantized_attention(cache, q, workspace=torch.empty(4, device="cuda")), lambda: qk.quantized_attention(cache, "q")]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was taken")
