"""Continuous batching over the 8-bit paged K/V cache: wk_batch_plan,
wk_kv8_store, wk_kv8_attention and wk_attention_packed against plain
implementations in 64 bits, their refusals, and a serving loop of all four.

Tolerances.  Attention: with u the rounding of the output type, u_p that of the
softmax weights as the kernel multiplies them with V (their type has the
output's significand or a longer one), S the largest scale * sum |q||k| of a row
and A = sum p |v|, every output is within
    u |o| + A (u_p + 2 (D 2^-24 S + 2^-20) + len 2^-24) (1 + u) + tiny
of the exact one: the product sums of D and of len terms in fp32, an exponential
good to 2^-21 and the two roundings.  Plans and stored codes are exact.
"""
import ctypes
import math

import numpy as np
import pytest

import wukong_b200 as wk
from tests.gpu_util import alloc, bf16_bits, bf16_to_f32, down, free, up

PAGE = 64
E4M3_MAX = 448.0


# ------------------------------------------------------------------ e4m3 and scales in 64 bits

def _code_values():
    v = np.zeros(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        v[c] = -x if c & 128 else x
    v[0x7F] = v[0xFF] = np.nan
    return v


CODES = _code_values()
_POS = CODES[:0x7F]  # ascending


def e4m3_codes(x):
    """Codes of the nearest e4m3 values, ties to the even code, saturating; NaN is 0x7f."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(x), E4M3_MAX)
    hi = np.searchsorted(_POS, np.nan_to_num(a), side="left").clip(0, 0x7E)
    lo = (hi - 1).clip(0)
    dl, dh = a - _POS[lo], _POS[hi] - a
    c = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    c = np.where(_POS[hi] == a, hi, c)
    c = np.where(np.isnan(x), 0x7F, c | np.where(np.signbit(x), 0x80, 0))
    return c.astype(np.uint8)


def scale_for(amax):
    if amax == 0:
        return 2.0 ** -100
    f, e = math.frexp(amax)
    return 2.0 ** max(e - 9 + (f > 0.875), -100)


def same_codes(got, want):
    """Equal, any NaN code for another."""
    return (got == want) | (((got & 0x7F) == 0x7F) & ((want & 0x7F) == 0x7F))


# ------------------------------------------------------------------ types

def to_bits(x, dt):
    return np.asarray(x, np.float32).astype(np.float16) if dt == wk.F16 else bf16_bits(x)


def from_bits(b, dt):
    return b.astype(np.float64) if dt == wk.F16 else bf16_to_f32(b).astype(np.float64)


def rounded(x, dt):
    return from_bits(to_bits(x, dt), dt)


RAW = {wk.F16: np.float16, wk.BF16: np.uint16}
UNIT = {wk.F16: 2.0 ** -11, wk.BF16: 2.0 ** -8}


def as_p(a):
    return a.ctypes.data_as(ctypes.c_void_p)


def attend(q, k, v, visible, dt):
    """softmax(q k^T / sqrt(d)) v for one query over its visible keys, and how far off a kernel may be."""
    d = q.shape[-1]
    if visible <= 0:
        return np.zeros(d), np.zeros(d)
    k, v = k[:visible], v[:visible]
    s = k @ q / math.sqrt(d)
    p = np.exp(s - s.max())
    p /= p.sum()
    o, A = p @ v, p @ np.abs(v)
    S = (np.abs(k) @ np.abs(q)).max() / math.sqrt(d)
    u = UNIT[dt]
    tol = u * np.abs(o) + A * (u + 2 * (d * 2.0 ** -24 * S + 2.0 ** -20) + visible * 2.0 ** -24) * (1 + u)
    return o, tol + 2.0 ** -24 * (1 + np.abs(v).max())


# ------------------------------------------------------------------ refusals (no GPU)

FAKE = 4096


def _refused(call, words):
    L = wk.lib()
    assert call(L) == -1
    assert words in L.wk_last_error().decode()


@pytest.mark.parametrize("change,words", [
    (dict(n=0), "n 0"), (dict(n=8193), "n 8193"), (dict(rows_cap=-1), "bad sizes"), (dict(max_pages=0), "bad sizes"),
    (dict(free_cap=-1), "bad sizes"), (dict(n=8192, max_pages=1 << 20), "2^31"), (dict(starts=None), "null"),
    (dict(row_pos=None), "null"), (dict(n_free=None), "null"), (dict(free_pages=None), "null"),
    (dict(ctx=2 * FAKE + 2), "misaligned"), (dict(row_slot=FAKE + 4), "misaligned"), (dict(lens=2 * FAKE), "must not be"),
    (dict(starts=3 * FAKE), "must not be"),
])
def test_plan_refusals(change, words):
    a = dict(starts=FAKE, lens=FAKE, row_seq=FAKE, row_pos=FAKE, row_slot=None, rows_cap=8, table=FAKE, max_pages=4,
             status=FAKE, ctx=2 * FAKE, add=3 * FAKE, n=2, free_pages=FAKE, n_free=FAKE, free_cap=3)
    a.update(change)
    _refused(lambda L: L.wk_batch_plan(*a.values()), words)


@pytest.mark.parametrize("change,words", [
    (dict(n=-1), "bad sizes"), (dict(rows=-1), "bad sizes"), (dict(n_pages=0), "bad sizes"),
    (dict(kv_heads=0), "bad sizes"), (dict(hd=96), "head_dim 96"), (dict(dt=wk.F32), "dtype 0"),
    (dict(k=None), "null"), (dict(vscale=None), "null"), (dict(k_rs=127), "stride"), (dict(v_rs=0), "stride"),
    (dict(kpool=FAKE + 8), "aligned"), (dict(k=FAKE + 1), "misaligned"), (dict(vscale=FAKE + 2), "misaligned"),
])
def test_store_refusals(change, words):
    a = dict(kpool=FAKE, vpool=FAKE, kscale=FAKE, vscale=FAKE, n_pages=9, k=FAKE, k_rs=128, v=FAKE, v_rs=128,
             starts=FAKE, ctx=FAKE, n=1, rows=4, table=FAKE, max_pages=4, kv_heads=2, hd=64, dt=wk.F16)
    a.update(change)
    _refused(lambda L: L.wk_kv8_store(*a.values()), words)


@pytest.mark.parametrize("change,words", [
    (dict(rows=-1), "bad sizes"), (dict(n_seqs=0), "bad sizes"), (dict(max_len=-1), "bad sizes"),
    (dict(ws_bytes=-1), "bad sizes"), (dict(heads=3), "3 heads over 2"), (dict(heads=0), "heads"),
    (dict(hd=32), "head_dim 32"), (dict(dt=wk.Q8_0), "dtype 8"), (dict(q=None), "null"), (dict(pos=None), "null"),
    (dict(q_rs=255), "stride"), (dict(out_rs=1), "stride"), (dict(vpool=FAKE + 4), "aligned"),
    (dict(ws=FAKE + 4, ws_bytes=99), "workspace"), (dict(max_pages=1 << 26), "bad sizes"),
    (dict(q=FAKE + 1), "misaligned"), (dict(pos=FAKE + 2), "misaligned"),
])
def test_decode_refusals(change, words):
    a = dict(out=FAKE, out_rs=256, q=FAKE, q_rs=256, kpool=FAKE, vpool=FAKE, kscale=FAKE, vscale=FAKE, n_pages=4,
             table=FAKE, n_seqs=1, max_pages=4, seq=FAKE, pos=FAKE, rows=1, max_len=9, heads=4, kv_heads=2, hd=64,
             dt=wk.F16, ws=None, ws_bytes=0)
    a.update(change)
    _refused(lambda L: L.wk_kv8_attention(*a.values()), words)


@pytest.mark.parametrize("change,words", [
    (dict(n=-1), "bad sizes"), (dict(q_rows=-1), "bad sizes"), (dict(k_rows=-1), "bad sizes"),
    (dict(heads=5), "5 heads over 2"), (dict(kv_heads=0), "heads"), (dict(hd=80), "head_dim 80"),
    (dict(dt=wk.F32), "dtype 0"), (dict(out=None), "null"), (dict(k=None), "null"), (dict(k_starts=None), "null"),
    (dict(v_rs=127), "stride"), (dict(out_rs=255), "stride"), (dict(out=FAKE + 1), "misaligned"),
    (dict(q_starts=FAKE + 2), "misaligned"),
])
def test_packed_refusals(change, words):
    a = dict(out=FAKE, out_rs=256, q=FAKE, q_rs=256, k=FAKE, k_rs=128, v=FAKE, v_rs=128, q_starts=FAKE, k_starts=FAKE,
             n=1, q_rows=4, k_rows=4, heads=4, kv_heads=2, hd=64, dt=wk.F16)
    a.update(change)
    _refused(lambda L: L.wk_attention_packed(*a.values()), words)


def test_empty_calls_launch_nothing():
    L = wk.lib()
    assert L.wk_kv8_store(FAKE, FAKE, FAKE, FAKE, 1, None, 64, None, 64, None, None, 0, 0, None, 1, 1, 64, wk.F16) == 0
    assert L.wk_kv8_attention(None, 64, None, 64, FAKE, FAKE, FAKE, FAKE, 1, None, 1, 1, None, None, 0, 0, 1, 1, 64,
                              wk.F16, None, 0) == 0
    assert L.wk_attention_packed(None, 64, None, 64, None, 64, None, 64, None, None, 3, 0, 0, 1, 1, 64, wk.F16) == 0


def test_e4m3_rounding_of_the_tests_themselves():
    assert e4m3_codes([0.0, 1.0, 448.0, 1e9, -448.0, 2.0 ** -9, 2.0 ** -10, 1.0625, 1.1875]).tolist() == \
        [0, 0x38, 0x7E, 0x7E, 0xFE, 1, 0, 0x38, 0x3A]
    assert scale_for(448.0) == 1.0 and scale_for(448.5) == 2.0 and scale_for(224.0) == 0.5


# ------------------------------------------------------------------ plan

def ref_plan(ctx, add, table, free_pages, n_free, rows_cap):
    n, max_pages = table.shape
    table = table.copy()
    starts = np.concatenate([[0], np.cumsum(np.maximum(add, 0))])
    seq, pos, slot = (np.full(rows_cap, -1, np.int64) for _ in range(3))
    used = want = 0
    for i in range(n):
        c, a = max(int(ctx[i]), 0), max(int(add[i]), 0)
        have, need = min(-(-c // PAGE), max_pages), min(-(-(c + a) // PAGE), max_pages)
        for p in range(have, need):
            table[i, p] = free_pages[used] if used < n_free else -1
            used, want = used + (used < n_free), want + 1
        for j in range(a):
            r, p = starts[i] + j, c + j
            if r < rows_cap:
                seq[r], pos[r] = i, p
                if p // PAGE < max_pages and table[i, p // PAGE] >= 0:
                    slot[r] = int(table[i, p // PAGE]) * PAGE + p % PAGE
    return dict(starts=starts, lens=np.maximum(ctx, 0) + np.maximum(add, 0), row_seq=seq, row_pos=pos, row_slot=slot,
                table=table, status=np.array([starts[-1], used, want - used]))


def run_plan(dev, ctx, add, table, free_pages, n_free, rows_cap, slots=True):
    n, max_pages = table.shape
    bufs = dict(starts=alloc(4 * (n + 1)), lens=alloc(4 * n), row_seq=alloc(4 * rows_cap), row_pos=alloc(4 * rows_cap),
                row_slot=up(np.full(rows_cap, 77, np.int64)), table=up(table.astype(np.int32)), status=alloc(12),
                ctx=up(ctx.astype(np.int32)), add=up(add.astype(np.int32)), free=up(free_pages.astype(np.int32)),
                n_free=up(np.array([n_free], np.int32)))
    wk.check(dev.wk_batch_plan(bufs["starts"], bufs["lens"], bufs["row_seq"], bufs["row_pos"],
                               bufs["row_slot"] if slots else None, rows_cap, bufs["table"], max_pages,
                               bufs["status"], bufs["ctx"], bufs["add"], n, bufs["free"], bufs["n_free"],
                               len(free_pages)))
    got = dict(starts=down(bufs["starts"], n + 1, np.int32), lens=down(bufs["lens"], n, np.int32),
               row_seq=down(bufs["row_seq"], rows_cap, np.int32), row_pos=down(bufs["row_pos"], rows_cap, np.int32),
               row_slot=down(bufs["row_slot"], rows_cap, np.int64), table=down(bufs["table"], table.shape, np.int32),
               status=down(bufs["status"], 3, np.int32))
    free(*bufs.values())
    return got


PLANS = [
    # n, context lengths up to, tokens up to, max_pages, free pages beyond those needed (negative: too few), rows beyond
    (1, 0, 1, 1, 0, 0),
    (1, 200, 1, 4, 3, 5),
    (3, 64, 0, 2, 0, 4),          # nobody brings anything
    (64, 1000, 1, 17, 0, 0),
    (257, 700, 130, 14, 9, 100),
    (40, 300, 90, 8, -11, 3),     # the free list runs out
    (40, 300, 900, 8, 5, 0),      # sequences outgrow their table
    (40, 300, 90, 8, 5, -200),    # more rows than the caller has room for
    (1000, 5000, 3, 80, 1, 1),
    (8192, 100, 2, 3, 0, 64),
]


@pytest.mark.gpu
@pytest.mark.parametrize("n,ctx_max,add_max,max_pages,spare,beyond", PLANS)
def test_plan_matches_the_plain_one(dev, n, ctx_max, add_max, max_pages, spare, beyond):
    rng = np.random.default_rng(n + ctx_max)
    ctx, add = rng.integers(0, ctx_max + 1, n), rng.integers(0, add_max + 1, n)
    if n > 2:
        ctx[1], add[1], add[2] = -5, max(add_max, 1), -3  # negative lengths count as 0
        add[0] = 0
    have = -(-np.maximum(ctx, 0) // PAGE)
    want = (np.minimum(-(-(np.maximum(ctx, 0) + np.maximum(add, 0)) // PAGE), max_pages) - np.minimum(have, max_pages)).sum()
    n_free = max(int(want) + spare, 0)
    ids = rng.permutation(int(have.sum()) + n_free + 2)
    table = rng.integers(-3, 1000, (n, max_pages))
    rows_cap = max(int(np.maximum(add, 0).sum()) + beyond, 0)
    w = ref_plan(ctx, add, table, ids, n_free, rows_cap)
    for slots in (True, False):
        g = run_plan(dev, ctx, add, table, ids, n_free, rows_cap, slots)
        for k in w:
            if k != "row_slot" or slots:
                assert np.array_equal(g[k], w[k]), k
        if not slots:
            assert (g["row_slot"] == 77).all()
    n_over = len(ids) + 40  # a count above the list's capacity is cut to it
    w = ref_plan(ctx, add, table, ids, len(ids), rows_cap)
    g = run_plan(dev, ctx, add, table, ids, n_over, rows_cap)
    assert all(np.array_equal(g[k], w[k]) for k in w)


# ------------------------------------------------------------------ store

def ref_store(codes, scales, x, starts, ctx, table, n_pages):
    """One of K or V: x [rows, kv, hd] in 64 bits."""
    codes, scales = codes.copy(), scales.astype(np.float64)
    for i in range(len(ctx)):
        row, pos, end = starts[i], ctx[i], ctx[i] + starts[i + 1] - starts[i]
        while pos < end:
            m = min(PAGE - pos % PAGE, end - pos)
            pi, off = pos // PAGE, pos % PAGE
            page = table[i, pi] if pi < table.shape[1] else -1
            if 0 <= page < n_pages:
                for h in range(codes.shape[1]):
                    b = x[row:row + m, h]
                    a = np.abs(b)
                    s = scale_for(a[np.isfinite(a)].max(initial=0.0))
                    if off:
                        s = max(s, scales[page, h])
                        if s != scales[page, h]:
                            codes[page, h, :off] = e4m3_codes(CODES[codes[page, h, :off]] * (scales[page, h] / s))
                    codes[page, h, off:off + m] = e4m3_codes(b / s)
                    scales[page, h] = s
            row, pos = row + m, pos + m
    return codes, scales


STORES = [
    # context and added tokens per sequence, kv_heads, head_dim, dtype, row stride beyond the row, offset of the first row
    ([0], [1], 1, 64, wk.F16, 0, 0),
    ([63], [2], 2, 128, wk.BF16, 0, 0),
    ([64, 5, 0, 127], [1, 1, 1, 1], 8, 128, wk.F16, 4096, 0),
    ([0, 17, 300], [200, 64, 129], 3, 64, wk.BF16, 64, 0),
    ([1, 62, 0, 9, 9], [63, 3, 0, 0, 65], 2, 128, wk.F16, 3, 1),  # rows that are not 16-byte aligned
    ([0, 0, 0], [0, 0, 0], 2, 64, wk.F16, 0, 0),
    (list(range(300)), [1 + i % 3 for i in range(300)], 1, 64, wk.BF16, 0, 0),
]


def make_store(ctx, add, kv, hd, dt, extra, shift, seed, loud=4.0):
    rng = np.random.default_rng(seed)
    ctx, add = np.array(ctx), np.array(add)
    starts = np.concatenate([[0], np.cumsum(add)])
    rows = int(starts[-1])
    pages_of = -(-(ctx + add) // PAGE)
    n_pages = int(pages_of.sum()) + 3
    max_pages = int(pages_of.max()) + 1
    perm = rng.permutation(n_pages)
    table = np.full((len(ctx), max_pages), -1)
    at = 0
    for i, p in enumerate(pages_of):
        table[i, :p] = perm[at:at + p]
        at += p
    shape = (n_pages, kv, PAGE, hd)
    old = [e4m3_codes(rng.standard_normal(shape) * 60) for _ in range(2)]
    olds = [2.0 ** rng.integers(-9, -5, shape[:2]) for _ in range(2)]
    rs = kv * hd + extra
    raw, x = [], []
    for _ in range(2):
        full = rng.standard_normal((rows + 2, rs)) * loud ** rng.integers(-1, 2, (rows + 2, 1))
        bits = to_bits(full, dt).reshape(-1)
        raw.append(bits)
        x.append(from_bits(bits[shift:shift + rows * rs].reshape(rows, rs)[:, :kv * hd], dt).reshape(rows, kv, hd))
    return dict(ctx=ctx, starts=starts, rows=rows, table=table, n_pages=n_pages, old=old, olds=olds, raw=raw, x=x, rs=rs,
                shift=shift, kv=kv, hd=hd, dt=dt)


def run_store(dev, c, rows=None):
    b = [up(v) for v in (*c["old"], *(s.astype(np.float32) for s in c["olds"]), *c["raw"], c["starts"].astype(np.int32),
                         c["ctx"].astype(np.int32), c["table"].astype(np.int32))]
    o = 2 * c["shift"]
    wk.check(dev.wk_kv8_store(b[0], b[1], b[2], b[3], c["n_pages"], b[4] + o, c["rs"], b[5] + o, c["rs"], b[6], b[7],
                              len(c["ctx"]), c["rows"] if rows is None else rows, b[8], c["table"].shape[1], c["kv"],
                              c["hd"], c["dt"]))
    got = [down(b[0], c["old"][0].shape, np.uint8), down(b[1], c["old"][0].shape, np.uint8),
           down(b[2], c["olds"][0].shape, np.float32), down(b[3], c["olds"][0].shape, np.float32)]
    free(*b)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("ctx,add,kv,hd,dt,extra,shift", STORES)
def test_store_is_exact(dev, ctx, add, kv, hd, dt, extra, shift):
    c = make_store(ctx, add, kv, hd, dt, extra, shift, seed=len(ctx) * 100 + hd)
    got = run_store(dev, c)
    for i in range(2):
        codes, scales = ref_store(c["old"][i], c["olds"][i], c["x"][i], c["starts"], c["ctx"], c["table"], c["n_pages"])
        assert np.array_equal(got[2 + i].astype(np.float64), scales)
        assert same_codes(got[i], codes).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n,some", [(256, 256), (257, 200), (1000, 900), (70000, 150)])
@pytest.mark.parametrize("late", [0, 90])
def test_store_finds_each_sequence(dev, n, some, late):
    """Many sequences, some without rows, of one token or of several pages; rows of nobody before the first."""
    rng = np.random.default_rng(n + late)
    add, ctx = np.zeros(n + 1, int), np.zeros(n + 1, int)
    on = 1 + np.sort(rng.permutation(n)[:some])
    add[on] = rng.choice([1, 1, 1, 2, 64, 65, 66, 130], some)
    ctx[on] = rng.integers(0, 70, some)
    add[0] = late
    c = make_store(ctx, add, 1, 64, wk.F16, 0, 0, seed=n)
    c = dict(c, starts=c["starts"][1:], ctx=c["ctx"][1:], table=c["table"][1:])
    got = run_store(dev, c)
    for i in range(2):
        codes, scales = ref_store(c["old"][i], c["olds"][i], c["x"][i], c["starts"], c["ctx"], c["table"], c["n_pages"])
        assert np.array_equal(got[2 + i].astype(np.float64), scales)
        assert same_codes(got[i], codes).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [wk.F16, wk.BF16])
def test_store_extremes(dev, dt):
    """Zeros, infinities, NaN, the type's largest and smallest values; a page without an id; a table that ends."""
    c = make_store([3, 0, 10, 64, 0], [4, 64, 30, 6, 70], 2, 64, dt, 0, 0, seed=5)
    top = 65504.0 if dt == wk.F16 else float(np.float64(2.0 ** 127 * (2 - 2.0 ** -7)))
    tiny = 2.0 ** -24 if dt == wk.F16 else 2.0 ** -133
    for i in range(2):
        x = c["x"][i]
        x[0:2, 0] = 0.0
        x[2, 0, :4] = [np.inf, -np.inf, np.nan, 1.0]
        x[4:68, 1] = 0.0                       # a fresh page of zeros
        x[68, :] = top
        x[70:98, 1, 5] = tiny
        x[98:104] = tiny
        c["raw"][i] = to_bits(np.concatenate([x.reshape(c["rows"], -1), np.zeros((2, c["rs"]))]), dt).reshape(-1)
        c["x"][i] = from_bits(c["raw"][i][: c["rows"] * c["rs"]].reshape(c["rows"], c["rs"]), dt).reshape(x.shape)
    c["table"][2, 0] = c["n_pages"]            # no such page: dropped
    c["table"] = c["table"][:, :2].copy()
    c["table"][4, 1] = -1
    with np.errstate(invalid="ignore", over="ignore"):
        want = [ref_store(c["old"][i], c["olds"][i], c["x"][i], c["starts"], c["ctx"], c["table"], c["n_pages"])
                for i in range(2)]
    got = run_store(dev, c)
    for i in range(2):
        assert np.array_equal(got[2 + i].astype(np.float64), want[i][1])
        assert same_codes(got[i], want[i][0]).all()


@pytest.mark.gpu
def test_store_twice_changes_nothing_more_and_rows_bound_the_call(dev):
    c = make_store([30, 0], [20, 100], 2, 128, wk.F16, 0, 0, seed=9)
    first = run_store(dev, c)
    again = run_store(dev, dict(c, old=first[:2], olds=first[2:]))
    assert all(np.array_equal(a, b) for a, b in zip(first, again))
    cut = run_store(dev, c, rows=50)
    starts = np.minimum(c["starts"], 50)
    for i in range(2):
        codes, scales = ref_store(c["old"][i], c["olds"][i], c["x"][i], starts, c["ctx"], c["table"], c["n_pages"])
        assert np.array_equal(cut[i], codes) and np.array_equal(cut[2 + i], scales)


# ------------------------------------------------------------------ decode attention

DECODES = [
    # position per row, heads, kv_heads, head_dim, dtype, max_len beyond the longest, workspace
    ([0], 1, 1, 64, wk.F16, 0, False),
    ([62, 63, 64], 4, 4, 128, wk.BF16, 0, False),
    ([776], 16, 4, 64, wk.F16, 3, True),
    ([1, 700, 65, -1, 300], 32, 8, 128, wk.F16, 0, True),
    ([2047], 8, 1, 128, wk.BF16, 0, True),
    ([1500, 127, 128], 24, 2, 64, wk.F16, 100, False),       # 12 heads per K/V head
    ([900, 3], 32, 1, 128, wk.F16, 0, True),                 # 32 heads over one
    ([555] * 5, 15, 3, 64, wk.BF16, 5000, True),             # 5 per K/V head, max_len far above
    (list(range(0, 640, 7)), 8, 8, 64, wk.F16, 0, True),     # 92 rows
    ([20000], 2, 1, 64, wk.F16, 0, True),
    ([4000, 9], 7, 1, 128, wk.BF16, -3000, True),            # max_len below the longest: still right
]


def make_decode(pos, heads, kv, hd, dt, seed, shared=False):
    rng = np.random.default_rng(seed)
    pos = np.array(pos)
    rows = len(pos)
    seq = np.zeros(rows, int) if shared else np.arange(rows)
    lens = np.array([pos.max() + 1]) if shared else pos + 1
    pages_of = -(-np.maximum(lens, 0) // PAGE)
    n_pages, max_pages = int(pages_of.sum()) + 2, max(int(pages_of.max()), 1)
    perm = rng.permutation(n_pages)
    table = np.full((len(lens), max_pages), 1 << 30)
    at = 0
    for i, p in enumerate(pages_of):
        table[i, :p] = perm[at:at + p]
        at += p
    codes = [e4m3_codes(rng.standard_normal((n_pages, kv, PAGE, hd)) * 80) for _ in range(2)]
    scales = [2.0 ** rng.integers(-8, -5, (n_pages, kv)).astype(float) for _ in range(2)]
    for i, n in enumerate(lens):  # NaN behind the end of each sequence, and in the pages of none
        if n > 0 and n % PAGE:
            for c in codes:
                c[table[i, n // PAGE], :, n % PAGE:] = 0x7F
    for c, s in zip(codes, scales):
        c[perm[at:]] = 0x7F
        s[perm[at:]] = np.nan
    q = rounded(rng.standard_normal((rows, heads * hd)) * 1.5, dt)
    return dict(pos=pos, seq=seq, table=table, codes=codes, scales=scales, q=q, heads=heads, kv=kv, hd=hd, dt=dt,
                n_pages=n_pages)


def ref_decode(c):
    rows, g, hd = len(c["pos"]), c["heads"] // c["kv"], c["hd"]
    out, tol = np.zeros((rows, c["heads"], hd)), np.zeros((rows, c["heads"], hd))
    for r in range(rows):
        n = int(c["pos"][r]) + 1
        if n <= 0 or not 0 <= c["seq"][r] < len(c["table"]):
            continue
        pages = c["table"][c["seq"][r], : -(-n // PAGE)]
        there = np.repeat((pages >= 0) & (pages < c["n_pages"]), PAGE)[:n]
        pages = np.where((pages >= 0) & (pages < c["n_pages"]), pages, 0)
        for a in range(c["kv"]):
            k, v = ((CODES[c["codes"][x][pages, a]] * c["scales"][x][pages, a][:, None, None]).reshape(-1, hd)[:n][there]
                    for x in range(2))
            for h in range(a * g, (a + 1) * g):
                out[r, h], tol[r, h] = attend(c["q"][r].reshape(-1, hd)[h], k, v, len(k), c["dt"])
    return out.reshape(rows, -1), tol.reshape(rows, -1)


def run_decode(dev, c, max_len, ws=False, extra=0, shift=0, short_ws=None):
    rows, w = c["q"].shape
    rs = w + extra
    q = np.full((rows, rs), np.nan)
    q[:, :w] = c["q"]
    bits = np.concatenate([np.zeros(shift, RAW[c["dt"]]), to_bits(q, c["dt"]).reshape(-1)])
    sent = np.full(rows * rs + shift + 8, 0x3555, np.uint16)
    b = [up(v) for v in (sent, bits, *c["codes"], *(s.astype(np.float32) for s in c["scales"]),
                         c["table"].astype(np.int32), c["seq"].astype(np.int32), c["pos"].astype(np.int32))]
    nws = dev.wk_kv8_attention_ws(rows, max_len, c["heads"], c["kv"], c["hd"]) if ws else 0
    if short_ws is not None:
        nws = short_ws
    pws = up(np.zeros(max(nws, 16), np.uint8)) if nws else None
    for _ in range(2):  # the second call finds what the first left in the workspace
        wk.check(dev.wk_kv8_attention(b[0] + 2 * shift, rs, b[1] + 2 * shift, rs, b[2], b[3], b[4], b[5], c["n_pages"],
                                      b[6], c["table"].shape[0], c["table"].shape[1], b[7], b[8], rows, max_len,
                                      c["heads"], c["kv"], c["hd"], c["dt"], pws, nws))
    raw = down(b[0], sent.shape, np.uint16)
    free(*b, pws)
    body = raw[shift:shift + rows * rs].reshape(rows, rs)
    assert (body[:, w:] == 0x3555).all() and (raw[:shift] == 0x3555).all() and (raw[shift + rows * rs:] == 0x3555).all()
    return from_bits(np.ascontiguousarray(body[:, :w]).view(RAW[c["dt"]]), c["dt"])


def close(got, want, tol):
    assert np.isfinite(got).all()
    worst = float((np.abs(got - want) / np.maximum(tol, 1e-300)).max()) if want.size else 0.0
    print(f"largest error / tolerance {worst:.3f}, normwise {np.linalg.norm(got - want) / max(np.linalg.norm(want), 1e-30):.2e}")
    assert (np.abs(got - want) <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pos,heads,kv,hd,dt,beyond,ws", DECODES)
def test_decode_attention(dev, pos, heads, kv, hd, dt, beyond, ws):
    c = make_decode(pos, heads, kv, hd, dt, seed=heads * 31 + hd)
    want, tol = ref_decode(c)
    close(run_decode(dev, c, max(pos) + 1 + beyond, ws), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("ws", [False, True])
def test_decode_rows_of_one_sequence_strides_and_empty_rows(dev, ws):
    """Rows that share a sequence, odd strides and alignment, rows of no sequence, keys of no page."""
    c = make_decode([400, 401, 402, 10, 0], 6, 2, 64, wk.F16, seed=3, shared=True)
    want, tol = ref_decode(c)
    close(run_decode(dev, c, 403, ws, extra=3, shift=1), want, tol)
    c["seq"] = np.array([0, -1, 0, 1, 0])
    c["table"][0, 1], c["table"][0, 3] = -1, c["n_pages"]
    want, tol = ref_decode(c)
    assert not want[1].any() and not want[3].any()
    close(run_decode(dev, c, 403, ws), want, tol)
    c["table"][:] = -1
    assert not run_decode(dev, c, 403, ws).any()


@pytest.mark.gpu
def test_decode_workspace_too_small_and_repeatable(dev):
    c = make_decode([30000], 4, 1, 64, wk.F16, seed=8)
    want, tol = ref_decode(c)
    full = run_decode(dev, c, 30001, ws=True)
    close(full, want, tol)
    close(run_decode(dev, c, 30001, short_ws=4096), want, tol)
    assert np.array_equal(full, run_decode(dev, c, 30001, ws=True))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [wk.F16, wk.BF16])
def test_decode_large_and_uneven_values(dev, dt):
    """Queries whose scores differ by thousands; pages whose scales differ by 2^40; queries beyond fp16 in bf16."""
    c = make_decode([500, 130], 4, 2, 128, dt, seed=21)
    c["q"][0, :128] = rounded(c["q"][0, :128] * 300, dt)
    c["scales"][1][c["table"][0, 2]] *= 2.0 ** -40
    c["scales"][0][c["table"][1, 0]] *= 2.0 ** -20
    if dt == wk.BF16:
        c["q"][1] = rounded(c["q"][1] * 2.0 ** 100, dt)
        c["scales"][0][c["table"][1, :3]] = 2.0 ** -104
    want, tol = ref_decode(c)
    close(run_decode(dev, c, 501, ws=True), want, tol)


@pytest.mark.gpu
def test_decode_nan_stays_in_its_row_and_dimension(dev):
    c = make_decode([200, 300], 4, 2, 64, wk.F16, seed=4)
    c["codes"][1][c["table"][0, 1], 1, 5, 7] = 0x7F  # a NaN in V that row 0 sees, K/V head 1, dimension 7
    clean = {**c, "codes": [c["codes"][0], np.where(c["codes"][1] == 0x7F, 0, c["codes"][1])]}
    want, tol = ref_decode(clean)
    got = run_decode(dev, c, 301, ws=True)
    bad = np.zeros_like(want, bool).reshape(2, 4, 64)
    bad[0, 2:, 7] = True
    bad = bad.reshape(want.shape)
    assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
    assert (np.abs(got - want) <= tol)[~bad].all()


# ------------------------------------------------------------------ packed attention

PACKED = [
    # query and key lengths per sequence, heads, kv_heads, head_dim, dtype, row stride beyond the row, offset
    ([1], [1], 1, 1, 64, wk.F16, 0, 0),
    ([97], [97], 8, 2, 128, wk.F16, 0, 0),
    ([127, 128, 129], [127, 128, 129], 4, 4, 64, wk.BF16, 0, 0),
    ([255, 1, 257, 64], [255, 1, 257, 64], 4, 1, 128, wk.BF16, 8, 0),
    ([0, 300, 0, 0, 17], [0, 300, 0, 5, 17], 6, 2, 64, wk.F16, 64, 0),         # empty sequences
    ([10, 200, 3], [500, 200, 1000], 4, 2, 128, wk.F16, 0, 0),                 # behind a context
    ([150, 40, 5], [20, 0, 300], 3, 1, 64, wk.BF16, 0, 0),                     # queries that see nothing
    ([513], [1025], 16, 1, 64, wk.F16, 0, 0),
    ([70, 33], [70, 133], 14, 2, 128, wk.BF16, 0, 0),                          # 7 heads per K/V head
    ([90], [90], 24, 1, 64, wk.F16, 0, 0),                                     # 24 heads over one
    ([50, 260], [50, 400], 130, 1, 64, wk.BF16, 0, 0),                         # more heads than a tile has rows
    ([140, 30], [140, 90], 4, 2, 64, wk.F16, 3, 1),                            # not 16-byte aligned
    ([700] + [1] * 40 + [65] * 6, [700] + [1] * 40 + [65] * 6, 2, 1, 128, wk.F16, 0, 0),
    ([2100], [2100], 2, 2, 64, wk.BF16, 0, 0),
]


def make_packed(ql, kl, heads, kv, hd, dt, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    qs, ks = (np.concatenate([[0], np.cumsum(x)]) for x in (ql, kl))
    q = rounded(rng.standard_normal((qs[-1], heads * hd)) * spread, dt)
    k, v = (rounded(rng.standard_normal((ks[-1], kv * hd)), dt) for _ in range(2))
    return dict(q=q, k=k, v=v, qs=qs, ks=ks, heads=heads, kv=kv, hd=hd, dt=dt)


def ref_packed(c, rows=None):
    g, hd = c["heads"] // c["kv"], c["hd"]
    out, tol = np.zeros(c["q"].shape), np.zeros(c["q"].shape)
    for i in range(len(c["qs"]) - 1):
        q0, k0 = c["qs"][i], c["ks"][i]
        ql, kl = c["qs"][i + 1] - q0, c["ks"][i + 1] - k0
        for h in range(c["heads"]):
            a = h // g
            k, v = (c[x][k0:k0 + kl, a * hd:(a + 1) * hd] for x in "kv")
            for j in range(ql):
                n = kl - ql + j + 1
                at = slice(h * hd, (h + 1) * hd)
                out[q0 + j, at], tol[q0 + j, at] = attend(c["q"][q0 + j, at], k, v, n, c["dt"])
    return out, tol


def run_packed(dev, c, extra=0, shift=0, tail=3):
    def laid(x):
        full = np.full((len(x) + tail, x.shape[1] + extra), np.nan)  # what is behind rows and sequences must not matter
        full[: len(x), : x.shape[1]] = x
        return np.concatenate([np.zeros(shift, RAW[c["dt"]]), to_bits(full, c["dt"]).reshape(-1)]), x.shape[1] + extra
    (q, q_rs), (k, k_rs), (v, v_rs) = (laid(c[x]) for x in "qkv")
    rows = len(c["q"])
    sent = np.full(len(q), 0x3555, np.uint16)
    b = [up(x) for x in (sent, q, k, v, c["qs"].astype(np.int32), c["ks"].astype(np.int32))]
    o = 2 * shift
    wk.check(dev.wk_attention_packed(b[0] + o, q_rs, b[1] + o, q_rs, b[2] + o, k_rs, b[3] + o, v_rs, b[4], b[5],
                                     len(c["qs"]) - 1, rows + tail, len(c["k"]) + tail, c["heads"], c["kv"], c["hd"],
                                     c["dt"]))
    raw = down(b[0], sent.shape, np.uint16)
    assert dev.wk_device_error(0) == 0
    free(*b)
    body = raw[shift:].reshape(rows + tail, q_rs)
    assert (body[rows:] == 0x3555).all() and (body[:, c["q"].shape[1]:] == 0x3555).all()
    return from_bits(np.ascontiguousarray(body[:rows, : c["q"].shape[1]]).view(RAW[c["dt"]]), c["dt"])


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,heads,kv,hd,dt,extra,shift", PACKED)
def test_packed_attention(dev, ql, kl, heads, kv, hd, dt, extra, shift):
    c = make_packed(ql, kl, heads, kv, hd, dt, seed=sum(ql) + heads)
    want, tol = ref_packed(c)
    close(run_packed(dev, c, extra, shift), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,heads,kv,hd,dt,extra,shift", PACKED)
def test_packed_attention_beside_a_long_sequence(dev, ql, kl, heads, kv, hd, dt, extra, shift):
    """The same with a token behind a long context, whose length decides how all of them are computed."""
    c = make_packed([*ql, 1], [*kl, 250 * (len(kl) + 1)], heads, kv, hd, dt, seed=sum(ql) + heads)
    want, tol = ref_packed(c)
    close(run_packed(dev, c, extra, shift), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("ql,kl,heads,kv,hd,dt,extra", [
    ([1] * 9, [1, 2, 3, 4, 60, 64, 65, 100, 130], 4, 1, 128, wk.BF16, 8),
    ([64, 63, 65, 31, 1, 40], [64, 63, 65, 31, 1, 90], 6, 6, 64, wk.F16, 0),       # one head per K/V head
    ([33, 100, 7], [33, 100, 7], 15, 3, 64, wk.BF16, 0),                             # 5: units begin inside a position
    ([20, 50], [100, 5], 64, 1, 128, wk.F16, 64),
    ([4, 9, 2], [40, 9, 120], 65, 1, 64, wk.F16, 0),
    ([100], [120], 7, 1, 128, wk.BF16, 0),
    ([3, 0, 0, 120, 5] * 30, [10, 0, 7, 120, 2] * 30, 4, 2, 64, wk.F16, 0),          # more of them than a CTA has threads
    ([1, 700, 2] + [1] * 27, [1, 700, 2] + [1] * 27, 4, 2, 128, wk.F16, 0),          # one among them is long
])
def test_packed_short_sequences(dev, ql, kl, heads, kv, hd, dt, extra):
    c = make_packed(ql, kl, heads, kv, hd, dt, seed=len(ql) + hd)
    want, tol = ref_packed(c)
    got = run_packed(dev, c, extra)
    close(got, want, tol)
    assert np.array_equal(got, run_packed(dev, c, extra))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [wk.F16, wk.BF16])
def test_packed_short_steep_scores(dev, dt):
    c = make_packed([70, 20], [110, 20], 4, 2, 128, dt, seed=2, spread=12.0)
    ramp = np.linspace(0.01, 3.0, 130)[:, None]
    c["k"] = rounded(np.abs(c["k"]) * ramp, dt)
    c["q"] = rounded(np.abs(c["q"]), dt)
    want, tol = ref_packed(c)
    close(run_packed(dev, c), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("hd", [64, 128])
def test_packed_short_later_keys_do_not_touch_earlier_queries(dev, bad, hd):
    c = make_packed([100, 20], [100, 30], 6, 2, hd, wk.F16, seed=7)
    want, tol = ref_packed(c)
    for name in "kv":
        d = dict(c, **{name: c[name].copy()})
        d[name][37, 3] = bad  # sequence 0, K/V head 0, dimension 3
        got = run_packed(dev, d)
        same = np.ones(want.shape, bool)
        same[37:100, :3 * hd] = False
        if name == "v":
            seen = np.zeros(want.shape, bool)
            seen[37:100, [3, hd + 3, 2 * hd + 3]] = True
            assert not np.isfinite(got[seen]).any() and (np.isnan(got[seen]) == np.isnan(bad)).all()
            same = ~seen
        assert (np.abs(got - want) <= tol)[same].all()


@pytest.mark.gpu
@pytest.mark.parametrize("shift,extra", [(1, 0), (0, 3)])
def test_packed_short_with_an_output_of_any_alignment(dev, shift, extra):
    c = make_packed([40, 9], [40, 25], 4, 2, 64, wk.BF16, seed=3)
    want, tol = ref_packed(c)
    w = c["q"].shape[1]
    b = [up(to_bits(c[x], wk.BF16)) for x in "qkv"] + [up(c[x].astype(np.int32)) for x in ("qs", "ks")]
    out = up(np.full(49 * (w + extra) + shift, 0x3555, np.uint16))
    wk.check(dev.wk_attention_packed(out + 2 * shift, w + extra, b[0], w, b[1], 128, b[2], 128, b[3], b[4], 2, 49, 65, 4, 2,
                                     64, wk.BF16))
    raw = down(out, 49 * (w + extra) + shift, np.uint16)
    free(*b, out)
    body = raw[shift:].reshape(49, w + extra)
    assert (raw[:shift] == 0x3555).all() and (body[:, w:] == 0x3555).all()
    close(from_bits(np.ascontiguousarray(body[:, :w]).view(RAW[wk.BF16]), wk.BF16), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [wk.F16, wk.BF16])
def test_packed_steep_scores(dev, dt):
    """Scores that differ by hundreds, with the largest at the last keys, so that the running maximum keeps growing."""
    c = make_packed([300], [700], 4, 2, 128, dt, seed=2, spread=12.0)
    ramp = np.linspace(0.01, 3.0, 700)[:, None]
    c["k"] = rounded(np.abs(c["k"]) * ramp, dt)
    c["q"] = rounded(np.abs(c["q"]), dt)
    want, tol = ref_packed(c)
    close(run_packed(dev, c), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_packed_sequences_do_not_touch_each_other(dev, bad):
    """NaN or infinities throughout one sequence leave its neighbours as they are without it."""
    ql, kl = [70, 60, 90], [100, 60, 90]
    c = make_packed(ql, kl, 4, 2, 64, wk.F16, seed=6)
    want, tol = ref_packed(c)
    d = dict(c, **{x: c[x].copy() for x in "qkv"})
    d["k"][c["ks"][1]:c["ks"][2]] = bad
    d["v"][c["ks"][1]:c["ks"][2]] = bad
    d["q"][c["qs"][1]:c["qs"][2]] = bad
    got = run_packed(dev, d)
    for i in (0, 2):
        at = slice(c["qs"][i], c["qs"][i + 1])
        close(got[at], want[at], tol[at])
    assert not np.isfinite(got[c["qs"][1]:c["qs"][2]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("hd", [64, 128])
def test_packed_later_keys_do_not_touch_earlier_queries(dev, bad, hd):
    """A NaN or an infinity in K or V reaches the queries that see it, and no other."""
    c = make_packed([300], [300], 4, 2, hd, wk.BF16, seed=7)
    want, tol = ref_packed(c)
    for name in "kv":
        d = dict(c, **{name: c[name].copy()})
        d[name][137, 3] = bad  # K/V head 0, dimension 3
        got = run_packed(dev, d)
        close(got[:137], want[:137], tol[:137])
        close(got[137:, 2 * hd:], want[137:, 2 * hd:], tol[137:, 2 * hd:])  # the heads of K/V head 1
        if name == "v":
            seen = np.zeros(want.shape, bool)
            seen[137:, [3, hd + 3]] = True
            assert not np.isfinite(got[seen]).any()
            assert (np.abs(got - want) <= tol)[~seen].all()
        elif np.isnan(bad):
            assert np.isnan(got[137:, : 2 * hd]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [wk.F16, wk.BF16])
def test_packed_many_short_sequences_and_a_late_start(dev, dt):
    """More sequences than one pass over their lengths takes; the first starts behind rows of nobody."""
    rng = np.random.default_rng(5)
    ql = rng.integers(0, 4, 900)
    kl = ql + rng.integers(0, 3, 900)
    c = make_packed([7, *ql], [9, *kl], 6, 3, 64, dt, seed=17)
    want, tol = ref_packed(c)
    d = dict(c, qs=c["qs"][1:], ks=c["ks"][1:])
    got = run_packed(dev, d)
    assert (to_bits(got[:7], dt).view(np.uint16) == 0x3555).all()  # not written
    close(got[7:], want[7:], tol[7:])
    assert np.array_equal(got[7:], run_packed(dev, d)[7:])


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0, 1])
def test_packed_without_keys(dev, shift):
    c = make_packed([5, 70], [0, 0], 4, 2, 64, wk.F16, seed=1)
    assert not run_packed(dev, c, shift=shift, tail=0).any()


# ------------------------------------------------------------------ other ways to share the work out

@pytest.mark.gpu
@pytest.mark.parametrize("lens,heads,kv,hd,dt", [
    (list(range(3, 2400, 57)), 8, 2, 64, wk.F16),            # equal runs, parts joined by the last to arrive
    ([0, 1800, -1, 900, 33, 0, 1200, 64] * 4, 32, 8, 128, wk.BF16),
    ([4000, 1, 30, 70] * 5, 32, 2, 128, wk.F16),             # 16 heads per K/V head; long rows among short ones
    ([150000], 4, 1, 64, wk.F16),                            # one row: several clusters to a head group
    ([70000, 0, 70000], 40, 2, 128, wk.BF16),                # a second launch joins the parts
    ([5] * 2100, 2, 1, 64, wk.F16),                          # more rows than equal runs take
    ([0, 1800, -1, 900, 33, 0, 1200, 64] * 8, 16, 8, 128, wk.F16),
    ([2500, 1, 30, 70] * 25, 32, 2, 128, wk.BF16),
    (list(range(1, 2600, 33)), 8, 8, 64, wk.BF16),
])
def test_decode_shares(dev, lens, heads, kv, hd, dt):
    c = make_decode([n - 1 for n in lens], heads, kv, hd, dt, seed=len(lens) + hd)
    want, tol = ref_decode(c)
    got = run_decode(dev, c, max(lens), ws=True)
    close(got, want, tol)
    assert np.array_equal(got, run_decode(dev, c, max(lens), ws=True))
    close(run_decode(dev, c, max(lens), ws=False), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("n,heads,kv,hd,dt", [
    (16383, 32, 8, 128, wk.BF16),
    (40001, 7, 1, 128, wk.F16),   # 7 heads: the last CTA of a cluster joins fewer outputs
    (9000, 40, 4, 128, wk.F16),   # 10 heads per K/V head, in one CTA
    (19000, 40, 4, 128, wk.BF16),
    (20000, 24, 1, 64, wk.BF16),  # 24 of them, in two
    (33000, 3, 3, 64, wk.F16),
])
def test_decode_one_long_row(dev, n, heads, kv, hd, dt):
    """Several clusters to a head group; the row as long as announced, much shorter, a padding row."""
    c = make_decode([n - 1], heads, kv, hd, dt, seed=n)
    need = dev.wk_kv8_attention_ws(1, n, heads, kv, hd)
    for pos in (n - 1, 1000, 0, -1):
        d = dict(c, pos=np.array([pos]))
        want, tol = ref_decode(d)
        got = run_decode(dev, d, n, ws=True)
        close(got, want, tol)
        assert np.array_equal(got, run_decode(dev, d, n, ws=True))
        close(run_decode(dev, d, n, short_ws=max(need - 1, 0)), want, tol)


@pytest.mark.gpu
def test_decode_workspace_serves_calls_of_other_sizes(dev):
    """One workspace through calls of different shapes, in turn, each as from a fresh one."""
    cases = [make_decode([n - 1 for n in lens], *shape, seed=7) for lens, shape in (
        ([0, 1800, -1, 900, 33, 0, 1200, 64] * 8, (16, 8, 128, wk.F16)), ([150000], (4, 1, 64, wk.F16)),
        ([2500, 1, 30, 70] * 25, (32, 2, 128, wk.F16)), (list(range(1, 2600, 33)), (8, 8, 64, wk.F16)))]
    n = max(dev.wk_kv8_attention_ws(len(c["pos"]), int(c["pos"].max()) + 1, c["heads"], c["kv"], c["hd"]) for c in cases)
    ws = up(np.zeros(n, np.uint8))
    wants = [ref_decode(c) for c in cases]
    for c, (want, tol) in [*zip(cases, wants), *zip(cases[::-1], wants[::-1])]:
        rows, w = c["q"].shape
        b = [up(v) for v in (np.zeros((rows, w), np.float16), to_bits(c["q"], c["dt"]), *c["codes"],
                             *(s.astype(np.float32) for s in c["scales"]), c["table"].astype(np.int32),
                             c["seq"].astype(np.int32), c["pos"].astype(np.int32))]
        wk.check(dev.wk_kv8_attention(b[0], w, b[1], w, b[2], b[3], b[4], b[5], c["n_pages"], b[6], *c["table"].shape,
                                      b[7], b[8], rows, int(c["pos"].max()) + 1, c["heads"], c["kv"], c["hd"], c["dt"],
                                      ws, n))
        close(down(b[0], (rows, w), np.float16).astype(np.float64), want, tol)
        free(*b)
    free(ws)


@pytest.mark.gpu
def test_offsets_beyond_32_bits(dev):
    """A cache of more than 2^32 bytes: stored to and read from pages at both ends."""
    kv, hd = 8, 128
    page_bytes = kv * PAGE * hd
    n_pages = (1 << 32) // page_bytes + 40
    pools = [alloc(n_pages * page_bytes) for _ in range(2)]
    scales = [up(np.ones((n_pages, kv), np.float32)) for _ in range(2)]
    rng = np.random.default_rng(3)
    lens = np.array([150, 70])
    table = np.array([[n_pages - 1, 0, n_pages - 3], [n_pages - 2, 1, -1]])
    starts = np.array([0, 150, 220])
    x = [rounded(rng.standard_normal((220, kv * hd)), wk.F16) for _ in range(2)]
    b = [up(to_bits(v, wk.F16)) for v in x] + [up(v.astype(np.int32)) for v in (starts, np.zeros(2), table)]
    wk.check(dev.wk_kv8_store(*pools, *scales, n_pages, b[0], kv * hd, b[1], kv * hd, b[2], b[3], 2, 220, b[4], 3, kv, hd,
                              wk.F16))
    c = dict(pos=lens - 1, seq=np.arange(2), table=np.where(table < 0, -1, np.searchsorted([0, 1, n_pages - 3, n_pages - 2,
             n_pages - 1], table)), heads=16, kv=kv, hd=hd, dt=wk.F16, n_pages=5,
             q=rounded(rng.standard_normal((2, 16 * hd)), wk.F16))
    codes, sc = zip(*(ref_store(np.zeros((5, kv, PAGE, hd), np.uint8), np.ones((5, kv)), v.reshape(220, kv, hd), starts,
                                [0, 0], c["table"], 5) for v in x))
    want, tol = ref_decode(dict(c, codes=list(codes), scales=list(sc)))
    q, out, seq, pos = up(to_bits(c["q"], wk.F16)), alloc(2 * c["q"].size), up(np.arange(2, dtype=np.int32)), \
        up((lens - 1).astype(np.int32))
    wk.check(dev.wk_kv8_attention(out, 16 * hd, q, 16 * hd, *pools, *scales, n_pages, b[4], 2, 3, seq, pos, 2, 150, 16, kv,
                                  hd, wk.F16, None, 0))
    close(down(out, c["q"].shape, np.float16).astype(np.float64), want, tol)
    free(*pools, *scales, *b, q, out, seq, pos)


@pytest.mark.gpu
def test_packed_rows_beyond_32_bits(dev):
    """Rows so far apart that the last ones lie more than 2^32 bytes behind the first."""
    c = make_packed([30, 9], [30, 40], 2, 1, 64, wk.F16, seed=3)
    rs = 1 << 26  # elements: 128 MB from row to row
    q, k, v, out = (alloc(2 * (n - 1) * rs + 2 * w) for n, w in ((39, 128), (70, 64), (70, 64), (39, 128)))
    L = wk.lib()
    for p, x in ((q, c["q"]), (k, c["k"]), (v, c["v"])):
        bits = to_bits(x, wk.F16)
        for r in range(len(x)):
            L.cuda_to_device(p + 2 * r * rs, as_p(np.ascontiguousarray(bits[r])), bits[r].nbytes)
    qs, ks = up(c["qs"].astype(np.int32)), up(c["ks"].astype(np.int32))
    wk.check(L.wk_attention_packed(out, rs, q, rs, k, rs, v, rs, qs, ks, 2, 39, 70, 2, 1, 64, wk.F16))
    got = np.stack([down(out + 2 * r * rs, 128, np.float16) for r in range(39)]).astype(np.float64)
    want, tol = ref_packed(c)
    close(got, want, tol)
    free(q, k, v, out, qs, ks)


# ------------------------------------------------------------------ a serving loop

class Loop:
    """Sequences of one layer over the four entry points, and what the cache should hold, in 64 bits."""

    def __init__(self, dev, n, heads, kv, hd, dt, n_pages, max_pages, rows_cap, seed):
        self.dev, self.n, self.heads, self.kv, self.hd, self.dt = dev, n, heads, kv, hd, dt
        self.n_pages, self.max_pages, self.rows_cap = n_pages, max_pages, rows_cap
        self.rng = np.random.default_rng(seed)
        self.w = (heads + 2 * kv) * hd
        self.ws_bytes = dev.wk_kv8_attention_ws(rows_cap, max_pages * PAGE, heads, kv, hd)
        i32 = lambda *s: up(np.zeros(s, np.int32))  # noqa: E731
        self.free_list = self.rng.permutation(n_pages)
        self.taken = 0
        self.d = dict(k=up(np.zeros(n_pages * kv * PAGE * hd, np.uint8)), v=up(np.zeros(n_pages * kv * PAGE * hd, np.uint8)),
                      ks=up(np.ones((n_pages, kv), np.float32)), vs=up(np.ones((n_pages, kv), np.float32)),
                      table=up(np.full((n, max_pages), -1, np.int32)), starts=i32(n + 1), ctx=i32(n), lens=i32(n),
                      seq=i32(rows_cap), pos=i32(rows_cap), slot=up(np.zeros(rows_cap, np.int64)), status=i32(3),
                      add=i32(n), free=up(self.free_list.astype(np.int32)), n_free=up(np.array([n_pages], np.int32)),
                      qkv=up(np.zeros((rows_cap, self.w), np.uint16)), out=up(np.zeros((rows_cap, heads * hd), np.uint16)),
                      ws=up(np.zeros(max(self.ws_bytes, 16), np.uint8)))
        self.ctx = np.zeros(n, int)
        self.table = np.full((n, max_pages), -1)
        self.codes = [np.zeros((n_pages, kv, PAGE, hd), np.uint8) for _ in range(2)]
        self.scales = [np.ones((n_pages, kv)) for _ in range(2)]

    def put(self, name, x):
        x = np.ascontiguousarray(x)
        self.dev.cuda_to_device(self.d[name], as_p(x), x.nbytes)

    def inputs(self, add):
        """New rows of the sequences, the lengths and the rest of the free list."""
        self.add = np.array(add)
        rows = int(self.add.sum())
        self.x = rounded(self.rng.standard_normal((rows, self.w)) * self.rng.choice([0.5, 1.0, 3.0], (rows, 1)), self.dt)
        self.put("qkv", to_bits(self.x, self.dt))
        self.put("ctx", self.ctx.astype(np.int32))
        self.put("add", self.add.astype(np.int32))
        self.put("free", np.roll(self.free_list, -self.taken).astype(np.int32))
        self.put("n_free", np.array([self.n_pages - self.taken], np.int32))

    def launch(self, prompts):
        """One step: its calls, and nothing that waits."""
        D, d, es = self.dev, self.d, 2
        wk.check(D.wk_batch_plan(d["starts"], d["lens"], d["seq"], d["pos"], d["slot"], self.rows_cap, d["table"],
                                 self.max_pages, d["status"], d["ctx"], d["add"], self.n, d["free"], d["n_free"],
                                 self.n_pages))
        q, k, v = d["qkv"], d["qkv"] + es * self.heads * self.hd, d["qkv"] + es * (self.heads + self.kv) * self.hd
        wk.check(D.wk_kv8_store(d["k"], d["v"], d["ks"], d["vs"], self.n_pages, k, self.w, v, self.w, d["starts"], d["ctx"],
                                self.n, self.rows_cap, d["table"], self.max_pages, self.kv, self.hd, self.dt))
        ow = self.heads * self.hd
        if prompts:
            wk.check(D.wk_attention_packed(d["out"], ow, q, self.w, k, self.w, v, self.w, d["starts"], d["starts"], self.n,
                                           self.rows_cap, self.rows_cap, self.heads, self.kv, self.hd, self.dt))
        else:
            wk.check(D.wk_kv8_attention(d["out"], ow, q, self.w, d["k"], d["v"], d["ks"], d["vs"], self.n_pages,
                                        d["table"], self.n, self.max_pages, d["seq"], d["pos"], self.rows_cap,
                                        self.max_pages * PAGE, self.heads, self.kv, self.hd, self.dt, d["ws"],
                                        self.ws_bytes))

    def verify(self, prompts):
        p = ref_plan(self.ctx, self.add, self.table, np.roll(self.free_list, -self.taken), self.n_pages - self.taken,
                     self.rows_cap)
        for name, key, t in (("seq", "row_seq", np.int32), ("pos", "row_pos", np.int32), ("slot", "row_slot", np.int64),
                             ("table", "table", np.int32), ("lens", "lens", np.int32), ("status", "status", np.int32)):
            assert np.array_equal(down(self.d[name], p[key].shape, t), p[key]), name
        self.table = p["table"]
        rows, H, kv, hd = len(self.x), self.heads * self.hd, self.kv, self.hd
        for i, name in enumerate("kv"):
            x = self.x[:, H + i * kv * hd:H + (i + 1) * kv * hd].reshape(rows, kv, hd)
            self.codes[i], self.scales[i] = ref_store(self.codes[i], self.scales[i], x, p["starts"], self.ctx, self.table,
                                                      self.n_pages)
            got = down(self.d[name], self.codes[i].shape, np.uint8)
            assert same_codes(got, self.codes[i]).all()
            assert np.array_equal(down(self.d[name + "s"], (self.n_pages, kv), np.float32), self.scales[i])
        out = from_bits(down(self.d["out"], (self.rows_cap, H), RAW[self.dt]), self.dt)
        c = dict(heads=self.heads, kv=kv, hd=hd, dt=self.dt, q=self.x[:, :H])
        if prompts:
            want, tol = ref_packed(dict(c, k=self.x[:, H:H + kv * hd], v=self.x[:, H + kv * hd:], qs=p["starts"],
                                        ks=p["starts"]))
        else:
            want, tol = ref_decode(dict(c, pos=p["row_pos"][:rows], seq=p["row_seq"][:rows], table=self.table,
                                        codes=self.codes, scales=self.scales, n_pages=self.n_pages))
            assert not out[rows:].any()  # the rows behind the last sequence have no position: zeros
        close(out[:rows], want, tol)
        self.taken += int(p["status"][1])
        self.ctx = p["lens"]

    def end(self):
        free(*self.d.values())


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,dt", [(8, 2, 64, wk.F16), (8, 1, 128, wk.BF16)])
def test_serving_loop(dev, heads, kv, hd, dt):
    """Prompts, then steps in which sequences bring one token, several, or none; pages are taken as they fill."""
    loop = Loop(dev, 5, heads, kv, hd, dt, n_pages=40, max_pages=8, rows_cap=400, seed=hd)
    adds = [[64, 130, 1, 63, 0], [1, 1, 1, 1, 0], [1, 0, 1, 1, 0], [3, 1, 62, 1, 90], [1, 1, 1, 1, 1]]
    for i, add in enumerate(adds):
        loop.inputs(add)
        loop.launch(prompts=i == 0)
        loop.verify(prompts=i == 0)
    loop.end()


@pytest.mark.gpu
def test_serving_loops_captured_and_replayed_in_turn(dev):
    """Two loops' steps as graphs that run in turn, each with a workspace of its own, beside calls made directly."""
    torch = pytest.importorskip("torch")
    stream = torch.cuda.ExternalStream(dev.wk_stream())
    loops = [Loop(dev, 6, 8, 2, 128, wk.F16, 60, 8, 128, seed=1), Loop(dev, 3, 4, 4, 64, wk.BF16, 40, 16, 96, seed=2)]
    graphs = []
    for loop, prompt in zip(loops, ([20, 30, 1, 0, 5, 64], [90, 1, 3])):
        loop.inputs(prompt)
        loop.launch(prompts=True)
        loop.verify(prompts=True)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            loop.launch(prompts=False)
        graphs.append(g)
    for step in range(4):
        for loop, g in zip(loops, graphs):
            loop.inputs([1] * loop.n if step % 2 == 0 else [int(i != step % loop.n) for i in range(loop.n)])
            with torch.cuda.stream(stream):
                g.replay()
            loop.verify(prompts=False)
        loops[0].inputs([2] * loops[0].n)
        loops[0].launch(prompts=False)
        loops[0].verify(prompts=False)
    torch.cuda.synchronize()
    del graphs, g
    for loop in loops:
        loop.end()
