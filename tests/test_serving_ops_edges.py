"""Edges of the serving operators: an attention sink far ahead of the keys that carry the output.

Tolerances.  As in the other file, with what it leaves out: a softmax weight is
multiplied with V in 16 bits, and in fp16 it is exact to half of 2^-24 at the
least.  The kernels multiply the weights by 2^9 or more, relative to a score that
some key of the row reaches, so that this is at most 2^-34 of that key's weight,
and the weights sum to at least one such: 2^-34 sum |v| of the keys that a row
sees.  An output in fp16 is exact to 2^-25 at the least.
"""
import math
import os
import subprocess
import sys

import numpy as np
import pytest

import wukong_b200 as wk
from tests import test_serving_ops as ops
from tests.gpu_util import alloc, down, free, up
from tests.test_serving_ops import CODES, PAGE, UNIT, e4m3_codes, rounded, run_decode, run_packed, to_bits


def attend(q, k, v, dt):
    """softmax(q k^T / sqrt(d)) v for one query, and how far off a kernel may be."""
    d, n = q.shape[-1], len(k)
    s = k @ q / math.sqrt(d)
    p = np.exp(s - s.max())
    p /= p.sum()
    o, A = p @ v, p @ np.abs(v)
    S = (np.abs(k) @ np.abs(q)).max() / math.sqrt(d)
    u = UNIT[dt]
    tol = u * np.abs(o) + A * (u + 2 * (d * 2.0 ** -24 * S + 2.0 ** -20) + n * 2.0 ** -24) * (1 + u)
    return o, tol + 2.0 ** -34 * np.abs(v).sum(0) + (2.0 ** -25 if dt == wk.F16 else 0.0)


def near(got, want, tol):
    assert np.isfinite(got).all()
    print(f"largest error / tolerance {float((np.abs(got - want) / np.maximum(tol, 1e-300)).max()):.3f}")
    assert (np.abs(got - want) <= tol).all()


def sinks(rng, n, hd, gap, every):
    """Keys with scores near 0, every so many of them one whose score is `gap` for a query of gap / sqrt(hd)
    throughout and whose V is zero."""
    k, v = 0.3 * rng.standard_normal((n, hd)), 1000.0 * (1 + 0.3 * rng.standard_normal((n, hd)))
    k[::every], v[::every] = 1.0, 0.0
    return k, v


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [12.0, 15.0, 18.0])
@pytest.mark.parametrize("lens,heads,kv,hd,dt,ws", [
    ([777], 16, 4, 64, wk.F16, True),
    ([300, 5, 1, 450, 333] * 6, 16, 8, 128, wk.BF16, False),
    ([40, 2000, 130, 700] * 8, 32, 2, 128, wk.F16, True),   # 16 heads per K/V head, equal runs
    ([9000], 8, 1, 128, wk.BF16, True),                     # several clusters to a head group
])
def test_decode_keeps_the_weights_behind_a_sink(dev, lens, heads, kv, hd, dt, ws, gap):
    rng = np.random.default_rng(int(gap) + heads)
    c = ops.make_decode([n - 1 for n in lens], heads, kv, hd, dt, seed=int(gap))
    c["scales"] = [np.full_like(c["scales"][0], 2.0 ** -5), np.full_like(c["scales"][1], 2.0 ** 4)]
    c["q"] = rounded(np.full(c["q"].shape, gap / math.sqrt(hd)), dt)
    want, tol = np.zeros((len(lens), heads, hd)), np.zeros((len(lens), heads, hd))
    for r, n in enumerate(lens):
        pages = c["table"][r, : -(-n // PAGE)]
        for a in range(kv):
            kv_values = []
            for x, values in enumerate(sinks(rng, n, hd, gap, 32)):
                codes = e4m3_codes(values / c["scales"][x][0, 0])
                for j, page in enumerate(pages):
                    part = codes[j * PAGE:(j + 1) * PAGE]
                    c["codes"][x][page, a, : len(part)] = part
                kv_values.append(CODES[codes] * c["scales"][x][0, 0])
            for h in range(a * heads // kv, (a + 1) * heads // kv):
                want[r, h], tol[r, h] = attend(c["q"][r].reshape(heads, hd)[h], *kv_values, dt)
    near(run_decode(dev, c, max(lens), ws), want.reshape(len(lens), -1), tol.reshape(len(lens), -1))


def huge_scores(n, hd, score):
    """Keys whose scores are `score`, and minus it for the odd ones, for a query of 2^10 throughout; key 5 leads with half as much again."""
    k = np.zeros((n, hd))
    k[:, 0] = score * math.sqrt(hd) / 2.0 ** 10
    k[1::2, 0] *= -1
    k[5, 0] *= -1.5
    return k


@pytest.mark.gpu
@pytest.mark.parametrize("score", [3e5, 1e7, 3e7, 6e7, 9e7])
@pytest.mark.parametrize("heads,kv,hd,dt", [(16, 4, 64, wk.F16), (32, 2, 128, wk.BF16)])
def test_decode_scores_of_any_size(dev, score, heads, kv, hd, dt):
    """One key leads the others by millions: its V comes out."""
    c = ops.make_decode([400, 130], heads, kv, hd, dt, seed=5)
    k = huge_scores(401, hd, score)
    c["scales"][0][:] = 2.0 ** math.ceil(math.log2(np.abs(k).max() / 448))
    c["q"] = rounded(np.full(c["q"].shape, 2.0 ** 10), dt)
    codes = e4m3_codes(k / c["scales"][0][0, 0])
    for r, n in enumerate([401, 131]):
        for j, page in enumerate(c["table"][r, : -(-n // PAGE)]):
            part = codes[j * PAGE:min((j + 1) * PAGE, n)]
            c["codes"][0][page, :, : len(part)] = part
    want, tol = ops.ref_decode(c)
    ops.close(run_decode(dev, c, 401, ws=True), want, tol)


def packed_with_sinks(ql, kl, heads, kv, hd, dt, gap, seed):
    rng = np.random.default_rng(seed)
    c = ops.make_packed(ql, kl, heads, kv, hd, dt, seed)
    c["q"] = rounded(np.full(c["q"].shape, gap / math.sqrt(hd)), dt)
    for i in range(len(kl)):
        for a in range(kv):
            at = slice(c["ks"][i], c["ks"][i + 1]), slice(a * hd, (a + 1) * hd)
            c["k"][at], c["v"][at] = (rounded(x, dt) for x in sinks(rng, kl[i], hd, gap, 200))
    want, tol = np.zeros(c["q"].shape), np.zeros(c["q"].shape)
    for i in range(len(ql)):
        for h in range(heads):
            a = h * kv // heads
            k, v = (c[x][c["ks"][i]:c["ks"][i + 1], a * hd:(a + 1) * hd] for x in "kv")
            for j in range(ql[i]):
                n, at = kl[i] - ql[i] + j + 1, (c["qs"][i] + j, slice(h * hd, (h + 1) * hd))
                want[at], tol[at] = attend(c["q"][at], k[:n], v[:n], dt)
    return c, want, tol


@pytest.mark.gpu
@pytest.mark.parametrize("gap", [12.0, 15.0, 18.0])
@pytest.mark.parametrize("ql,kl,heads,kv,hd,dt", [
    ([300], [700], 4, 2, 128, wk.F16),
    ([400, 90], [400, 500], 2, 1, 64, wk.F16),
    ([60], [2600], 2, 1, 128, wk.F16),              # a cluster shares the keys
    ([300], [700], 4, 2, 128, wk.BF16),
    ([50, 90], [60, 90], 6, 2, 64, wk.F16),         # the kernel of short sequences
])
def test_packed_keeps_the_weights_behind_a_sink(dev, ql, kl, heads, kv, hd, dt, gap):
    c, want, tol = packed_with_sinks(ql, kl, heads, kv, hd, dt, gap, seed=int(gap) + heads)
    near(run_packed(dev, c), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("score", [3e5, 1e7, 3e7, 6e7, 9e7])
@pytest.mark.parametrize("ql,kl,heads,kv,hd,dt", [
    ([300], [700], 4, 2, 128, wk.F16),
    ([40], [2600], 2, 1, 64, wk.F16),
    ([50, 90], [60, 90], 6, 2, 64, wk.F16),
    ([50, 90], [60, 90], 6, 2, 128, wk.BF16),
    ([300], [400], 4, 4, 64, wk.BF16),
])
def test_packed_scores_of_any_size(dev, ql, kl, heads, kv, hd, dt, score):
    c = ops.make_packed(ql, kl, heads, kv, hd, dt, seed=3)
    c["q"] = rounded(np.full(c["q"].shape, 2.0 ** 10), dt)
    for i, n in enumerate(kl):
        one = huge_scores(n, hd, score)[:, :1] / hd
        c["k"][c["ks"][i]:c["ks"][i + 1]] = rounded(np.repeat(one, kv * hd, 1), dt)
    want, tol = ops.ref_packed(c)
    ops.close(run_packed(dev, c), want, tol)


# bf16 holds values up to 2^128: a mean of such values is one too, and the sum on the way to it must not pass fp32's range

@pytest.mark.gpu
@pytest.mark.parametrize("power", [127, 120, 0, -90, -100])
@pytest.mark.parametrize("ql,kl,heads,kv,hd,extra,shift", [
    ([300], [700], 4, 2, 128, 0, 0),
    ([40], [2600], 2, 1, 64, 0, 0),
    ([50, 90], [60, 90], 6, 2, 64, 0, 0),
    ([50, 90], [60, 90], 6, 2, 128, 0, 0),
    ([9, 40], [60, 40], 2, 1, 128, 3, 1),
])
def test_packed_values_of_any_size(dev, ql, kl, heads, kv, hd, extra, shift, power):
    c = ops.make_packed(ql, kl, heads, kv, hd, wk.BF16, seed=4)
    rng = np.random.default_rng(4)
    c["v"] = rounded(rng.uniform(0.5, 1.0, c["v"].shape), wk.BF16) * 2.0 ** power
    want, tol = np.zeros(c["q"].shape), np.zeros(c["q"].shape)
    for i in range(len(ql)):
        for h in range(heads):
            a = h * kv // heads
            k, v = (c[x][c["ks"][i]:c["ks"][i + 1], a * hd:(a + 1) * hd] for x in "kv")
            for j in range(ql[i]):
                n, at = kl[i] - ql[i] + j + 1, (c["qs"][i] + j, slice(h * hd, (h + 1) * hd))
                want[at], tol[at] = attend(c["q"][at], k[:n], v[:n], wk.BF16)
    near(run_packed(dev, c, extra, shift), want, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("power", [119, 100, 0, -90, -100])
@pytest.mark.parametrize("lens,heads,kv,hd,ws", [
    ([777], 16, 4, 64, True),
    ([300, 5, 1, 450, 333] * 6, 16, 8, 128, False),
    ([40, 2000, 130, 700] * 8, 32, 2, 128, True),
    ([9000], 8, 1, 128, True),
])
def test_decode_values_of_any_size(dev, lens, heads, kv, hd, ws, power):
    """Page scales from the least to the largest that bf16 rows give, codes up to 448."""
    c = ops.make_decode([n - 1 for n in lens], heads, kv, hd, wk.BF16, seed=6)
    rng = np.random.default_rng(6)
    values = np.where(c["codes"][1] == 0x7F, np.nan, rng.uniform(200.0, 448.0, c["codes"][1].shape))
    c["codes"][1] = e4m3_codes(values)
    c["scales"][1] = np.where(np.isnan(c["scales"][1]), np.nan, 2.0 ** power)
    want, tol = np.zeros((len(lens), heads, hd)), np.zeros((len(lens), heads, hd))
    for r, n in enumerate(lens):
        pages = c["table"][r, : -(-n // PAGE)]
        for a in range(kv):
            k, v = ((CODES[c["codes"][x][pages, a]] * c["scales"][x][pages, a][:, None, None]).reshape(-1, hd)[:n]
                    for x in range(2))
            for h in range(a * heads // kv, (a + 1) * heads // kv):
                want[r, h], tol[r, h] = attend(c["q"][r].reshape(heads, hd)[h], k, v, wk.BF16)
    near(run_decode(dev, c, max(lens), ws), want.reshape(len(lens), -1), tol.reshape(len(lens), -1))


@pytest.mark.gpu
def test_plan_with_the_largest_row_capacity(dev):
    """2^31 - 1 rows of room, which no step in 32 bits may leave."""
    cap = 2 ** 31 - 1
    ctx, add, table = np.array([70, 0]), np.array([2, 130]), np.array([[4, 3, -1, -1], [-1, -1, -1, -1]])
    want = ops.ref_plan(ctx, add, table, np.array([7, 8, 9]), 3, 140)
    b = [up(np.asarray(x, np.int32)) for x in (np.zeros(3), np.zeros(2), table, np.zeros(3), ctx, add, [7, 8, 9], [3])]
    starts, lens, tab, status, pctx, padd, pages, n_free = b
    seq, pos = alloc(4 * cap), alloc(4 * cap)
    wk.check(dev.wk_batch_plan(starts, lens, seq, pos, None, cap, tab, 4, status, pctx, padd, 2, pages, n_free, 3))
    for p, name in ((seq, "row_seq"), (pos, "row_pos")):
        assert np.array_equal(down(p, 140, np.int32), want[name])
        assert (down(p + 4 * (cap - 100000), 100000, np.int32) == -1).all()
    assert np.array_equal(down(tab, (2, 4), np.int32), want["table"])
    assert np.array_equal(down(status, 3, np.int32), want["status"])
    free(*b, seq, pos)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,extra", [(64, 0), (64, 1), (128, 0), (128, 1)])
@pytest.mark.parametrize("lens,room", [([30, 50, 20], 61), ([30, 50, 20], 30), ([400, 300], 550)])
def test_packed_prompts_with_less_room_than_rows(dev, lens, room, hd, extra):
    """Starts of a plan that go beyond the rows: the rows that there are come out as their sequence gives them."""
    c = ops.make_packed(lens, lens, 4, 2, hd, wk.F16, seed=9)
    cut = dict(c, q=c["q"][:room], k=c["k"][:room], v=c["v"][:room], qs=np.minimum(c["qs"], room), ks=np.minimum(c["ks"], room))
    want, tol = ops.ref_packed(cut)

    def laid(x):
        full = np.full((room, x.shape[1] + extra), np.nan)
        full[:, : x.shape[1]] = x
        return up(to_bits(full, wk.F16))
    q, k, v = (laid(cut[x]) for x in "qkv")
    starts, w = up(c["qs"].astype(np.int32)), 4 * hd
    out = up(np.full((room + 9) * w, 0x3555, np.uint16))
    wk.check(dev.wk_attention_packed(out, w, q, w + extra, k, 2 * hd + extra, v, 2 * hd + extra, starts, starts, len(lens),
                                     room, room, 4, 2, hd, wk.F16))
    got = down(out, (room + 9, w), np.uint16)
    free(q, k, v, starts, out)
    assert (got[room:] == 0x3555).all()
    ops.close(got[:room].view(np.float16).astype(np.float64), want, tol)


def bits(x, dt):
    return to_bits(x, dt).view(np.uint16)


@pytest.mark.gpu
@pytest.mark.parametrize("n,heads,kv,hd,dt", [(512, 8, 1, 128, wk.F16), (760, 16, 4, 64, wk.BF16), (512, 32, 8, 128, wk.BF16)])
def test_packed_prompt_too_short_for_a_cluster(dev, n, heads, kv, hd, dt):
    """A prompt whose keys would not repay sharing them: the very results that it has among many, where CTAs are few enough."""
    c = ops.make_packed([n] + [250] * 40, [n] + [250] * 40, heads, kv, hd, dt, seed=n)
    alone = dict(c, qs=c["qs"][:2], ks=c["ks"][:2], **{x: c[x][:n] for x in "qkv"})
    assert np.array_equal(bits(run_packed(dev, alone), dt), bits(run_packed(dev, c)[:n], dt))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [700, 2000])
@pytest.mark.parametrize("heads,kv,hd,dt", [(16, 8, 128, wk.F16), (16, 16, 64, wk.BF16)])
@pytest.mark.parametrize("others", [[0] * 63, [1] * 90, [5, 0, 40] * 20])
def test_packed_long_prompt_among_idle_and_short_sequences(dev, n, heads, kv, hd, dt, others):
    """Sequences without rows and short ones do not change how a long prompt is computed: its results are the very same."""
    lens = others[: len(others) // 2] + [n] + others[len(others) // 2:]
    c = ops.make_packed(lens, lens, heads, kv, hd, dt, seed=n)
    i = len(others) // 2
    at = slice(c["qs"][i], c["qs"][i + 1])
    # alone: beside three of its like, so that CTAs are not few
    like = dict(c, qs=np.arange(4) * n, ks=np.arange(4) * n, **{x: np.concatenate([c[x][at]] * 3) for x in "qkv"})
    got = run_packed(dev, c)
    assert np.array_equal(bits(got[at], dt), bits(run_packed(dev, like)[:n], dt))
    rest = np.ones(len(got), bool)
    rest[at] = False
    short = dict(c, qs=np.concatenate([c["qs"][: i + 1], c["qs"][i + 2:] - n]),
                 ks=np.concatenate([c["ks"][: i + 1], c["ks"][i + 2:] - n]), **{x: c[x][rest] for x in "qkv"})
    want, tol = ops.ref_packed(short)
    ops.close(got[rest], want, tol)


# The tcgen05 kernel where sequences are many, far apart or beside others that are not finite: lengths
# that send them to it.

@pytest.mark.gpu
@pytest.mark.parametrize("hd,dt,keys", [(64, wk.F16, 130), (128, wk.BF16, 60)])
def test_packed_many_sequences_behind_contexts_and_a_late_start(dev, hd, dt, keys):
    """More sequences than one pass over their lengths takes; the first starts behind rows of nobody."""
    rng = np.random.default_rng(5)
    ql = rng.integers(0, 4, 900)
    kl = ql + rng.integers(keys, keys + 9, 900)
    c = ops.make_packed([7, *ql], [9, *kl], 4, 2, hd, dt, seed=17)
    want, tol = ops.ref_packed(c)
    d = dict(c, qs=c["qs"][1:], ks=c["ks"][1:])
    got = run_packed(dev, d)
    assert (bits(got[:7], dt) == 0x3555).all()  # not written
    ops.close(got[7:], want[7:], tol[7:])
    assert np.array_equal(got[7:], run_packed(dev, d)[7:])


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("hd,dt", [(64, wk.F16), (128, wk.F16), (64, wk.BF16)])
def test_packed_longer_sequences_do_not_touch_each_other(dev, bad, hd, dt):
    c = ops.make_packed([70, 60, 90], [400, 360, 390], 4, 2, hd, dt, seed=6)
    want, tol = ops.ref_packed(c)
    d = dict(c, **{x: c[x].copy() for x in "qkv"})
    d["k"][c["ks"][1]:c["ks"][2]] = bad
    d["v"][c["ks"][1]:c["ks"][2]] = bad
    d["q"][c["qs"][1]:c["qs"][2]] = bad
    got = run_packed(dev, d)
    for i in (0, 2):
        at = slice(c["qs"][i], c["qs"][i + 1])
        ops.close(got[at], want[at], tol[at])
    assert not np.isfinite(got[c["qs"][1]:c["qs"][2]]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("hd,dt", [(64, wk.BF16), (128, wk.F16)])
@pytest.mark.parametrize("key", [137, 2580])
def test_packed_non_finite_values_in_a_cluster(dev, bad, hd, dt, key):
    """A NaN or an infinity in V where a cluster shares the keys: it reaches the queries that see its key, in its dimension."""
    c = ops.make_packed([40], [2600], 2, 1, hd, dt, seed=8)
    want, tol = ops.ref_packed(c)
    d = dict(c, v=c["v"].copy())
    d["v"][key, 3] = bad
    got = run_packed(dev, d)
    seen = np.zeros(want.shape, bool)
    seen[max(key - 2560, 0):, [3, hd + 3]] = True
    assert not np.isfinite(got[seen]).any()
    assert (np.abs(got - want) <= tol)[~seen].all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt,hd", [(wk.F16, 64), (wk.BF16, 128)])
def test_packed_long_context_with_rows_beyond_32_bits(dev, dt, hd):
    """Rows so far apart that the last ones lie more than 2^32 bytes behind the first, in K, V, the queries and the output."""
    c = ops.make_packed([40], [600], 2, 1, hd, dt, seed=3)
    q_rs, k_rs = 1 << 26, 1 << 22
    q, k, v, out = (alloc(2 * ((n - 1) * rs + w)) for n, rs, w in ((40, q_rs, 2 * hd), (600, k_rs, hd), (600, k_rs, hd),
                                                                   (40, q_rs, 2 * hd)))
    for p, x, rs in ((q, c["q"], q_rs), (k, c["k"], k_rs), (v, c["v"], k_rs)):
        rows = to_bits(x, dt)
        for r in range(len(x)):
            dev.cuda_to_device(p + 2 * r * rs, ops.as_p(np.ascontiguousarray(rows[r])), rows[r].nbytes)
    qs, ks = up(c["qs"].astype(np.int32)), up(c["ks"].astype(np.int32))
    wk.check(dev.wk_attention_packed(out, q_rs, q, q_rs, k, k_rs, v, k_rs, qs, ks, 1, 40, 600, 2, 1, hd, dt))
    got = ops.from_bits(np.stack([down(out + 2 * r * q_rs, 2 * hd, ops.RAW[dt]) for r in range(40)]), dt)
    free(q, k, v, out, qs, ks)
    want, tol = ops.ref_packed(c)
    ops.close(got, want, tol)


WITHOUT_TCGEN05 = r"""
import sys
sys.path.insert(0, sys.argv[1])
import numpy as np
import wukong_b200 as wk
from tests import test_serving_ops as ops
L = wk.lib()
L.cuda_init(0)
for case in (([300, 1, 70], [700, 1, 70], 4, 2, 128, wk.F16), ([40], [2600], 2, 1, 64, wk.BF16),
             ([50, 260], [50, 400], 130, 1, 64, wk.BF16), ([5] * 30 + [300], [5] * 30 + [300], 4, 2, 64, wk.F16)):
    c = ops.make_packed(*case, seed=5)
    want, tol = ops.ref_packed(c)
    ops.close(ops.run_packed(L, c), want, tol)
print("ok")
"""


@pytest.mark.gpu
def test_packed_without_the_tcgen05_kernel():
    """What serves where a compiler gave that kernel other registers than its split counts on."""
    env = dict(os.environ, WUKONG_TC_ATTN="0")
    r = subprocess.run([sys.executable, "-c", WITHOUT_TCGEN05, wk.ROOT], capture_output=True, text=True, env=env, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout + r.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv,hd,dt", [(8, 2, 64, wk.F16), (8, 1, 128, wk.BF16)])
@pytest.mark.parametrize("run,adds", [(3, [1, 1, 3, 90, 20, 1]), (0, [5, 64, 0, 130, 1, 63]), (6, [1, 2, 1, 1, 0, 1]),
                                      (2, [1, 0, 300, 0, 7, 1])])
def test_step_of_running_and_starting_sequences(dev, heads, kv, hd, dt, run, adds):
    """Running sequences first, over the cache; those that start behind them, over their own rows."""
    loop = ops.Loop(dev, 6, heads, kv, hd, dt, n_pages=40, max_pages=8, rows_cap=700, seed=run)
    if run:
        loop.inputs([70 + 9 * i if i < run else 0 for i in range(6)])
        loop.launch(prompts=True)
        loop.verify(prompts=True)
    loop.inputs(adds)
    d, n, w, ow = loop.d, loop.n, loop.w, heads * hd
    run_rows = sum(adds[:run])
    q, k, v = d["qkv"], d["qkv"] + 2 * ow, d["qkv"] + 2 * (heads + kv) * hd
    loop.put("out", np.full((loop.rows_cap, ow), 0x3555, np.uint16))
    wk.check(dev.wk_batch_plan(d["starts"], d["lens"], d["seq"], d["pos"], d["slot"], loop.rows_cap, d["table"],
                               loop.max_pages, d["status"], d["ctx"], d["add"], n, d["free"], d["n_free"], loop.n_pages))
    wk.check(dev.wk_kv8_store(d["k"], d["v"], d["ks"], d["vs"], loop.n_pages, k, w, v, w, d["starts"], d["ctx"], n,
                              loop.rows_cap, d["table"], loop.max_pages, kv, hd, dt))
    wk.check(dev.wk_kv8_attention(d["out"], ow, q, w, d["k"], d["v"], d["ks"], d["vs"], loop.n_pages, d["table"], n,
                                  loop.max_pages, d["seq"], d["pos"], run_rows, loop.max_pages * PAGE, heads, kv, hd, dt,
                                  d["ws"], loop.ws_bytes))
    wk.check(dev.wk_attention_packed(d["out"], ow, q, w, k, w, v, w, d["starts"] + 4 * run, d["starts"] + 4 * run, n - run,
                                     loop.rows_cap, loop.rows_cap, heads, kv, hd, dt))
    out = down(d["out"], (loop.rows_cap, ow), ops.RAW[dt])
    p = ops.ref_plan(loop.ctx, loop.add, loop.table, np.roll(loop.free_list, -loop.taken), loop.n_pages - loop.taken,
                     loop.rows_cap)
    rows = len(loop.x)
    for i in range(2):
        x = loop.x[:, ow + i * kv * hd:ow + (i + 1) * kv * hd].reshape(rows, kv, hd)
        loop.codes[i], loop.scales[i] = ops.ref_store(loop.codes[i], loop.scales[i], x, p["starts"], loop.ctx, p["table"],
                                                      loop.n_pages)
    c = dict(heads=heads, kv=kv, hd=hd, dt=dt, q=loop.x[:, :ow])
    over_cache = ops.ref_decode(dict(c, pos=p["row_pos"][:rows], seq=p["row_seq"][:rows], table=p["table"],
                                     codes=loop.codes, scales=loop.scales, n_pages=loop.n_pages))
    over_rows = ops.ref_packed(dict(c, k=loop.x[:, ow:ow + kv * hd], v=loop.x[:, ow + kv * hd:], qs=p["starts"], ks=p["starts"]))
    want, tol = (np.concatenate([a[:run_rows], b[run_rows:]]) for a, b in zip(over_cache, over_rows))
    ops.close(ops.from_bits(out[:rows], dt), want, tol)
    assert (out[rows:].view(np.uint16) == 0x3555).all()
    loop.end()


CAPTURED_FIRST = r"""
import sys
sys.path.insert(0, sys.argv[1])
import numpy as np
import torch
import wukong_b200 as wk
from tests import test_serving_ops as ops
L = wk.lib()
L.cuda_init(0)
stream = torch.cuda.ExternalStream(L.wk_stream())
loop = ops.Loop(L, 4, 8, 2, 128, wk.F16, 80, 16, 900, seed=2)
loop.inputs([20, 700, 1, 64])
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=stream):
    loop.launch(prompts=True)
with torch.cuda.stream(stream):
    g.replay()
loop.verify(prompts=True)
loop.inputs([1, 1, 0, 5])
g2 = torch.cuda.CUDAGraph()
with torch.cuda.graph(g2, stream=stream):
    loop.launch(prompts=False)
with torch.cuda.stream(stream):
    g2.replay()
loop.verify(prompts=False)
torch.cuda.synchronize()
print("ok")
"""


@pytest.mark.gpu
def test_first_calls_of_a_process_captured():
    """Kernels that are set up within a capture."""
    pytest.importorskip("torch")
    r = subprocess.run([sys.executable, "-c", CAPTURED_FIRST, wk.ROOT], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.endswith("ok\n"), r.stdout + r.stderr
