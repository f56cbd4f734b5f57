"""The paged K/V cache on the GPU against numpy in 64 bits (kv_model.py).

Attention tolerance. Everything is held in fp32 or in three bf16 terms (2^-24
relative), so a score of magnitude S is off by a few 2^-24 S (sums of up to
256 products grow that by about sqrt(256) / 2 = 8), its weight by as much
relatively, and sums over entries average these out. The scores below stay
under 16 in magnitude: 8 * 16 * 2^-24 = 8e-6 for one weight at the worst; with
entries' errors independent the relative L2 error of an output is bounded by
the rms one, about a quarter: 2e-6. lse: absolute error of the scores plus the
rounding of its own value (2^-24 * 32): 4e-6 + 2e-6.
Running sums: fp32 sums of at most 20 heads' weights: 20 * 2^-24 and the
weights' own 2e-6.
"""
import numpy as np
import pytest

import kv_model as km
import pywelvet as pw
from test_gpu_dense import rel_l2

pytestmark = pytest.mark.gpu

OUT_TOL, LSE_TOL, SUM_TOL = 2e-6, 6e-6, 3.2e-6


@pytest.fixture(scope="module")
def hip(gpu):
    return pw.Hip()


def rows(rng, n, r, kv, hd):
    return [rng.standard_normal((n, r, kv, hd)).astype(np.float32) for _ in range(2)]


def query(rng, c):
    return (2 * rng.standard_normal((c.nseq, c.heads, c.hd))).astype(np.float32)


def filled(hip, oracle, lens, dtype, heads, kv, hd, page=16, seed=1, room=1, **kw):
    """A cache whose sequences hold `lens` entries, all other memory NaN."""
    max_pages = max(1, -(-(max(lens) + room) // page))
    kw.setdefault("poison", True)
    c = km.Cache(hip, dtype, heads, kv, hd, len(lens), max_pages, page, seed=seed, **kw)
    if max(lens):
        c.append(*rows(c.rng, len(lens), max(lens), kv, hd), oracle, counts=list(lens))
    return c


def check(c, q, **kw):
    track = c.weight.copy() if c.d_weight else None
    sums = np.zeros(c.weight.shape)
    out, lse = c.attend(q, **kw)
    kw.pop("stream", None)
    want, want_lse = c.want(q, track=sums, **kw)
    err = rel_l2(out, want) if np.any(want) else float(np.abs(out).max())
    print(f"attend {km.NAMES[c.dtype]} heads {c.heads}/{c.kv} hd {c.hd} lens {c.lens.tolist()[:6]}: {err:.2e}")
    assert err <= OUT_TOL
    seen = np.isfinite(want_lse)
    assert np.array_equal(seen, np.isfinite(lse)) and np.all(lse[~seen] == -np.inf)
    assert np.all(np.abs(lse[seen] - want_lse[seen]) <= LSE_TOL)
    assert np.all(out[~seen] == 0)
    if c.d_weight:
        got = c.device_weight()
        # entries that the call does not see keep their sums to the bit
        idle = sums == 0
        assert np.array_equal(got[idle], track[idle])
        assert np.all(np.abs(got - (track + sums)) <= SUM_TOL * np.maximum(1, track + sums))
        c.weight = got.copy()
    return out


# ---------------------------------------------------------------- append ---
@pytest.mark.parametrize("dtype,hd,page,kv", [
    (km.F32, 1, 16, 1), (km.F32, 33, 48, 3), (km.F32, 256, 16, 2), (km.BF16, 7, 16, 2),
    (km.BF16, 64, 64, 4), (km.BF16, 80, 16, 1), (km.BF16, 255, 32, 1), (km.E4M3, 1, 16, 2),
    (km.E4M3, 33, 16, 1), (km.E4M3, 64, 16, 5), (km.E4M3, 128, 80, 8), (km.E4M3, 250, 16, 1),
])
def test_append_writes_its_entries_and_nothing_else(hip, oracle, dtype, hd, page, kv):
    c = km.Cache(hip, dtype, kv, kv, hd, 3, 3, page, seed=hd)
    c.append(*rows(c.rng, 3, 20, kv, hd), oracle, counts=[20, 0, 7])
    before = c.pool()
    lens = c.lens.copy()
    c.append(*rows(c.rng, 3, page + 3, kv, hd), oracle, counts=[page + 3, 1, -2])
    after = c.pool()
    touched = np.zeros((c.num_pages, page), bool)
    for b in range(3):
        for e in range(lens[b], c.lens[b]):
            touched[c.table[b, e // page], e % page] = True
    keep = ~np.repeat(touched[:, None], kv, 1)
    for x, y in zip(before, after):
        assert np.array_equal(x[keep], y[keep])
    if c.pitch > hd:  # the elements that fill a row up are zero
        assert not after[0][..., hd * c.elem:].any() and not after[1][..., hd * c.elem:].any()
    # read back: the stored values to the bit, zeros behind the counts
    n = int(c.lens.max())
    k, v = (hip.upload(np.full((3, n, kv, hd), 5, np.float32)) for _ in range(2))
    c.c.read(c.seqs, n, k, v, None, c.d_lens)
    for got, want in ((k, c.k), (v, c.v)):
        got = c.down(got, (3, n, kv, hd))
        assert np.array_equal(got, want.transpose(0, 2, 1, 3)[:, :n].astype(np.float32))
    assert np.array_equal(c.down(c.d_pos, c.pos.shape, np.int32), c.pos)
    assert np.array_equal(c.device_weight(), c.weight)
    assert np.array_equal(c.down(c.d_lens, (3,), np.int32), c.lens)
    hip.free(k), hip.free(v)
    c.close()


def test_append_strides_unaligned_rows_and_values(hip, oracle):
    kv, hd = 2, 24
    for dtype in (km.F32, km.BF16, km.E4M3):
        c = km.Cache(hip, dtype, kv, kv, hd, 2, 1)
        k, v = rows(c.rng, 2, 5, kv, hd)
        k[0, 0, 0, :4] = [3e38, -3e38, 1e-39, -0.0]     # past bf16's largest: inf
        k[0, 1, 0] = 0                                   # a row of zeros
        k[0, 2, 0] = np.ldexp(1.0, -110) * np.sign(k[0, 2, 0])
        k[1, 0, 1, 3], v[1, 0, 0, 5] = np.inf, np.nan
        k[1, 1, 0, 0] = -np.inf
        wide = np.full((10, 2 * kv * hd + 7), 9, np.float32)  # K, V and more in one row
        wide[:, 1:1 + kv * hd] = k.reshape(10, -1)
        wide[:, 1 + kv * hd:1 + 2 * kv * hd] = v.reshape(10, -1)
        d = hip.upload(wide)
        c.c.append(c.seqs, 5, d + 4, d + 4 + 4 * kv * hd, None, wide.shape[1], wide.shape[1])
        b = c.c.buffers()
        dk, dv = (hip.upload(np.zeros((2, 5, kv, hd), np.float32)) for _ in range(2))
        c.c.read(c.seqs, 5, dk, dv)
        for got, x in ((c.down(dk, k.shape), k), (c.down(dv, v.shape), v)):
            if dtype == km.E4M3:  # one element that is not finite takes its row with it
                bad = ~np.isfinite(x).all(-1)
                assert np.isnan(got[bad]).all()
                want = km.stored(np.where(bad[..., None], 0, x), dtype, oracle)
                assert np.array_equal(got[~bad], want[~bad])
            else:
                with np.errstate(over="ignore", invalid="ignore"):
                    want = km.stored(x, dtype, oracle)
                bad = np.isnan(x)
                assert np.isnan(got[bad]).all() and np.array_equal(got[~bad], want[~bad])
        assert b.pitch >= hd
        for p in (d, dk, dv):
            hip.free(p)
        c.close()


def test_append_past_the_capacity_and_into_holes(hip, oracle):
    for dtype in (km.F32, km.BF16, km.E4M3):
        table = np.array([[0, -1, 2], [5, 2 ** 31 - 1, -2 ** 31], [3, 4, 6]], np.int32)
        c = km.Cache(hip, dtype, 2, 2, 32, 3, 3, table=table, num_pages=6)
        c.append(*rows(c.rng, 3, 40, 2, 32), oracle)
        c.append(*rows(c.rng, 3, 30, 2, 32), oracle)      # 22 of them past the capacity of 48
        assert c.lens.tolist() == [48] * 3
        k, v = (hip.upload(np.full((3, 48, 2, 32), 5, np.float32)) for _ in range(2))
        c.c.read(c.seqs, 48, k, v)
        ok = np.array([[c.valid(b, e) for e in range(48)] for b in range(3)])
        for got, want in ((k, c.k), (v, c.v)):
            got, want = c.down(got, (3, 48, 2, 32)), want.transpose(0, 2, 1, 3)
            assert np.array_equal(got[ok], want[ok].astype(np.float32)) and not got[~ok].any()
        # page 1 belongs to nobody
        assert not any(x[1].any() for x in c.pool())
        check(c, query(c.rng, c))
        hip.free(k), hip.free(v)
        c.close()


# ---------------------------------------------------------------- attend ---
LENS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 130, 400]


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
@pytest.mark.parametrize("heads,kv,hd,page", [
    (1, 1, 64, 16), (4, 4, 32, 16), (6, 2, 64, 32), (12, 4, 64, 48), (8, 1, 128, 16),
    (20, 1, 80, 16), (3, 3, 33, 16), (5, 5, 1, 16), (2, 1, 256, 16), (40, 2, 96, 64), (7, 7, 17, 16),
    (16, 1, 128, 32), (17, 1, 128, 32), (6, 3, 160, 16), (4, 1, 250, 16), (66, 2, 8, 16), (3, 1, 200, 16),
])
def test_attend_over_edge_lengths(hip, oracle, dtype, heads, kv, hd, page):
    c = filled(hip, oracle, LENS, dtype, heads, kv, hd, page, seed=heads * 1000 + hd)
    check(c, query(c.rng, c))
    c.close()


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
@pytest.mark.parametrize("lens,heads,kv,hd", [
    ([9001], 8, 2, 128), ([5000, 1, 3000], 4, 4, 64), ([2047] * 3, 3, 1, 72), ([4097, 0], 2, 2, 256),
    ([3333], 32, 1, 192),
])
def test_attend_over_long_caches(hip, oracle, dtype, lens, heads, kv, hd):
    c = filled(hip, oracle, lens, dtype, heads, kv, hd, 32, seed=sum(lens))
    q = query(c.rng, c)
    first = check(c, q)
    # the same call gives the same bits
    again, _ = c.attend(q)
    assert np.array_equal(first, again)
    c.close()


@pytest.mark.parametrize("nseq,most,heads,kv,hd,dtype", [
    (70, 700, 2, 1, 64, km.E4M3), (130, 300, 20, 1, 32, km.BF16), (64, 900, 4, 4, 16, km.F32),
    (65, 2000, 1, 1, 64, km.BF16), (3, 4000, 34, 2, 64, km.BF16),
    # (workgroups of one wave: 2048 rows of heads and more)
    (300, 70, 8, 8, 64, km.BF16), (520, 40, 4, 4, 20, km.E4M3), (200, 400, 16, 16, 32, km.F32),
    # (the same with several query heads to a K/V head, up to all columns of a tile)
    (300, 40, 12, 4, 64, km.BF16), (330, 35, 20, 1, 128, km.BF16), (110, 50, 64, 4, 256, km.BF16),
    (200, 60, 16, 4, 80, km.E4M3), (450, 33, 5, 1, 250, km.E4M3), (210, 45, 48, 3, 128, km.F32),
])
def test_attend_over_many_unequal_sequences(hip, oracle, nseq, most, heads, kv, hd, dtype):
    """Sequences of none to many parts in one call, joined by kind."""
    rng = np.random.default_rng(nseq)
    lens = (most * rng.random(nseq) ** 3).astype(int)
    lens[rng.random(nseq) < 0.2] = 0
    lens[nseq // 2] = most
    c = filled(hip, oracle, lens.tolist(), dtype, heads, kv, hd, 16, seed=nseq)
    check(c, query(c.rng, c))
    check(c, query(c.rng, c), window=257)
    c.close()


@pytest.mark.parametrize("nseq,most,heads,kv,hd,dtype", [
    (24, 2300, 16, 16, 64, km.BF16), (40, 1500, 32, 8, 128, km.E4M3), (33, 1200, 32, 16, 40, km.F32),
    (12, 2100, 20, 10, 250, km.BF16), (100, 2050, 16, 8, 72, km.E4M3), (70, 2048, 16, 16, 128, km.F32),
])
@pytest.mark.parametrize("kind", ["plain", "track", "window"])
def test_attend_runs_over_sequences(hip, oracle, nseq, most, heads, kv, hd, dtype, kind):
    """Workgroups that take several sequences: empty ones between long ones, one
    entry, whole tiles; with running sums, and windows over given positions."""
    rng = np.random.default_rng(nseq + hd)
    lens = rng.integers(most // 2, most + 1, nseq)
    lens[rng.random(nseq) < 0.2] = 0
    lens[rng.random(nseq) < 0.1] = 1
    lens[rng.random(nseq) < 0.1] = most // 64 * 32
    lens[nseq // 3] = most
    c = filled(hip, oracle, lens.tolist(), dtype, heads, kv, hd, 32, seed=nseq,
               track=kind == "track", positions=kind != "plain")
    q = query(c.rng, c)
    if kind == "window":
        check(c, q, window=most // 2, alibi=True)
    else:
        first = check(c, q)
        again, _ = c.attend(q)
        assert np.array_equal(first, again)
    c.close()


@pytest.mark.parametrize("window,alibi,tail,scale", [
    (1, False, 0, 0.0), (17, False, 1, 0.0), (64, True, 0, 0.0), (1000, True, 1, 0.05),
    (0, True, 0, 0.0), (0, False, 1, 0.3), (2 ** 31 - 1, False, 0, 0.0), (300, False, 5, 0.0),
])
@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
@pytest.mark.parametrize("positions", [True, False])
def test_attend_windows_alibi_tails(hip, oracle, dtype, window, alibi, tail, scale, positions):
    lens = [3, 0, 16, 33, 100, 1200]
    c = filled(hip, oracle, lens, dtype, 6, 2, 64, 16, seed=window % 97 + tail, positions=positions, room=8)
    if tail:
        k, v = rows(c.rng, len(lens), tail, 2, 64)
        dk, dv = c.up(k), c.up(v)
        c.c.append(c.seqs, tail, dk, dv)
        c.note_append(k, v, oracle)
    check(c, query(c.rng, c), window=window, alibi=alibi, tail=tail, scale=scale)
    c.close()


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_attend_positions_after_eviction(hip, oracle, dtype):
    """Entries in any order of positions, heads with different tokens, windows
    that leave some heads nothing."""
    c = filled(hip, oracle, [40, 90, 17], dtype, 4, 2, 64, 16)
    for b in range(3):
        for h in range(2):
            n = c.lens[b]
            c.pos[b, h, :n] = c.rng.permutation(5 * n)[:n] + (200 if h and b == 2 else 0)
    c.next = np.array([300, 500, 300], np.int32)
    c.put(c.d_pos, c.pos), c.put(c.d_next, c.next)
    for window, alibi in ((0, True), (150, False), (260, True), (3, False)):
        check(c, query(c.rng, c), window=window, alibi=alibi)
    c.close()


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_attend_holes_and_nothing_left(hip, oracle, dtype):
    table = np.array([[-1, 1, 9], [9, -5, 2 ** 31 - 1], [4, 9, 5], [6, 7, 8]], np.int32)
    c = km.Cache(hip, dtype, 4, 2, 64, 4, 3, table=table, num_pages=9, poison=True)
    c.append(*rows(c.rng, 4, 41, 2, 64), oracle)
    check(c, query(c.rng, c))          # sequence 1 has no page in the pool
    # a window that lies behind every position
    c.next = c.next + 1000
    c.put(c.d_next, c.next)
    check(c, query(c.rng, c), window=500)
    c.close()


def test_attend_shared_pages_and_odd_lengths_given(hip, oracle):
    """Two sequences over the same prefix pages; lengths outside [0, capacity]."""
    table = np.array([[0, 1, 2], [0, 1, 3], [4, 5, 6], [7, 8, 9]], np.int32)
    c = km.Cache(hip, km.BF16, 4, 2, 64, 4, 3, table=table, num_pages=10, poison=True)
    k, v = rows(c.rng, 4, 48, 2, 64)
    k[1, :32], v[1, :32] = k[0, :32], v[0, :32]
    c.append(k, v, oracle)
    real = c.lens.copy()
    c.put(c.d_lens, np.array([48, 40, -9, 2 ** 31 - 1], np.int32))
    c.lens = np.array([48, 40, 0, 48], np.int32)
    check(c, query(c.rng, c))
    assert real.tolist() == [48] * 4
    c.close()


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_attend_exact_weights(hip, oracle, dtype):
    """Queries of zero: every weight is 1/n, and values of small integers (in
    E4M3 codes: +-240 s) sum without rounding: only the division rounds."""
    n = 256
    c = km.Cache(hip, dtype, 2, 1, 64, 1, 16)
    k, _ = rows(c.rng, 1, n, 1, 64)
    v = c.rng.choice([-1.0, 1.0], (1, n, 1, 64)).astype(np.float32) * 240
    c.append(k, v, oracle)
    out, lse = c.attend(np.zeros((1, 2, 64), np.float32))
    assert np.array_equal(out[0, 0], v[0, :, 0].mean(0)) and np.array_equal(out[0, 0], out[0, 1])
    assert np.all(np.abs(lse - np.log(n)) <= 4 * 2.0 ** -24 * 8)
    assert np.all(c.device_weight()[0, 0, :n] == 2.0 / n)
    c.close()


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_attend_large_scores_and_small_values(hip, oracle, dtype):
    """Scores of hundreds, rising along the cache (the running maximum moves at
    every tile) and falling; values of 2^-90 and of 2^90."""
    n = 700
    for sign in (1, -1):
        for size in (2.0 ** -90, 2.0 ** 90):
            c = km.Cache(hip, dtype, 1, 1, 64, 1, 48, track=False)
            k, v = rows(c.rng, 1, n, 1, 64)
            k *= 0.125
            k[0, :, 0, 0] = np.linspace(-4, 4, n, dtype=np.float32) * sign
            v = (v * np.float32(size)).astype(np.float32)
            c.append(k, v, oracle)
            q = np.zeros((1, 1, 64), np.float32)
            q[0, 0, :8] = 1
            q[0, 0, 0] = 800
            out, lse = c.attend(q)
            want, want_lse = c.want(q)
            # scores up to 400: rounded to 2^-16 (and their product to as much)
            assert rel_l2(out, want) <= 400 * 2.0 ** -23
            assert abs(lse[0, 0] - want_lse[0, 0]) <= 400 * 2.0 ** -23
            c.close()


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_attend_values_that_are_not_finite(hip, oracle, dtype):
    """NaN in a seen entry reaches its K/V head's outputs, in others nothing."""
    c = filled(hip, oracle, [50, 50], dtype, 4, 2, 64, 16, track=False)
    k, v = rows(c.rng, 2, 1, 2, 64)
    v[0, 0, 0, 3] = np.nan
    dk, dv = c.up(k), c.up(v)
    c.c.append(c.seqs, 1, dk, dv)
    q = query(c.rng, c)
    good = check(c, q)                                    # not counted: no effect
    out, _ = c.attend(q, tail=1)
    assert np.isnan(out[0, :2, 3]).all()
    assert np.isfinite(out[0, 2:]).all() and np.isfinite(out[1]).all()
    if dtype != km.E4M3:
        assert np.isfinite(np.delete(out[0], 3, axis=-1)).all()
    # out of the window: no effect again
    c.next += 1
    c.put(c.d_next, c.next)
    k2, v2 = rows(c.rng, 2, 1, 2, 64)
    c.put(c.d_lens, c.lens + 1)
    dk, dv = c.up(k2), c.up(v2)
    c.c.append(c.seqs, 1, dk, dv)
    c.put(c.d_lens, c.lens + 2)
    c.put(c.d_next, c.next + 1)
    out, _ = c.attend(q, window=1)
    # one entry is seen: its value, after at most five roundings of half a step
    # (2^-24): weight times scale, the two sums over that product's terms, the
    # reciprocal of the weights' sum and the product with it
    one = np.repeat(km.stored(v2, dtype, oracle)[:, 0], 2, 1).reshape(out.shape)
    assert np.all(np.abs(out - one) <= 5 * 2.0 ** -24 * np.abs(one))
    assert np.isfinite(good).all()
    q[1, 3, 5] = np.nan
    out, lse = c.attend(q, window=1)
    assert np.isnan(out[1, 3]).all() and np.isnan(lse[1, 3])
    assert np.isfinite(np.delete(out.reshape(8, 64), 7, 0)).all()
    c.close()


def test_attend_strides_and_neighbours(hip, oracle):
    c = filled(hip, oracle, [70, 5, 33], km.BF16, 6, 2, 40, 16, track=False)
    q = query(c.rng, c)
    w = 6 * 40
    qs, os_ = w + 3, w + 5
    qb = np.full((3, qs), np.nan, np.float32)
    qb[:, :w] = q.reshape(3, w)
    dq = hip.upload(np.concatenate([[np.float32(0)], qb.ravel()]).astype(np.float32))
    out = hip.upload(np.full((3, os_), 777, np.float32))
    c.c.attend(c.seqs, dq + 4, out, q_stride=qs, out_stride=os_)
    got = c.down(out, (3, os_))
    want, _ = c.want(q)
    assert rel_l2(got[:, :w].reshape(want.shape), want) <= OUT_TOL
    assert np.all(got[:, w:] == 777)
    hip.free(dq), hip.free(out)
    c.close()


def test_fewer_sequences_than_mounted(hip, oracle):
    """Rows behind the call's last sequence stay as they were."""
    c = filled(hip, oracle, [40, 20, 30], km.E4M3, 4, 2, 64, 16)
    weight = c.device_weight()
    c.seqs.nseq = 2
    q = query(c.rng, c)
    out, lse = c.attend(q)
    want, _ = c.want(q)
    assert rel_l2(out[:2], want[:2]) <= OUT_TOL
    assert np.all(out[2] == 777) and np.all(lse[2] == 777)
    assert np.array_equal(c.device_weight()[2], weight[2])
    c.seqs.nseq = 0
    c.attend(q)
    c.close()


def test_rows_past_4_gib(hip, oracle):
    """Pages at the far end of a pool of 5 GiB each of K and V."""
    pages = 5 * 2 ** 30 // (16 * 8 * 128 * 4)
    table = np.array([[pages - 1, 0], [pages - 2, pages // 2]], np.int32)
    c = km.Cache(hip, km.F32, 8, 8, 128, 2, 2, table=table, num_pages=pages)
    c.append(*rows(c.rng, 2, 30, 8, 128), oracle, counts=[30, 27])
    check(c, query(c.rng, c))
    src = np.full((2, 8, 16), -1, np.int32)
    src[:, :, :3] = [0, 20, 17]
    c.c.compact(c.seqs, 16, c.up(src))
    for x in (c.k, c.v, c.weight, c.pos):
        x[:, :, [1, 2]] = x[:, :, [20, 17]]
    c.lens = np.array([3, 3], np.int32)
    c.put(c.d_lens, c.lens)
    check(c, query(c.rng, c))
    c.close()


# ---------------------------------------------------------------- evict ----
def weights(rng, shape, kind):
    w = np.exp(2 * rng.standard_normal(shape)).astype(np.float32)
    if kind == "ties":
        w = rng.integers(0, 4, shape).astype(np.float32)
    elif kind == "same":
        w[:] = 0.25
    elif kind == "odd":
        flat = w.reshape(-1)
        flat[rng.permutation(flat.size)[:flat.size // 3]] = np.nan
        flat[rng.permutation(flat.size)[:flat.size // 9]] = np.inf
        flat[rng.permutation(flat.size)[:flat.size // 9]] = -np.inf
        flat[rng.permutation(flat.size)[:flat.size // 9]] = -0.0
        flat[rng.permutation(flat.size)[:flat.size // 9]] = 1e-42
    return w


@pytest.mark.parametrize("kind", ["plain", "ties", "same", "odd"])
@pytest.mark.parametrize("lens,budget,sinks,recent,positions", [
    ([1, 2, 0, 17], 1, 0, 0, False), ([33, 32, 31, 100], 32, 4, 16, False),
    ([1024, 1025, 1026, 2500], 1024, 4, 200, True), ([2100, 3000, 1, 700], 2100, 0, 2100, False),
    ([2100, 3000, 1, 700], 5, 5, 0, True), ([5000, 4999, 64, 65], 64, 0, 0, True),
    ([4096, 4000, 2049, 2047], 2048, 1000, 1000, True), ([16384, 9000], 9000, 4, 100, False),
    # (one workgroup's most entries; several segments, their edges, long and short rows together)
    ([32768, 20001], 16384, 4, 1000, True), ([32785, 32768, 500, 40000, 1], 1, 0, 1, False),
    # (many rows: a workgroup each up to 32768 entries)
    ([20000, 16385, 1, 0, 32768, 32767] + [300] * 27, 250, 4, 30, True),
    ([70001, 16384, 16385, 49152], 16384, 4, 1000, True), ([70001, 60000, 34000], 33000, 40, 20000, False),
])
def test_choose(hip, lens, budget, sinks, recent, positions, kind):
    page = 16
    c = km.Cache(hip, km.BF16, 3, 3, 8, len(lens), -(-max(max(lens), budget) // page), page,
                 positions=positions, seed=budget)
    c.lens = np.array(lens, np.int32)
    c.weight = weights(c.rng, c.weight.shape, kind)
    c.next = c.lens * 3 if positions else c.lens.copy()
    for b, n in enumerate(lens):
        for h in range(3):
            c.pos[b, h, :n] = c.rng.permutation(3 * n)[:n] if positions else np.arange(n)
    c.put(c.d_lens, c.lens), c.put(c.d_weight, c.weight), c.put(c.d_next, c.next)
    if positions:
        c.put(c.d_pos, c.pos)
    src = c.up(np.full((len(lens) + 1, 3, budget), 99, np.int32))
    for _ in range(2):  # (the second call finds the scratch as it was)
        c.c.choose(c.seqs, budget, sinks, recent, src)
    got = c.down(src, (len(lens) + 1, 3, budget), np.int32)
    for b, n in enumerate(lens):
        for h in range(3):
            want = km.choose(c.weight[b, h, :n], c.pos[b, h, :n], c.next[b], budget, sinks, recent)
            assert np.array_equal(got[b, h], want), (b, h)
    assert np.all(got[-1] == 99)
    assert np.array_equal(c.device_weight().view(np.uint32), c.weight.view(np.uint32))
    c.close()


def evict_model(c, src, budget):
    for b in range(c.nseq):
        for h in range(c.kv):
            for j, e in enumerate(src[b, h]):
                if budget <= e < c.cap:
                    for x in (c.k, c.v, c.pos, c.weight):
                        x[b, h, j] = x[b, h, e]
    c.lens = np.minimum(c.lens, budget).astype(np.int32)


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
@pytest.mark.parametrize("hd,page,budget", [(64, 16, 40), (33, 48, 16), (256, 16, 70), (1, 32, 31)])
def test_evict_moves_what_was_chosen(hip, oracle, dtype, hd, page, budget):
    lens = [100, budget + 1, budget, 3, 0]
    c = filled(hip, oracle, lens, dtype, 4, 2, hd, page)
    for _ in range(2):
        check(c, query(c.rng, c))
    src = c.up(np.zeros((5, 2, budget), np.int32))
    c.c.choose(c.seqs, budget, 2, 5, src)
    chosen = c.down(src, (5, 2, budget), np.int32)
    for b, n in enumerate(lens):
        for h in range(2):
            assert np.array_equal(chosen[b, h], km.choose(c.weight[b, h, :n], c.pos[b, h, :n],
                                                          c.next[b], budget, 2, 5))
    before = c.pool()
    for _ in range(2):  # the second time changes nothing
        c.c.compact(c.seqs, budget, src)
    c.c.advance(c.nseq, c.d_lens, cap=budget)
    evict_model(c, chosen, budget)
    assert np.array_equal(c.down(c.d_lens, (5,), np.int32), c.lens)
    got_w, got_p = c.device_weight(), c.down(c.d_pos, c.pos.shape, np.int32)
    assert np.array_equal(got_w, c.weight) and np.array_equal(got_p, c.pos)
    # rows that no slot below the budget names keep their bits
    moved = np.zeros((c.num_pages, 2, page), bool)
    for b in range(5):
        for h in range(2):
            for j in np.flatnonzero(chosen[b, h] >= budget):
                moved[c.table[b, j // page], h, j % page] = True
    for x, y in zip(before, c.pool()):
        assert np.array_equal(x[~moved], y[~moved])
    check(c, query(c.rng, c), alibi=True)
    c.close()


def test_compact_with_holes_and_entries_outside(hip, oracle):
    table = np.array([[0, 1, -1, 2], [3, 99, 4, 5]], np.int32)
    c = km.Cache(hip, km.BF16, 2, 2, 64, 2, 4, table=table, num_pages=6)
    c.append(*rows(c.rng, 2, 64, 2, 64), oracle)
    before = c.pool()
    src = np.tile(np.arange(32, dtype=np.int32), (2, 2, 1))
    src[0, :, 3], src[0, :, 4], src[0, :, 5] = 40, 64, 2 ** 31 - 1   # a hole, past the capacity
    src[1, :, 17], src[1, :, 18] = 50, -2 ** 31                       # into a hole
    src[1, 0, 2] = 63
    c.c.compact(c.seqs, 32, c.up(src))
    after = c.pool()
    for x, y in zip(before, after):
        x[3, 0, 2] = x[5, 0, 15]
        assert np.array_equal(x, y)
    c.close()


# ---------------------------------------------------------------- loops ----
@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_decode_loop_with_eviction(hip, oracle, dtype):
    """Append, attend and advance step by step; at 48 entries down to 32."""
    lens = [20, 3, 31]
    c = filled(hip, oracle, lens, dtype, 6, 3, 64, 16, room=33)
    src = c.up(np.zeros((3, 3, 32), np.int32))
    for step in range(40):
        k, v = rows(c.rng, 3, 1, 3, 64)
        dk, dv = c.up(k), c.up(v)
        c.c.append(c.seqs, 1, dk, dv)
        c.note_append(k, v, oracle)
        check(c, query(c.rng, c), tail=1, window=90 if step % 3 else 0, alibi=step % 2 == 1)
        c.c.advance(3, c.d_lens, c.d_next, add=1)
        c.count(1)
        if c.lens.max() >= 48:
            c.c.choose(c.seqs, 32, 2, 8, src)
            c.c.compact(c.seqs, 32, src)
            c.c.advance(3, c.d_lens, cap=32)
            evict_model(c, c.down(src, (3, 3, 32), np.int32), 32)
            assert np.array_equal(c.down(c.d_pos, c.pos.shape, np.int32)[:, :, :32], c.pos[:, :, :32])
        assert np.array_equal(c.down(c.d_next, (3,), np.int32), c.next)
    c.close()


def test_captured_decode_step(hip, oracle):
    """One step as a graph: append, attend, advance, evict, every replay
    against the numpy model, with eager calls of the same session between."""
    c = filled(hip, oracle, [10, 29], km.BF16, 4, 2, 64, 16, room=40)
    stream = hip.stream()
    k, v = (hip.malloc(4 * 2 * 2 * 64) for _ in range(2))
    q, out = hip.malloc(4 * 2 * 4 * 64), hip.malloc(4 * 2 * 4 * 64)
    lse, src = hip.malloc(4 * 2 * 4), hip.malloc(4 * 2 * 2 * 32)

    def step():
        c.c.append(c.seqs, 1, k, v, stream=stream)
        c.c.attend(c.seqs, q, out, tail=1, alibi=True, lse=lse, stream=stream)
        c.c.advance(2, c.d_lens, c.d_next, add=1, stream=stream)
        c.c.choose(c.seqs, 32, 2, 8, src, stream=stream)
        c.c.compact(c.seqs, 32, src, stream=stream)
        c.c.advance(2, c.d_lens, cap=32, stream=stream)

    graph = hip.capture(stream, step)
    for i in range(12):
        nk, nv = rows(c.rng, 2, 1, 2, 64)
        nq = query(c.rng, c)
        for p, x in ((k, nk), (v, nv), (q, nq)):
            c.put(p, x)
        hip.launch(graph, stream)
        hip.stream_sync(stream)
        c.note_append(nk, nv, oracle)
        sums = np.zeros(c.weight.shape)
        want, want_lse = c.want(nq, tail=1, alibi=True, track=sums)
        assert rel_l2(c.down(out, want.shape), want) <= OUT_TOL, i
        assert np.all(np.abs(c.down(lse, want_lse.shape) - want_lse) <= LSE_TOL)
        c.weight = (c.weight + sums).astype(np.float32)
        c.count(1)
        chosen = c.down(src, (2, 2, 32), np.int32)
        evict_model(c, chosen, 32)
        got = c.device_weight()
        for b in range(2):
            n = c.lens[b]
            assert np.all(np.abs(got[b, :, :n] - c.weight[b, :, :n]) <= 2e-5)
            assert np.array_equal(c.down(c.d_pos, c.pos.shape, np.int32)[b, :, :n], c.pos[b, :, :n])
        c.weight = got.copy()
        if i % 3 == 0:
            check(c, query(c.rng, c))
    hip.graph_free(graph)
    hip.h.hipStreamDestroy(stream)
    for p in (k, v, q, out, lse, src):
        hip.free(p)
    c.close()


# -------------------------------------------------------------- refusals ---
def test_refusals(hip, oracle):
    c = filled(hip, oracle, [5, 6], km.BF16, 4, 2, 64, 16)
    L, s, h = pw.lib(), c.seqs, c.c.h
    import ctypes
    r = ctypes.byref(s)
    p = c.d_weight
    before = c.pool()

    def app(rows=1, k=p, ks=0, v=p, vs=0, q=r):
        return L.welvet_kv_append_device(h, q, rows, None, k, ks, v, vs, None).code

    assert app(-1) == 1 and app(c.cap + 1) == 1 and app(k=None) == 1 and app(v=None) == 1
    assert app(ks=127) == 1 and app(vs=-1) == 1 and app(0) == 0 and app(q=None) == 1

    def att(tail=0, q=p, qs=0, scale=0.0, window=0, out=p, os_=0, seqs=r, sess=h):
        return L.welvet_kv_attend_device(sess, seqs, tail, q, qs, scale, window, 0, out, os_, None, None).code

    assert att(tail=-1) == 1 and att(tail=c.cap + 1) == 1 and att(q=None) == 1 and att(out=None) == 1
    assert att(qs=255) == 1 and att(os_=-256) == 1 and att(window=-1) == 1
    assert att(scale=-1.0) == 1 and att(scale=float("nan")) == 1 and att(scale=float("inf")) == 1
    assert att(scale=1e39) == 1

    def cho(budget=2, sinks=0, recent=0, src=p, seqs=r):
        return L.welvet_kv_choose_device(h, seqs, budget, sinks, recent, src, None).code

    assert cho(0) == 1 and cho(-1) == 1 and cho(c.cap + 1) == 1 and cho(2, 1, 2) == 1
    assert cho(2, -1) == 1 and cho(2, 0, -1) == 1 and cho(src=None) == 1
    assert cho(2, 2 ** 31 - 1, 2 ** 31 - 1) == 1
    assert L.welvet_kv_compact_device(h, r, 0, p, None).code == 1
    assert L.welvet_kv_compact_device(h, r, c.cap + 1, p, None).code == 1
    assert L.welvet_kv_compact_device(h, r, 2, None, None).code == 1
    assert L.welvet_kv_read_device(h, r, -1, None, None, p, p, None).code == 1
    assert L.welvet_kv_read_device(h, r, c.cap + 1, None, None, p, p, None).code == 1
    assert L.welvet_kv_read_device(h, r, 1, None, None, None, p, None).code == 1
    for kw in (dict(add=-1), dict(add=c.cap + 1), dict(cap=-1), dict(cap=c.cap + 1)):
        with pytest.raises(pw.WelvetError):
            c.c.advance(2, c.d_lens, **kw)
    with pytest.raises(pw.WelvetError):
        c.c.advance(3, c.d_lens, add=1)
    with pytest.raises(pw.WelvetError):
        c.c.advance(2, None, add=1)
    for bad in (dict(nseq=3), dict(nseq=-1), dict(table=None), dict(lens=None),
                dict(pos=c.d_pos + 4), dict(weight=c.d_weight + 8)):
        q = pw.KVSeqs(s.nseq, s.table, s.lens, s.next_pos, s.pos, s.weight)
        for name, value in bad.items():
            setattr(q, name, value)
        rq = ctypes.byref(q)
        assert app(q=rq) == 1 and att(seqs=rq) == 1 and cho(seqs=rq) == 1, bad
        assert L.welvet_kv_compact_device(h, rq, 2, p, None).code == 1
        assert L.welvet_kv_read_device(h, rq, 1, None, None, p, p, None).code == 1
    q = pw.KVSeqs(2, s.table, s.lens)                     # no running sums to choose by
    assert cho(seqs=ctypes.byref(q)) == 1
    plain = pw.KVCache(km.BF16, 4, 16, 4, 2, 64, 2, 2, track=False)
    assert att(sess=plain.h) == 1                         # sums asked of a session without them
    plain.close()
    for x, y in zip(before, c.pool()):
        assert np.array_equal(x, y)
    c.close()
