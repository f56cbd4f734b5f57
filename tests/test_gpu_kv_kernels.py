"""Every attention kernel of the K/V cache: type, padded head dims, plain and
general, runs over sequences, workgroups of four waves and of one. Which one a
case takes is asked of the library's own rules, so that a change of these cannot
leave a kernel untested."""
import numpy as np
import pytest

import kv_model as km
import kv_plan as kp
import pywelvet as pw
from test_gpu_kv_cache import check, filled, query

WAYS = ["parts", "one wave", "runs"]


def case(way, dtype, padded):
    """lens, heads, kv, hd, page: head dims that fill the kernel's, or do not."""
    i = kp.PADDED.index((dtype, padded))
    hd = padded - [0, 1, 8, 13][i % 4]
    rng = np.random.default_rng(padded + dtype)
    if way == "parts":
        return [0, 1, 31, 33, 400, 700], 6, 2, hd, 16
    if way == "one wave":
        lens = rng.integers(0, 60, 100)
        lens[3], lens[70] = 60, 0
        return lens.tolist(), 8 * (1 + i % 3), 8, hd, 16
    # (few entries: a little more than every workgroup's least part)
    target = 256 * (4 if hd <= 64 else 3 if hd <= 128 else 2) // 64
    rest = (256 * target - 1697) * 2 // 5
    return [0, 1697, 1, rest, rest + 17, rest - 31], 64 * (1 + i % 2), 64, hd, 32


def kernels(way, dtype, padded):
    lens, heads, kv, hd, page = case(way, dtype, padded)
    cap = -(-(max(lens) + 1) // page) * page
    return [kp.kernel(len(lens), heads, kv, hd, cap, dtype, gen) for gen in (False, True)]


def test_every_kernel_has_a_case():
    seen = {k for way in WAYS for d, p in kp.PADDED for k in kernels(way, d, p)}
    want = {(d, p, gen, runs, waves) for d, p in kp.PADDED for gen in (False, True)
            for runs, waves in ((False, 1), (False, 4), (True, 4))}
    assert seen == want


@pytest.fixture(scope="module")
def hip(gpu):
    return pw.Hip()


@pytest.mark.gpu
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("dtype,padded", kp.PADDED, ids=lambda x: km.NAMES.get(x, x))
def test_attend(hip, oracle, way, dtype, padded):
    lens, heads, kv, hd, page = case(way, dtype, padded)
    want = {"parts": (False, 4), "one wave": (False, 1), "runs": (True, 4)}[way]
    assert all(k == (dtype, padded, gen) + want for gen, k in enumerate(kernels(way, dtype, padded)))
    assert (way == "runs") == kp.takes_runs(lens, heads, kv, hd, dtype)
    c = filled(hip, oracle, lens, dtype, heads, kv, hd, page, seed=padded, positions=way != "runs")
    q = query(c.rng, c)
    check(c, q)  # with running sums
    c.seqs.weight = c.d_weight = None
    check(c, q)
    check(c, q, alibi=True)
    first = check(c, q, window=max(lens) // 2)
    assert np.array_equal(first, c.attend(q, window=max(lens) // 2)[0])
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,hd", [(km.F32, 40), (km.BF16, 64), (km.E4M3, 56)], ids=lambda x: km.NAMES.get(x, x))
def test_runs_over_many_sequences(hip, oracle, dtype, hd):
    """More sequences than a wave has lanes, most of them short."""
    n, heads, kv = 70, 16, 16
    rng = np.random.default_rng(hd)
    lens = rng.integers(0, 600, n)
    lens[rng.random(n) < 0.2] = 0
    lens[[0, 40, 69]] = 1, 2990, 700
    assert kp.kernel(n, heads, kv, hd, 3008, dtype, False)[3] and kp.takes_runs(lens, heads, kv, hd, dtype)
    c = filled(hip, oracle, lens.tolist(), dtype, heads, kv, hd, 16, seed=hd, track=False, room=18)
    q = query(c.rng, c)
    first = check(c, q)
    assert c.cap == 3008 and np.array_equal(first, c.attend(q)[0])
    check(c, q, alibi=True)
    c.close()
