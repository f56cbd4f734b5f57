"""Eviction with entries in holes of the page table (test_kv_kernels_cpu.py runs
the same on the CPU)."""
import numpy as np
import pytest

import kv_model as km
import pywelvet as pw

OUT_TOL = 2e-6  # (test_gpu_kv_cache.py)


def check_compact_from_a_hole(hip, oracle, dtype):
    """Entries 32 to 47 lie in a hole and are kept as the most recent ones: the
    slots that they would move to keep their own entries with their own positions
    and sums, and the attention is the one over these."""
    table = np.array([[3, 0, -1], [1, 2, 4]], np.int32)
    c = km.Cache(hip, dtype, 4, 2, 64, 2, 3, table=table, num_pages=5, poison=True)
    k, v = (c.rng.standard_normal((2, 48, 2, 64)).astype(np.float32) for _ in range(2))
    c.append(k, v, oracle)
    c.weight = c.rng.random(c.weight.shape, np.float32)
    c.put(c.d_weight, c.weight)
    src = c.up(np.zeros((2, 2, 32), np.int32))
    c.c.choose(c.seqs, 32, 0, 16, src)
    chosen = c.down(src, (2, 2, 32), np.int32)
    assert (chosen >= 32).any(-1).all()
    c.c.compact(c.seqs, 32, src)
    c.c.advance(2, c.d_lens, cap=32)
    for h in range(2):  # (sequence 0 has nothing behind the budget that could move)
        for j, e in enumerate(chosen[1, h]):
            for x in (c.k, c.v, c.pos, c.weight):
                x[1, h, j] = x[1, h, e]
    assert np.array_equal(c.device_weight(), c.weight)
    assert np.array_equal(c.down(c.d_pos, c.pos.shape, np.int32), c.pos)
    c.lens = np.array([32, 32], np.int32)
    q = (2 * c.rng.standard_normal((2, 4, 64))).astype(np.float32)
    got, _ = c.attend(q, alibi=True)
    want, _ = c.want(q, alibi=True)
    assert np.linalg.norm(got - want) <= OUT_TOL * np.linalg.norm(want)
    c.close()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_compact_from_a_hole(gpu, oracle, dtype):
    check_compact_from_a_hole(pw.Hip(), oracle, dtype)
