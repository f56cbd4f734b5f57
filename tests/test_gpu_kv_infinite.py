"""Infinite keys under the attention of a K/V cache (test_kv_kernels_cpu.py runs
the same on the CPU)."""
import numpy as np
import pytest

import kv_model as km
import pywelvet as pw

OUT_TOL, LSE_TOL = 2e-6, 6e-6  # (test_gpu_kv_cache.py)


def check_infinite_keys(hip, oracle, dtype, n=70):
    """Keys with one infinite element, also by bf16's rounding: a score of -inf
    is a weight of 0 whatever the query's low bits are, one of +inf makes its
    head's output NaN; in E4M3 caches such a row is NaN."""
    big = np.inf if dtype != km.BF16 else np.float32(3.4e38)  # (rounds to inf in bf16)
    for sign in (1, -1):
        for seed in range(4):  # other low bits of the query
            c = km.Cache(hip, dtype, 4, 1, 32, 1, 5, seed=seed, poison=True)
            k, v = (c.rng.standard_normal((1, n, 1, 32)).astype(np.float32) for _ in range(2))
            at = [0, 5, 17, n - 1]
            k[0, at, 0, 3] = sign * big
            with np.errstate(invalid="ignore"):
                c.append(k, v, oracle if dtype != km.E4M3 else Finite(oracle))
            q = (2 * c.rng.standard_normal((1, 4, 32))).astype(np.float32)
            q[0, 0, 3], q[0, 1, 3] = -1.25, 1 + 2.0 ** -20   # one term; a smaller term of the other sign
            q[0, 2, 3], q[0, 3, 3] = np.pi, -np.e
            out, lse = c.attend(q)
            low = q[0, :, 3] * sign < 0                       # heads whose scores of these are -inf
            if dtype == km.E4M3:
                assert np.isnan(out).all() and np.isnan(lse).all()
            else:
                assert np.isnan(out[0, ~low]).all() and np.isnan(lse[0, ~low]).all()
                rest = np.setdiff1d(np.arange(n), at)
                for j in np.flatnonzero(low):
                    want, want_lse, w = km.softmax_attention(q[0, j], c.k[0, 0, rest], c.v[0, 0, rest])
                    assert np.linalg.norm(out[0, j] - want) <= OUT_TOL * np.linalg.norm(want)
                    assert abs(lse[0, j] - want_lse) <= LSE_TOL
            # nothing but such entries
            c.put(c.d_lens, np.array([1], np.int32))
            out, lse = c.attend(q)
            if dtype != km.E4M3:
                assert not out[0, low].any() and np.all(lse[0, low] == -np.inf)
                assert np.isnan(out[0, ~low]).all()
            c.close()


class Finite:
    """The codec for rows that are not finite: their codes are not looked at."""

    def __init__(self, oracle):
        self.oracle = oracle

    def pack(self, dtype, x):
        return self.oracle.pack(dtype, np.where(np.isfinite(x), x, np.float32(0)))

    def decode(self, dtype, code):
        return self.oracle.decode(dtype, code)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
def test_infinite_keys(gpu, oracle, dtype):
    check_infinite_keys(pw.Hip(), oracle, dtype)
