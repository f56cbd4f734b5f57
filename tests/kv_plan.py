"""Which attention kernel a K/V cache call takes, by the library's own rules
built for the host."""
import ctypes
import functools
import os
import subprocess
import tempfile

import kv_model as km

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))
WHOLE, ONE_WAVE, RUNS = 1, 2, 4
PADDED = [(d, h) for d in (km.F32, km.BF16, km.E4M3) for h in (32, 64, 96, 128, 192, 256)
          if d != km.E4M3 or h % 64 == 0]


@functools.lru_cache(None)
def rules():
    out = os.path.join(tempfile.mkdtemp(prefix="kv_plan"), "plan.so")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC",
                           "-I" + os.path.join(ROOT, "welvet.cuda_amd", "csrc"),
                           os.path.join(ROOT, "tests", "host", "kv_plan_check.cpp"), "-o", out])
    L = ctypes.CDLL(out)
    L.kv_check_takes_runs.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    return L


def rows(heads, kv):
    return kv * -(-(heads // kv) // 16)


def plan(nseq, heads, kv, hd, cap, dtype, gen):
    return rules().kv_check_plan(nseq, rows(heads, kv), hd, cap, dtype, int(gen))


def kernel(nseq, heads, kv, hd, cap, dtype, gen):
    """(type, padded head dims, general, runs, waves)."""
    p = plan(nseq, heads, kv, hd, cap, dtype, gen)
    return dtype, rules().kv_check_padded_hd(dtype, hd), gen, p & RUNS != 0, 1 if p & ONE_WAVE else 4


def takes_runs(lens, heads, kv, hd, dtype):
    kt = 16 if dtype == km.F32 else 32
    return bool(rules().kv_check_takes_runs(sum(max(1, -(-int(n) // kt)) for n in lens), rows(heads, kv),
                                            hd, dtype))
