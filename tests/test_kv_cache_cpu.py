"""K/V cache rules that need no GPU: refusals before a device is touched, and
the index rules built for the host (lengths, holes in a page table, rows past
4 GiB, E4M3 scales, the order of running sums)."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest

import kv_model
import pywelvet as pw

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


@pytest.fixture(scope="module")
def rules():
    out = os.path.join(tempfile.mkdtemp(prefix="kv_rules"), "kv.so")
    subprocess.check_call(["g++", "-O1", "-std=c++17", "-shared", "-fPIC",
                           "-I" + os.path.join(ROOT, "welvet.cuda_amd", "csrc"),
                           os.path.join(ROOT, "tests", "host", "kv_check.cpp"), "-o", out])
    L = ctypes.CDLL(out)
    L.kv_check_row.restype = ctypes.c_longlong
    for name in ("most_parts", "most_slots"):
        getattr(L, "kv_check_" + name).restype = ctypes.c_longlong
    L.kv_check_runs.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]
    L.kv_check_part_tiles.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]
    L.kv_check_scale.restype = ctypes.c_float
    L.kv_check_scale.argtypes = [ctypes.c_float]
    L.kv_check_key.restype = ctypes.c_uint
    L.kv_check_key.argtypes = [ctypes.c_float]
    return L


def mount(dtype=3, pages=4, page=16, heads=4, kv=2, hd=64, seqs=2, max_pages=2, flags=0):
    h = ctypes.c_void_p()
    st = pw.lib().welvet_kv_mount(dtype, pages, page, heads, kv, hd, seqs, max_pages, flags,
                                  ctypes.byref(h))
    return st, h


@pytest.mark.parametrize("bad,code", [
    (dict(pages=0), 1), (dict(page=0), 1), (dict(page=17), 1), (dict(page=8), 1),
    (dict(heads=0), 1), (dict(kv=0), 1), (dict(heads=5), 1), (dict(hd=0), 1), (dict(hd=-4), 1),
    (dict(hd=257), 2), (dict(seqs=0), 1), (dict(seqs=65536), 1), (dict(max_pages=0), 1),
    (dict(max_pages=1 << 27), 1), (dict(max_pages=2 ** 31 - 1, page=2 ** 31 - 16), 1),
    (dict(pages=2 ** 31 - 1, heads=60000, kv=60000, page=2 ** 20), 1),  # rows past 64 bits of bytes
    (dict(pages=1, heads=65535, kv=1, seqs=65535, max_pages=2 ** 26, flags=1), 1),
    (dict(flags=2), 1), (dict(dtype=0), 2), (dict(dtype=2), 2), (dict(dtype=5), 2),
    (dict(dtype=16), 2), (dict(dtype=-1), 2),
])
def test_mount_refusals(bad, code):
    st, h = mount(**bad)
    assert st.code == code and st.message.startswith(b"kv"), st.message
    assert not h.value


@pytest.mark.parametrize("heads,seqs,max_pages", [(2048, 65535, 1024), (65535, 65535, 256), (1024, 40000, 1024)])
def test_mount_refuses_more_tiles_than_a_share_can_count(heads, seqs, max_pages, rules):
    """Shared pages allow lengths far above the pool's: a share of all sequences'
    tiles has to stay an int."""
    st, h = mount(pages=1, page=2 ** 20, heads=heads, kv=heads, hd=8, seqs=seqs, max_pages=max_pages)
    assert st.code == 1 and b"capacity" in st.message and not h.value
    tiles = seqs * (max_pages * 2 ** 20 // 16)
    assert tiles // rules.kv_check_target(heads, 8) > 2 ** 30


def test_mount_without_a_device_is_code_2():
    if pw.lib().welvet_cuda_available():
        pytest.skip("a GPU is visible here")
    st, h = mount()
    assert st.code == 2 and not h.value
    assert pw.lib().welvet_kv_mount(3, 4, 16, 4, 2, 64, 2, 2, 0, None).code == 1


def test_null_sessions_are_refused():
    L, q = pw.lib(), pw.KVSeqs(0, 16, 16)
    r = ctypes.byref(q)
    assert L.welvet_kv_append_device(None, r, 1, None, 16, 0, 16, 0, None).code == 1
    assert L.welvet_kv_read_device(None, r, 1, None, None, 16, 16, None).code == 1
    assert L.welvet_kv_attend_device(None, r, 0, 16, 0, 0.0, 0, 0, 16, 0, None, None).code == 1
    assert L.welvet_kv_choose_device(None, r, 1, 0, 0, 16, None).code == 1
    assert L.welvet_kv_compact_device(None, r, 1, 16, None).code == 1
    assert L.welvet_kv_advance_device(None, 1, 16, None, None, 1, 0, None).code == 1
    assert L.welvet_kv_get_buffers(None, None).code == 1
    L.welvet_kv_release(None)
    assert L.welvet_mha_prefill_device(None, None, r, 1, 16, 16, 16, None).code == 1
    assert L.welvet_mha_decode_device(None, None, r, 16, 16, 16, None).code == 1


@pytest.mark.parametrize("length,tail,cap,want", [
    (0, 0, 32, 0), (5, 0, 32, 5), (5, 1, 32, 6), (31, 1, 32, 32), (32, 1, 32, 32),
    (40, 0, 32, 32), (-3, 0, 32, 0), (-3, 1, 32, 1), (2 ** 31 - 1, 2 ** 31 - 1, 1 << 30, 1 << 30),
    (-2 ** 31, 7, 32, 7),
])
def test_entries_of_a_sequence(rules, length, tail, cap, want):
    assert rules.kv_check_entries(length, tail, cap) == want


def test_rows_and_holes(rules):
    table = (ctypes.c_int * 5)(3, -1, 0, 4, 2 ** 31 - 1)
    pages, kv, page = 4, 3, 48

    def row(e, h):
        return rules.kv_check_row(table, e, h, pages, kv, page)

    assert row(0, 0) == (3 * kv) * page and row(47, 2) == (3 * kv + 2) * page + 47
    assert row(48, 0) == -1 and row(95, 1) == -1       # a negative page
    assert row(96, 1) == page and row(100, 1) == page + 4
    assert row(144, 0) == -1 and row(239, 0) == -1     # the first id past the pool, and the last int
    big = (ctypes.c_int * 1)(2 ** 31 - 2)
    assert rules.kv_check_row(big, 15, 7, 2 ** 31 - 1, 8, 16) == ((2 ** 31 - 2) * 8 + 7) * 16 + 15


def test_pitch_is_whole_16_byte_pieces(rules):
    for hd in range(1, 257):
        for dtype, n in ((1, 4), (3, 8), (4, 16)):
            p = rules.kv_check_pitch(dtype, hd)
            assert p % n == 0 and hd <= p < hd + n


def test_e4m3_scales(rules):
    f = rules.kv_check_scale
    assert f(0.0) == 1.0 and f(240.0) == 1.0
    assert f(1.0) == np.float32(1) / np.float32(240)
    assert f(1e-35) == 2.0 ** -96 and f(np.float32(2.0 ** -100)) == 2.0 ** -96
    assert np.isnan(f(float("inf"))) and np.isnan(f(float("nan")))


def test_order_of_running_sums(rules):
    f = rules.kv_check_key
    w = [float("-inf"), -3.0, -1e-45, 0.0, 1e-45, 1e-3, 1.0, 3e38, float("inf")]
    keys = [f(x) for x in w]
    assert keys == sorted(set(keys)) and keys[-1] < 0xFFFFFFFF
    assert f(-0.0) == f(0.0)
    assert f(float("nan")) < keys[0]


def test_model_choice_of_entries():
    """The numpy model that the GPU is compared with, on cases done by hand."""
    f = kv_model.choose
    at = np.arange(6)
    w = np.float32([5, 1, 4, 4, 9, 4])
    assert f(w, at, 6, 3, 0, 0).tolist() == [0, 4, 2]
    assert f(w, at, 6, 2, 0, 0).tolist() == [0, 4]
    assert f(w, at, 6, 3, 0, 1).tolist() == [0, 4, 5]
    assert f(w, at, 6, 3, 2, 0).tolist() == [0, 1, 4]
    assert f(w, at, 6, 8, 2, 0).tolist() == [0, 1, 2, 3, 4, 5, -1, -1]
    assert f(np.float32([1, np.nan, 1, 1]), np.arange(4), 4, 3, 0, 0).tolist() == [0, 3, 2]


def test_parts_fit_the_grid_and_the_scratch(rules):
    """The attention's cut: every tile in one part, never more parts than the
    grid has, nor more slots than the scratch."""
    rng = np.random.default_rng(5)
    for _ in range(3000):
        kt = int(rng.choice([16, 32]))
        cap = 16 * int(np.exp(rng.uniform(0, 9)))
        nseq, rows = int(np.exp(rng.uniform(0, 6))), int(np.exp(rng.uniform(0, 7)))
        lens = rng.integers(0, cap + 1, nseq)
        if rng.random() < 0.5:  # a few long ones
            lens = np.where(rng.random(nseq) < 0.1, lens, lens // 50)
        tiles = [-(-int(n) // kt) for n in lens]
        units = [max(1, t) for t in tiles]
        target = rules.kv_check_target(rows, int(rng.integers(1, 257)))
        step = rules.kv_check_part_tiles(sum(units), target, kt)
        most, slots = rules.kv_check_most_parts(nseq, target, cap), rules.kv_check_most_slots(target)
        if rules.kv_check_runs(sum(units), target, kt):
            groups = -(-sum(units) // step)
            assert groups <= min(target, most) and 2 * groups <= slots
        else:
            parts = [rules.kv_check_parts(t, step) for t in tiles]
            assert all(p >= 1 and (p - 1) * step < max(t, 1) <= p * step for p, t in zip(parts, tiles))
            assert sum(parts) <= most
            assert sum(p for p in parts if p > 1) <= slots
        # one sequence by itself
        step = rules.kv_check_part_tiles(tiles[0], target, kt)
        assert rules.kv_check_parts(tiles[0], step) <= min(target, rules.kv_check_most_parts(1, target, cap))


def test_runs_over_unequal_sequences(rules):
    """Runs with the cost of a start: every tile in one of them, one first part
    per sequence (also of those without tiles), the others in the runs that
    follow it, a run's two slots never taken twice, and no more runs than target
    and grid hold."""
    rng = np.random.default_rng(6)
    walked = 0
    for _ in range(600):
        kt = int(rng.choice([16, 32]))
        cap = 16 * int(np.exp(rng.uniform(3, 8)))
        nseq = int(np.exp(rng.uniform(0, 5.5))) + 1
        lens = rng.integers(0, cap + 1, nseq) * (rng.random(nseq) < 0.8)
        tiles = np.ascontiguousarray(-(-lens // kt), np.int32)
        total = int(np.maximum(tiles, 1).sum())
        target = int(rng.integers(1, 1 + max(1, total // (rules.kv_check_start() // kt))))
        if not rules.kv_check_runs(total, target, kt):
            continue
        walked += 1
        step = rules.kv_check_part_tiles(total + nseq * (rules.kv_check_start() // kt), target, kt)
        out = np.zeros((2 * target + nseq, 6), np.int32)
        n = rules.kv_check_walk(tiles.ctypes.data_as(ctypes.c_void_p), nseq, kt, step,
                                out.ctypes.data_as(ctypes.c_void_p), len(out))
        assert n >= nseq
        out = out[:n]
        assert out[:, 0].max() < min(target, rules.kv_check_most_parts(nseq, target, cap))
        slots = set()
        for b in range(nseq):
            mine = out[out[:, 1] == b]
            assert mine[0, 4] == 0 and np.all(mine[1:, 4] == 1) and mine[0, 5] == len(mine)
            assert np.all(mine[:, 0] == mine[0, 0] + np.arange(len(mine)))
            assert mine[0, 2] == 0 and mine[-1, 3] == tiles[b]
            assert np.array_equal(mine[1:, 2], mine[:-1, 3])
            if len(mine) > 1:
                assert np.all(mine[:, 5] > 1) and np.all(mine[:, 3] > mine[:, 2])
                # (as the join finds them: the first part's slot, then every second one)
                at = 2 * mine[0, 0] + 1 + np.r_[0, 1 + 2 * np.arange(len(mine) - 1)]
                assert np.array_equal(at, 2 * mine[:, 0] + (mine[:, 4] == 0))
                assert not slots & set(at.tolist()) and at.max() < rules.kv_check_most_slots(target)
                slots |= set(at.tolist())
    assert walked > 300


def test_one_wave_takes_whole_sequences(rules):
    rules.kv_check_one_wave.argtypes = [ctypes.c_longlong, ctypes.c_int, ctypes.c_int]
    kinds = {rules.kv_check_one_wave(rows, hd, cap) for rows in (1, 399, 400, 600, 800, 5000, 2 ** 32)
             for hd in (1, 64, 65, 128, 129, 256) for cap in (16, 112, 256, 1264, 2 ** 20, 2 ** 30)}
    assert kinds == {0, 2}


def test_first_tile_of_a_window(rules):
    for n in (0, 1, 31, 32, 33, 500):
        for window in (0, 1, 5, 32, 499, 500, 2 ** 31 - 1):
            for qp in (0, n - 1, n, n + 3, n + 600):
                for kt in (16, 32):
                    t = rules.kv_check_first_tile(n, qp, window, kt)
                    seen = [e for e in range(n) if not window or qp - e < window]
                    assert 0 <= t * kt <= n
                    assert not seen or t * kt <= seen[0] < t * kt + kt
