"""The rule that keeps sequences whole, at the points where both sides were
measured (kv_rules.h, kv_one_part): the faster one is taken, or one within 5%."""
import pytest

import kv_model as km
import kv_plan as kp


@pytest.mark.parametrize("dtype,heads,kv,hd,nseq,cap,whole", [
    (km.E4M3, 32, 8, 128, 1, 400, True), (km.E4M3, 32, 8, 128, 1, 416, True), (km.E4M3, 32, 8, 128, 1, 608, True),
    (km.E4M3, 32, 8, 128, 4, 512, True), (km.E4M3, 32, 8, 128, 16, 640, True),
    (km.E4M3, 32, 8, 128, 16, 800, True), (km.E4M3, 32, 8, 128, 16, 1504, False),
    (km.E4M3, 32, 8, 128, 32, 800, True), (km.E4M3, 32, 8, 128, 64, 800, True),
    (km.E4M3, 32, 8, 128, 256, 4096, True), (km.E4M3, 32, 8, 128, 1000, 8000, True),
    (km.E4M3, 20, 1, 80, 24, 400, True), (km.E4M3, 20, 1, 80, 24, 1504, False),
    (km.BF16, 32, 8, 128, 1, 400, True), (km.BF16, 32, 8, 128, 16, 800, True),
    (km.BF16, 32, 8, 128, 64, 800, True), (km.BF16, 32, 8, 128, 64, 2048, False),
    (km.BF16, 12, 4, 64, 1, 608, True), (km.BF16, 12, 4, 64, 16, 800, True), (km.BF16, 12, 4, 64, 64, 1200, True),
    (km.F32, 16, 8, 256, 1, 400, False), (km.F32, 16, 8, 256, 16, 400, False), (km.F32, 16, 8, 256, 16, 800, False),
    (km.F32, 16, 8, 256, 64, 800, False), (km.F32, 16, 8, 256, 64, 1600, False),
    (km.F32, 16, 16, 64, 16, 800, True), (km.F32, 16, 16, 64, 8, 2048, False),
])
def test_whole_where_it_was_faster(dtype, heads, kv, hd, nseq, cap, whole):
    assert bool(kp.plan(nseq, heads, kv, hd, cap, dtype, False) & kp.WHOLE) == whole


def test_one_wave_takes_whole_sequences():
    for dtype, hd in ((d, h) for d in (km.F32, km.BF16, km.E4M3) for h in (1, 64, 65, 128, 129, 256)):
        for rows in (1, 399, 400, 600, 800, 5000, 65535):
            for cap in (16, 96, 112, 256, 1264, 16384, 2 ** 20):
                p = kp.plan(rows, 1, 1, hd, cap, dtype, False)
                assert not p & kp.ONE_WAVE or p & kp.WHOLE
                assert not (p & kp.WHOLE and p & kp.RUNS)
