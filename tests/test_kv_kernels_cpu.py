"""The K/V cache's kernels run lane by lane on the CPU (kv_host.py)."""
import pytest

import kv_host


def clean(code):
    r = kv_host.run(code)
    assert r.returncode == 0 and r.stdout.endswith("done\n"), (r.returncode, r.stdout[-300:], r.stderr[-1500:])


@pytest.mark.parametrize("cap,budget,launch", [(100016, 16384, 4)] + [
    (cap, budget, launch) for cap, budget in ((20000, 1), (16912, 8100)) for launch in range(1, 7)] + [
    (3008, 100, 1), (3008, 100, 2)])
def test_choose_while_its_inputs_arrive(cap, budget, launch):
    """Sums and lengths that change between the launches of a choice (a caller
    that does not wait for them): the answer is nobody's, but nothing outside the
    call's memory is read or written, and the next call is right."""
    clean(f"""
n, kv, cap, budget = 2, 1, {cap}, {budget}
rng = np.random.default_rng(cap + {launch})
c = pw.KVCache(km.BF16, 1, 16, kv, kv, 16, n, cap // 16, True)
for kind in ("sums", "lens", "both"):
    w = np.zeros((n, kv, cap), np.float32)
    dw, dl = hip.upload(w), hip.upload(np.array([cap - 13, cap // 3], np.int32))
    s = pw.KVSeqs(n, hip.upload(np.zeros((n, cap // 16), np.int32)), dl, None, None, dw)
    src = hip.upload(np.zeros((n, kv, budget), np.int32))
    later, lens = rng.random((n, kv, cap), np.float32) + 1, np.array([cap, cap], np.int32)
    count = [0]
    def change(what):
        count[0] += what == 0
        if what == 0 and count[0] == {launch}:
            if kind != "lens": hip.copy_in(dw, later)
            if kind != "sums": hip.copy_in(dl, lens)
    hip.hook(change)
    c.choose(s, budget, 0, 0, src)
    hip.hook(None)
    hip.copy_in(dw, later), hip.copy_in(dl, lens - 5)
    c.choose(s, budget, 0, 0, src)
    got = hip.download(src, (n, kv, budget), np.int32)
    for b in range(n):
        m, h = lens[b] - 5, 0
        assert np.array_equal(got[b, h], km.choose(later[b, h, :m], np.arange(m), m, budget, 0, 0))
print("done")
""")


# (one sequence in parts, parts of a few and of many sequences, runs over few and
# over many, whole sequences)
@pytest.mark.parametrize("nseq,heads,kv,cap,most,dtype", [
    (1, 4, 2, 3200, 3200, "BF16"), (3, 20, 1, 1600, 1600, "E4M3"), (70, 2, 1, 960, 960, "F32"),
    (2, 64, 64, 2064, 2064, "BF16"), (70, 16, 16, 2640, 500, "E4M3"), (130, 4, 4, 64, 64, "F32"),
])
def test_attend_while_lengths_change(nseq, heads, kv, cap, most, dtype):
    """Lengths, positions and pages that change between workgroups (a caller that
    does not wait for them): nothing outside the call's memory is touched, and
    the next call is right."""
    clean(f"""
n, heads, kv, cap, most = {nseq}, {heads}, {kv}, {cap}, {most}
rng = np.random.default_rng(n + cap)
pages = 40
c = pw.KVCache(km.{dtype}, pages, 16, heads, kv, 16, n, cap // 16, True)
def some(what):
    if what == "lens":
        x = rng.integers(-2, most + 2, n) * (rng.random(n) < 0.7)
        return (x if rng.random() < 0.8 else np.full(n, most * rng.integers(0, 2))).astype(np.int32)
    return rng.integers(-1, pages + 1, (n, cap // 16)).astype(np.int32)
dl, dn, dt = hip.upload(some("lens")), hip.upload(some("lens")), hip.upload(some("table"))
dp = hip.upload(np.tile(np.arange(cap, dtype=np.int32), (n, kv, 1)))
dw = hip.upload(np.zeros((n, kv, cap), np.float32))
q, out = hip.upload(np.zeros((n, heads, 16), np.float32)), hip.upload(np.zeros((n, heads, 16), np.float32))
for often in (1.0, 0.05):
    def change(what):
        if what == 0 or rng.random() < often:
            hip.copy_in(dl, some("lens")), hip.copy_in(dn, some("lens")), hip.copy_in(dt, some("table"))
    for pos, weight, window in ((None, None, 0), (dp, dw, 0), (None, dw, 300)):
        hip.hook(change)
        c.attend(pw.KVSeqs(n, dt, dl, dn, pos, weight), q, out, window=window)
        hip.hook(None)
lens, table = rng.integers(0, most + 1, n).astype(np.int32), rng.integers(0, pages, (n, cap // 16)).astype(np.int32)
hip.copy_in(dl, lens), hip.copy_in(dt, table)
b = c.buffers()
size = pages * kv * 16 * 16 * {{1: 4, 3: 2, 4: 1}}[km.{dtype}]
for p in (b.k, b.v): hip.memset(p, 0x3C, size)   # all values alike
if b.v_scale:
    for p in (b.k_scale, b.v_scale): hip.memset(p, 0x3C, pages * kv * 16 * 4)
c.attend(pw.KVSeqs(n, dt, dl, None, None, None), q, out)
got = hip.download(out, (n, heads * 16))
assert not got[lens == 0].any()
got = got[lens > 0]
# (sums of up to `most` equal terms, over as many: half a step of rounding in each)
assert got.max() > 0 and got.max() - got.min() <= 2 * most * 2.0 ** -24 * got.max()
print("done")
""")


@pytest.mark.parametrize("dtype", ["F32", "BF16", "E4M3"])
def test_compact_from_a_hole(dtype):
    clean(f"""
import oracle_lib, test_gpu_kv_holes
test_gpu_kv_holes.check_compact_from_a_hole(hip, oracle_lib.Oracle(), km.{dtype})
print("done")
""")


@pytest.mark.parametrize("dtype", ["F32", "BF16", "E4M3"])
def test_infinite_keys(dtype):
    clean(f"""
import oracle_lib, test_gpu_kv_infinite
test_gpu_kv_infinite.check_infinite_keys(hip, oracle_lib.Oracle(), km.{dtype})
print("done")
""")
