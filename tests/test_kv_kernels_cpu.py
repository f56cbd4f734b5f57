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
