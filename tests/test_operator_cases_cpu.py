"""perf/operators.py on the CPU: the plain forms against exact(), which is the
same from the definition in 64 bits and written apart, on small cases of every
kind.

The plain forms hold fp32 values. A score is a sum of hd products over
sqrt(hd): under 16 for queries of N(0, 4), and what ALiBi takes off leaves no
weight where it is more than 16 too. Such a sum is off by at most a few steps of
2^-24 of 32, 16 of them at hd 80: 3e-5 in lse, and relatively in a weight.
Values read back or moved are the same roundings: equal.
"""
import importlib.util
import os

import numpy as np
import pytest
import torch

ROOT = os.path.abspath(os.path.join(os.path.dirname(__file__), ".."))


class OnCpu(torch.overrides.TorchFunctionMode):
    """Tensors that are asked for on the GPU are made on the CPU."""

    def __torch_function__(self, func, types, args=(), kwargs=None):
        kwargs = dict(kwargs or {})
        if kwargs.get("device") == "cuda":
            kwargs["device"] = "cpu"
        return func(*args, **kwargs)


@pytest.fixture(scope="module")
def cases():
    spec = importlib.util.spec_from_file_location("operator_cases", os.path.join(ROOT, "perf", "operators.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m._gen = lambda seed: torch.Generator().manual_seed(seed)
    return m


def attend(nseq, cap, heads, kv, hd, dtype, window=0, alibi=False, track=False, page=16):
    return dict(kind="attend", nseq=nseq, cap=cap, ragged=True, dtype=dtype, heads=heads, kv=kv, hd=hd,
                page=page, window=window, alibi=alibi, track=track)


CASES = [
    attend(1, 1, 1, 1, 1, "f32"), attend(3, 100, 4, 2, 64, "bf16", track=True),
    attend(2, 643, 8, 2, 32, "bf16", alibi=True), attend(3, 700, 8, 4, 33, "e4m3", window=100),
    # (windows shorter than the sequences, with ALiBi)
    attend(1, 643, 8, 8, 16, "f32", window=19, alibi=True), attend(4, 900, 6, 2, 64, "bf16", 257, True, True),
    attend(2, 300, 20, 1, 80, "e4m3", 1, True, True, page=48), attend(2, 65, 4, 4, 40, "f32", 64, True),
    attend(2, 65, 4, 4, 40, "f32", 100, True),
    dict(kind="append", nseq=3, cap=70, rows=33, ragged=True, dtype="e4m3", heads=2, kv=2, hd=24, page=16),
    dict(kind="append", nseq=2, cap=40, rows=1, ragged=False, dtype="bf16", heads=4, kv=1, hd=7, page=32),
    dict(kind="append", nseq=2, cap=40, rows=5, ragged=True, dtype="f32", heads=4, kv=1, hd=7, page=16),
    dict(kind="compact", nseq=3, cap=70, ragged=True, dtype="e4m3", heads=2, kv=2, hd=24, page=16, budget=20),
    dict(kind="compact", nseq=2, cap=33, ragged=False, dtype="bf16", heads=2, kv=1, hd=5, page=16, budget=32),
    dict(kind="compact", nseq=2, cap=90, ragged=True, dtype="f32", heads=2, kv=2, hd=8, page=16, budget=64),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: f"{c['kind']}-{c['dtype']}-{c['nseq']}x{c['cap']}")
@pytest.mark.parametrize("seed", [1, 2])
def test_plain_forms_are_what_exact_says(cases, case, seed):
    with OnCpu():
        got = cases.run(cases.prepare(case, seed))
        want = cases.exact(case, seed)
    assert len(got) == len(want)
    for x, y in zip(got, want):
        if y is None:
            continue
        x, y = x.double().numpy(), y.numpy()
        assert x.shape == y.shape
        if case["kind"] != "attend":
            assert np.array_equal(x.astype(np.float32), y.astype(np.float32))
        else:
            assert np.abs(x - y).max() <= 3e-5 * max(1.0, np.abs(y).max())


class Order(OnCpu):
    """Notes when memory is written, waited for and handed to a call."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        # (without a write: views, sizes and addresses; memory of no content)
        if getattr(func, "__name__", "") not in ("data_ptr", "empty", "view", "__get__", "permute", "expand"):
            self.seen.append("write")
        return super().__torch_function__(func, types, args, kwargs)


@pytest.mark.parametrize("case", [CASES[1], CASES[9], CASES[12], dict(
    kind="choose", nseq=2, cap=100, ragged=True, heads=2, kv=2, budget=10, sinks=1, recent=4, moved=True)],
    ids=lambda c: c["kind"])
def test_calls_find_their_inputs_written(cases, case, monkeypatch):
    """The calls run on a stream of their own: whatever they read has to be
    waited for after its last write, by prepare() for run()."""
    order = Order()

    class Cache:
        def __init__(self, *a):
            pass

        def append(self, *a, **kw):
            order.seen.append("call")

        attend = choose = compact = read = append

    class Binding:
        KVCache = Cache
        KVSeqs = staticmethod(lambda *a: a)

    monkeypatch.setattr(cases, "own", True)
    monkeypatch.setattr(cases, "_stream", lambda: 1)
    monkeypatch.setattr(cases, "_binding", lambda: Binding)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda: order.seen.append("wait"))
    with order:
        state = cases.prepare(case, 3)
        cases.run(state)
    last = {"write": 0}
    for i, what in enumerate(order.seen):
        assert what != "call" or last.get("wait", -1) > last["write"], order.seen[max(0, i - 5):i + 1]
        last[what] = i
    assert "call" in last
