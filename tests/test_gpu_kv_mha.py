"""Attention layers over a K/V cache: prefill, then tokens one by one, against a
numpy decoder in 64 bits and against the layer's own forward of whole
sequences.

Q, K, V and O are signed permutations times a power of two and x multiples of
1/4 up to 2, so the projections round nothing that E4M3 weights and the
activations' terms do not hold: what is compared is the attention. Against the
numpy decoder the cache's tolerance holds (test_gpu_kv_cache.py: 2e-6), with RoPE's
results rounded to fp32 on both sides (half a step, 2^-24, of a pair's norm: in
scores of up to 16 another 1e-6 at the worst): 3e-6. The O projection adds its own
5e-5. The layer's forward holds K and P in two bf16 terms where there is no
ALiBi: 2e-5.
"""
import numpy as np
import pytest

import kv_model as km
import pywelvet as pw
from test_gpu_attention_masks import layer
from test_gpu_dense import rel_l2
from test_gpu_kv_cache import evict_model

pytestmark = pytest.mark.gpu

ROPE, NONE, ALIBI, ROPE_ALIBI = 0, 1, 2, 3


@pytest.fixture(scope="module")
def hip(gpu):
    return pw.Hip()


def turn(x, t, theta=10000.0):
    """RoPE of rows [heads][hd] at position t, rounded to fp32."""
    hd = x.shape[-1]
    half = hd // 2
    if not half:
        return x
    ang = t / theta ** (2 * np.arange(half) / hd)
    c, s = np.cos(ang), np.sin(ang)
    y = x.astype(np.float64).copy()
    a, b = y[:, :half].copy(), y[:, half:2 * half].copy()
    y[:, :half], y[:, half:2 * half] = a * c - b * s, a * s + b * c
    return y.astype(np.float32)


class Decoder:
    """The cache's numpy model driven by an attention layer's weights."""

    def __init__(self, c, weights, H, KVH, hd, pos, window=0):
        self.c, self.H, self.KVH, self.hd, self.pos, self.window = c, H, KVH, hd, pos, window
        self.Q, self.K, self.V, self.O = weights

    def rows(self, x, t):
        q, k, v = (x @ W.T for W in (self.Q, self.K, self.V))
        q, k, v = q.reshape(self.H, self.hd), k.reshape(self.KVH, self.hd), v.reshape(self.KVH, self.hd)
        if self.pos in (ROPE, ROPE_ALIBI):
            q, k = turn(q, t), turn(k, t)
        return q, k, v

    def step(self, x, oracle, track=None):
        """x [nseq][d]: attn [nseq][H][hd], lens and positions moved."""
        c = self.c
        q, k, v = zip(*(self.rows(x[b], c.next[b]) for b in range(c.nseq)))
        c.note_append(np.stack(k)[:, None], np.stack(v)[:, None], oracle)
        out, _ = c.want(np.stack(q), tail=1, window=self.window, alibi=self.pos in (ALIBI, ROPE_ALIBI),
                        track=track)
        c.count(1)
        return out


def sessions(batch, seq, H, KVH, hd, msl, mask, pos, W):
    return pw.MHASession(batch, seq, H * hd, H, KVH, hd, msl, mask, pos, pw.E4M3, pw.SCHEME_REF, *W)


@pytest.mark.parametrize("dtype", [km.F32, km.BF16, km.E4M3], ids=km.NAMES.get)
@pytest.mark.parametrize("H,KVH,hd,S,P,mask,pos,msl", [
    (4, 4, 64, 40, 25, 1, ROPE, 64), (12, 4, 64, 50, 33, 1, NONE, 64), (6, 2, 32, 70, 1, 1, ALIBI, 128),
    (2, 1, 128, 20, 19, 4, ROPE_ALIBI, 32), (4, 2, 48, 45, 40, 3, ROPE, 50), (3, 3, 20, 37, 30, 1, ROPE, 64),
])
def test_prefill_then_tokens_one_by_one(hip, oracle, dtype, H, KVH, hd, S, P, mask, pos, msl):
    Q, K, V, O, x = layer(S + hd, 1, S, H, KVH, hd)
    d = H * hd
    W = (Q, K, V, O)
    whole = sessions(1, S, H, KVH, hd, msl, mask, pos, W)
    full_attn, full_y = whole.execute(x)
    c = km.Cache(hip, dtype, H, KVH, hd, 1, 6, 16, seed=S, poison=True)
    dec = Decoder(c, W, H, KVH, hd, pos, msl if mask == 3 else 0)
    # the prompt, padded to the mounted length
    pre = sessions(1, P + 3, H, KVH, hd, msl, mask, pos, W)
    px = np.zeros((P + 3, d), np.float32)
    px[:P] = x[:P]
    dx, da, dy = c.up(px), c.up(np.zeros((P + 3, d), np.float32)), c.up(np.zeros((P + 3, d), np.float32))
    pre.prefill(c.c, c.seqs, P, dx, da, dy)
    hip.sync()
    assert rel_l2(c.down(da, (P + 3, d))[:P], full_attn[:P]) <= 4e-5  # (two forwards, 2e-5 each)
    for t in range(P):
        q, k, v = dec.rows(x[t], t)
        c.note_append(k[None, None], v[None, None], oracle)
        c.count(1)
    c.c.advance(1, c.d_lens, c.d_next, add=P)
    one = sessions(1, 1, H, KVH, hd, msl, mask, pos, W)
    dx, da, dy = c.up(x[:1]), c.up(np.zeros((1, d), np.float32)), c.up(np.zeros((1, d), np.float32))
    for t in range(P, S):
        c.put(dx, x[t:t + 1])
        one.decode(c.c, c.seqs, dx, da, dy)
        want = dec.step(x[t:t + 1], oracle).reshape(1, d)
        attn, y = c.down(da, (1, d)), c.down(dy, (1, d))
        assert rel_l2(attn, want) <= 3e-6, t
        assert rel_l2(y, attn @ O.T) <= 5e-5
        if dtype == km.F32:
            assert rel_l2(attn, full_attn[t:t + 1]) <= 2.3e-5
            assert rel_l2(y, full_y[t:t + 1]) <= 1.3e-4
        c.c.advance(1, c.d_lens, c.d_next, add=1)
    for s in (whole, pre, one):
        s.close()
    c.close()


@pytest.mark.parametrize("dtype,batch,H,KVH,hd,pos", [
    (km.BF16, 3, 4, 2, 64, ROPE), (km.E4M3, 7, 8, 8, 32, ROPE_ALIBI), (km.F32, 40, 4, 1, 64, ROPE),
    (km.BF16, 1, 2, 2, 40, ALIBI), (km.E4M3, 130, 2, 1, 64, ROPE),
])
def test_batches_decode_and_evict_in_a_graph(hip, oracle, dtype, batch, H, KVH, hd, pos):
    """A captured step of a batch: decode, advance, evict above 24 entries."""
    Q, K, V, O, _ = layer(batch, 1, 1, H, KVH, hd)
    d = H * hd
    c = km.Cache(hip, dtype, H, KVH, hd, batch, 2, 16, seed=batch, poison=True)
    dec = Decoder(c, (Q, K, V, O), H, KVH, hd, pos)
    m = sessions(batch, 1, H, KVH, hd, 64, 1, pos, (Q, K, V, O))
    x, attn, y = (c.up(np.zeros((batch, d), np.float32)) for _ in range(3))
    src = c.up(np.zeros((batch, KVH, 24), np.int32))
    stream = hip.stream()

    def step():
        m.decode(c.c, c.seqs, x, attn, y, stream=stream)
        c.c.advance(batch, c.d_lens, c.d_next, add=1, stream=stream)
        c.c.choose(c.seqs, 24, 2, 6, src, stream=stream)
        c.c.compact(c.seqs, 24, src, stream=stream)
        c.c.advance(batch, c.d_lens, cap=24, stream=stream)

    graph = hip.capture(stream, step)
    for i in range(30):
        nx = (c.rng.integers(-8, 9, size=(batch, d)) / 4).astype(np.float32)
        c.put(x, nx)
        if i % 5 == 3:  # eager calls between the replays
            step()
        else:
            hip.launch(graph, stream)
        hip.stream_sync(stream)
        sums = np.zeros(c.weight.shape)
        want = dec.step(nx, oracle, track=sums).reshape(batch, d)
        got = c.down(attn, (batch, d))
        assert rel_l2(got, want) <= 3e-6, i
        assert rel_l2(c.down(y, (batch, d)), got @ O.T) <= 5e-5
        c.weight = (c.weight + sums).astype(np.float32)
        evict_model(c, c.down(src, (batch, KVH, 24), np.int32), 24)
        kept = c.device_weight()
        for b in range(batch):
            n = c.lens[b]
            assert np.all(np.abs(kept[b, :, :n] - c.weight[b, :, :n]) <= 4e-6 * (i + 1))
        c.weight = kept
        assert np.array_equal(c.down(c.d_lens, (batch,), np.int32), c.lens)
        assert np.array_equal(c.down(c.d_next, (batch,), np.int32), c.next)
    hip.graph_free(graph)
    hip.h.hipStreamDestroy(stream)
    m.close()
    c.close()


def test_decode_at_the_capacity(hip, oracle):
    """A full sequence's token is dropped and attends to what is there."""
    Q, K, V, O, x = layer(3, 1, 40, 2, 2, 32)
    c = km.Cache(hip, km.F32, 2, 2, 32, 1, 2, 16)
    dec = Decoder(c, (Q, K, V, O), 2, 2, 32, ROPE)
    m = sessions(1, 1, 2, 2, 32, 64, 1, ROPE, (Q, K, V, O))
    dx, da, dy = (c.up(np.zeros((1, 64), np.float32)) for _ in range(3))
    for t in range(40):
        c.put(dx, x[t:t + 1])
        before = c.pool() if c.lens[0] == 32 else None
        m.decode(c.c, c.seqs, dx, da, dy)
        want = dec.step(x[t:t + 1], oracle).reshape(1, 64)
        assert rel_l2(c.down(da, (1, 64)), want) <= 3e-6, t
        if before:
            assert all(np.array_equal(a, b) for a, b in zip(before, c.pool()))
        c.c.advance(1, c.d_lens, c.d_next, add=1)
    m.close()
    c.close()


def test_refusals(hip):
    Q, K, V, O, x = layer(5, 1, 8, 4, 2, 32)
    c = km.Cache(hip, km.BF16, 4, 2, 32, 2, 1, 16)
    p = c.up(np.zeros((8, 128), np.float32))
    W = (Q, K, V, O)
    one, two, prompt = (sessions(b, s, 4, 2, 32, 64, 1, 0, W) for b, s in ((1, 1), (2, 1), (1, 8)))
    single = pw.KVSeqs(1, c.d_table, c.d_lens, c.d_next, c.d_pos, c.d_weight)

    def refused(f, *a):
        with pytest.raises(pw.WelvetError) as e:
            f(*a)
        assert e.value.code == 1

    refused(one.decode, c.c, c.seqs, p, p, p)             # two sequences, batch 1
    refused(prompt.decode, c.c, single, p, p, p)          # mounted for whole sequences
    refused(two.prefill, c.c, single, 1, p, p, p)         # batch 2
    refused(prompt.prefill, c.c, c.seqs, 1, p, p, p)      # two sequences
    refused(prompt.prefill, c.c, single, 9, p, p, p)
    refused(prompt.prefill, c.c, single, -1, p, p, p)
    refused(one.decode, c.c, single, None, p, p)
    refused(one.decode, c.c, single, p, None, p)
    refused(one.prefill, c.c, single, 1, p, p, None)
    for heads, kv, hd in ((4, 4, 32), (8, 2, 32), (4, 2, 64)):
        other = pw.KVCache(km.BF16, 2, 16, heads, kv, hd, 2, 1)
        refused(one.decode, other, single, p, p, p)
        refused(prompt.prefill, other, single, 1, p, p, p)
        other.close()
    plain = pw.KVCache(km.BF16, 2, 16, 4, 2, 32, 2, 1, track=False)
    refused(one.decode, plain, single, p, p, p)
    plain.close()
    L = pw.lib()
    assert L.welvet_mha_decode_device(None, c.c.h, None, p, p, p, None).code == 1
    assert L.welvet_mha_prefill_device(None, c.c.h, None, 1, p, p, p, None).code == 1
    assert L.welvet_mha_decode_device(one.h, None, None, p, p, p, None).code == 1
    for s in (one, two, prompt):
        s.close()
    c.close()
