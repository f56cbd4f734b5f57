"""A paged K/V cache in numpy: what the library's cache calls have to give.

Values are held as float64 of what an entry stands for in the cache's type;
nothing here is shared with the library but the E4M3 codec, which is the CPU
oracle's.
"""
import ctypes

import numpy as np

import pywelvet as pw

F32, BF16, E4M3 = pw.KV_F32, pw.KV_BF16, pw.KV_E4M3
NAMES = {F32: "f32", BF16: "bf16", E4M3: "e4m3"}


def bf16(x):
    """Nearest bfloat16, ties to even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    u = (u + 0x7FFF + ((u >> 16) & 1)) >> 16 << 16
    return u.astype(np.uint32).view(np.float32)


def stored(x, dtype, oracle):
    """fp32 rows [..., hd] as the cache holds them, in fp32."""
    x = np.ascontiguousarray(x, np.float32)
    if dtype == F32:
        return x
    if dtype == BF16:
        return bf16(x).reshape(x.shape)
    rows = x.reshape(-1, x.shape[-1])
    s = np.abs(rows).max(1) / np.float32(240)
    s = np.where(s == 0, np.float32(1), np.maximum(s, np.float32(2.0 ** -96)))
    codes = oracle.pack(pw.E4M3, np.ascontiguousarray(rows / s[:, None]))
    values = np.array([oracle.decode(pw.E4M3, c) for c in range(256)], np.float32)
    return (values[codes].reshape(rows.shape) * s[:, None]).reshape(x.shape)


def softmax_attention(q, k, v, bias=None, scale=None):
    """One query [hd] over k, v [n, hd] in f64: out, lse, weights."""
    if len(k) == 0:
        return np.zeros(q.shape[-1]), -np.inf, np.zeros(0)
    s = k.astype(np.float64) @ q.astype(np.float64) * (scale or 1 / np.sqrt(q.shape[-1]))
    if bias is not None:
        s = s + bias
    m = s.max()
    p = np.exp(s - m)
    return p @ v.astype(np.float64) / p.sum(), m + np.log(p.sum()), p / p.sum()


def choose(weight, pos, end, budget, sinks, recent):
    """src [budget] of one sequence and head; weight and pos of its entries."""
    n = len(weight)
    src = np.where(np.arange(budget) < n, np.arange(budget), -1).astype(np.int32)
    if n <= budget:
        return src
    w = weight.astype(np.float64)
    first = (pos < sinks) | (pos >= end - recent)
    # highest first: protected, then by value with NaN last; ties by index
    order = sorted(range(n), key=lambda e: (not first[e], np.isnan(w[e]) and not first[e],
                                            0.0 if first[e] or np.isnan(w[e]) else -w[e], e))
    keep = np.zeros(n, bool)
    keep[order[:budget]] = True
    src[~keep[:budget]] = np.flatnonzero(keep[budget:]) + budget
    return src


class Cache:
    """A mounted cache with its caller's buffers, and the same in numpy."""

    def __init__(self, hip, dtype, heads, kv, hd, nseq, max_pages, page=16, spare=3, seed=0,
                 positions=True, track=True, poison=False, table=None, num_pages=None):
        self.hip, self.dtype, self.heads, self.kv, self.hd = hip, dtype, heads, kv, hd
        self.nseq, self.page, self.max_pages, self.cap = nseq, page, max_pages, max_pages * page
        self.rng = np.random.default_rng(seed)
        self.num_pages = num_pages or nseq * max_pages + spare
        if table is None:
            table = self.rng.permutation(self.num_pages)[:nseq * max_pages].reshape(nseq, max_pages)
        self.table = np.ascontiguousarray(table, np.int32)
        self.c = pw.KVCache(dtype, self.num_pages, page, heads, kv, hd, nseq, max_pages, track)
        b = self.c.buffers()
        self.pitch = b.pitch
        self.elem = {F32: 4, BF16: 2, E4M3: 1}[dtype]
        self.rows = self.num_pages * kv * page
        if poison:  # memory that no entry was written to is all NaN
            for p in (b.k, b.v):
                hip.memset(p, 0xFF, self.rows * self.pitch * self.elem)
            if dtype == E4M3:
                for p in (b.k_scale, b.v_scale):
                    hip.memset(p, 0xFF, self.rows * 4)
            hip.sync()
        self.bufs = []
        self.d_table = self.up(self.table)
        self.lens = np.zeros(nseq, np.int32)
        self.next = np.zeros(nseq, np.int32)
        self.pos = np.full((nseq, kv, self.cap), -7, np.int32)
        self.weight = np.full((nseq, kv, self.cap), 9.0, np.float32)
        self.d_lens, self.d_next = self.up(self.lens), self.up(self.next)
        self.d_pos = self.up(self.pos) if positions else None
        self.d_weight = self.up(self.weight) if track else None
        # [nseq][kv][cap][hd] of what the entries stand for
        self.k = np.zeros((nseq, kv, self.cap, hd))
        self.v = np.zeros((nseq, kv, self.cap, hd))
        self.seqs = pw.KVSeqs(nseq, self.d_table, self.d_lens, self.d_next, self.d_pos, self.d_weight)

    def up(self, a):
        p = self.hip.upload(np.ascontiguousarray(a))
        self.bufs.append(p)
        return p

    def put(self, p, a):
        self.hip.copy_in(p, a)

    def down(self, p, shape, dtype=np.float32):
        self.hip.sync()
        return self.hip.download(p, shape, dtype)

    def pool(self):
        """K and V rows and the scales as raw bits."""
        b = self.c.buffers()
        n = self.rows * self.pitch * self.elem
        out = [self.down(p, (self.num_pages, self.kv, self.page, self.pitch * self.elem), np.uint8)
               for p in (b.k, b.v)]
        assert out[0].nbytes == n
        if self.dtype == E4M3:
            out += [self.down(p, (self.num_pages, self.kv, self.page), np.uint32)
                    for p in (b.k_scale, b.v_scale)]
        return out

    def valid(self, b, e):
        p = self.table[b, e // self.page]
        return 0 <= p < self.num_pages

    def append(self, k, v, oracle, counts=None, **kw):
        """k, v [nseq][rows][kv][hd]; the numpy side follows, lens too."""
        rows = k.shape[1]
        dk, dv = self.up(k), self.up(v)
        dc = self.up(np.asarray(counts, np.int32)) if counts is not None else None
        self.c.append(self.seqs, rows, dk, dv, dc, **kw)
        self.note_append(k, v, oracle, counts)
        self.c.advance(self.nseq, self.d_lens, self.d_next, dc, add=rows)
        self.count(rows, counts)

    def count(self, rows, counts=None):
        c = np.clip(counts if counts is not None else np.full(self.nseq, rows), 0, rows)
        self.lens = np.minimum(self.lens + c, self.cap).astype(np.int32)
        self.next = (self.next + c).astype(np.int32)

    def note_append(self, k, v, oracle, counts=None):
        rows = k.shape[1]
        sk, sv = stored(k, self.dtype, oracle), stored(v, self.dtype, oracle)
        for b in range(self.nseq):
            for i in range(rows if counts is None else min(rows, counts[b])):
                e = self.lens[b] + i
                if e >= self.cap:
                    break
                self.k[b, :, e], self.v[b, :, e] = sk[b, i], sv[b, i]
                self.pos[b, :, e], self.weight[b, :, e] = self.next[b] + i, 0.0

    def attend(self, q, tail=0, scale=0.0, window=0, alibi=False, lse=True, stream=None):
        """q [nseq][heads][hd] through the library: out, lse."""
        dq = self.up(q)
        out = self.up(np.full((self.nseq, self.heads * self.hd), 777, np.float32))
        dl = self.up(np.full((self.nseq, self.heads), 777, np.float32)) if lse else None
        self.c.attend(self.seqs, dq, out, tail, scale, window, alibi, dl, stream=stream)
        return (self.down(out, (self.nseq, self.heads, self.hd)),
                self.down(dl, (self.nseq, self.heads)) if lse else None)

    def want(self, q, tail=0, scale=0.0, window=0, alibi=False, track=None):
        """The same from the numpy side; with track, adds to self.weight."""
        out = np.zeros((self.nseq, self.heads, self.hd))
        lse = np.full((self.nseq, self.heads), -np.inf)
        group = self.heads // self.kv
        for b in range(self.nseq):
            n = min(int(self.lens[b]) + tail, self.cap)
            qp = int(self.next[b]) + tail - 1
            at = np.arange(n)
            ok = np.array([self.valid(b, e) for e in at], bool)
            for j in range(self.heads):
                h = j // group
                pos = self.pos[b, h, :n] if self.d_pos else at
                see = ok & ((qp - pos < window) if window else True)
                slope = 2.0 ** (-8.0 * (j + 1) / self.heads)
                bias = -slope * np.abs(qp - pos[see]) if alibi else None
                o, l, w = softmax_attention(q[b, j], self.k[b, h, :n][see], self.v[b, h, :n][see],
                                            bias, scale or None)
                out[b, j], lse[b, j] = o, l
                if track is not None:
                    track[b, h, :n][see] += w
        return out, lse

    def device_weight(self):
        return self.down(self.d_weight, self.weight.shape)

    def close(self):
        self.hip.sync()
        self.c.close()
        for p in self.bufs:
            self.hip.free(p)
        self.bufs = []
