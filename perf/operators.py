"""Performance cases of the paged K/V cache: filling it, the attention of one
new token per sequence over it, and eviction from it by accumulated attention
weight.

Kinds (field "kind" of a case):
  append   K and V rows of new tokens into the pages (E4M3 caches: and read
           back as the fp32 values that the codes and scales stand for)
  attend   one query per sequence over its entries, split over the length and
           joined; "track" adds every entry's weight to its running sum
  choose   the entries to keep, by running sum, sinks and recent ones first
  compact  the kept entries moved into the slots of those that go

A cache is a pool of pages of "page" entries; a table gives the pages of each
sequence. Inputs are made on the GPU from the seed alone: keys and values are
N(0, 1), as after a projection of normalised activations, and queries N(0, 4),
so that the softmax has a peak and a tail.

With `own` false, run() computes the same from elementary torch operations.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": 1, "bf16": 3, "e4m3": 4}
BYTES = {"f32": 4, "bf16": 2, "e4m3": 1}


def listed():
    return [
        # One decode step of 32 sequences: a token's K and V of each. Latency.
        dict(name="append_bf16_32x1", kind="append", nseq=32, cap=1024, rows=1, ragged=False,
             dtype="bf16", heads=12, kv=4, hd=64, page=16),
        # Prompts of up to 512 tokens into an FP8 cache, and what it then holds.
        dict(name="append_e4m3_8x512", kind="append", nseq=8, cap=1024, rows=512, ragged=True,
             dtype="e4m3", heads=16, kv=16, hd=64, page=64),
        # The first tokens of one conversation: the least work there is.
        dict(name="attend_bf16_1x96", kind="attend", nseq=1, cap=96, ragged=False, dtype="bf16",
             heads=16, kv=16, hd=64, page=16, window=0, alibi=False, track=False),
        # One sequence with a long context: only the split fills the GPU.
        dict(name="attend_bf16_1x131072", kind="attend", nseq=1, cap=131072, ragged=False,
             dtype="bf16", heads=32, kv=8, hd=128, page=64, window=0, alibi=False, track=False),
        # A serving batch of unequal sequences over an FP8 cache.
        dict(name="attend_e4m3_64x4096", kind="attend", nseq=64, cap=4096, ragged=True,
             dtype="e4m3", heads=32, kv=8, hd=128, page=32, window=0, alibi=False, track=False),
        # Decoding with eviction: running sums kept, ALiBi, odd lengths.
        dict(name="attend_track_bf16_16x8191", kind="attend", nseq=16, cap=8191, ragged=True,
             dtype="bf16", heads=12, kv=4, hd=64, page=32, window=0, alibi=True, track=True),
        # A full-precision cache with a head of its own for every query head.
        dict(name="attend_f32_8x2047", kind="attend", nseq=8, cap=2047, ragged=True, dtype="f32",
             heads=16, kv=16, hd=64, page=16, window=0, alibi=False, track=False),
        # Twenty query heads over one K/V head of an uncommon size, windowed.
        dict(name="attend_window_e4m3_24x1500", kind="attend", nseq=24, cap=1500, ragged=True,
             dtype="e4m3", heads=20, kv=1, hd=80, page=16, window=1024, alibi=False, track=False),
        # Half of a batch's entries go.
        dict(name="choose_8x4096_to_2048", kind="choose", nseq=8, cap=4096, ragged=True, heads=32,
             kv=8, budget=2048, sinks=4, recent=256, moved=False),
        # Long sequences that were evicted from before: positions of their own.
        dict(name="choose_2x100003_to_16384", kind="choose", nseq=2, cap=100003, ragged=True,
             heads=8, kv=8, budget=16384, sinks=4, recent=1024, moved=True),
        # One entry of each K/V head makes room for the next token.
        dict(name="compact_bf16_32x1025_to_1024", kind="compact", nseq=32, cap=1025, ragged=False,
             dtype="bf16", heads=12, kv=4, hd=64, page=32, budget=1024),
        # Half of the entries go, a quarter moves.
        dict(name="compact_bf16_16x8192_to_4096", kind="compact", nseq=16, cap=8192, ragged=True,
             dtype="bf16", heads=32, kv=8, hd=128, page=64, budget=4096),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        # no dearer than the largest listed case, and the plain form's
        # gathered fp32 copies within some GB
        if w["bytes"] <= 5.0e8 and w["flops"] <= 2.0e9 and c["nseq"] * c["cap"] * c["kv"] * c.get("hd", 1) <= 1 << 28:
            return c


def _draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "attend", "choose", "compact"])
    kv = rng.choice([1, 2, 4, 5, 8, 16])
    c = dict(kind=kind, nseq=_log(rng, 1, 128), heads=kv * rng.choice([1, 1, 2, 3, 4, 8, 20]), kv=kv,
             ragged=rng.random() < 0.7)
    if kind != "choose":
        c.update(dtype=rng.choice(sorted(DTYPES)), page=16 * rng.choice([1, 1, 2, 3, 4, 8]),
                 hd=rng.choice([32, 64, 64, 80, 96, 128, 128, 256, rng.randint(1, 256)]))
    if kind == "append":
        c["rows"] = 1 if rng.random() < 0.5 else _log(rng, 2, 1024)
        c["cap"] = c["rows"] + _log(rng, 1, 4096)
    elif kind == "attend":
        c.update(cap=_log(rng, 1, 131072), window=rng.choice([0, 0, 0, _log(rng, 1, 8192)]),
                 alibi=rng.random() < 0.25, track=rng.random() < 0.3)
    else:
        c["cap"] = _log(rng, 8, 131072 if kind == "choose" else 16384)
        c["budget"] = _log(rng, 4, c["cap"])
        if kind == "choose":
            c.update(sinks=rng.randint(0, c["budget"] // 4), recent=rng.randint(0, c["budget"] // 2),
                     moved=rng.random() < 0.5)
    return c


def _lens(case):
    """Entries of each sequence: all "cap", or spread from an eighth of it up."""
    n, cap = case["nseq"], case["cap"]
    if case["kind"] == "append":
        cap = max(1, cap - case["rows"])  # what the cache holds before the call
    if not case["ragged"]:
        return [cap] * n
    lo = (cap + 7) // 8
    return [cap - (cap - lo) * i // max(1, n - 1) for i in range(n)]


def _counts(case):
    """New tokens of each sequence of an append."""
    r, n = case["rows"], case["nseq"]
    return [r - (r - 1) * i // n for i in range(n)] if case["ragged"] else [r] * n


# ------------------------------------------------------------------ work ---
def _entry_bytes(case):
    """K and V of one entry and K/V head, with their scales."""
    return 2 * (case["hd"] * BYTES[case["dtype"]] + (4 if case["dtype"] == "e4m3" else 0))


def work(case):
    kind, n, kv = case["kind"], case["nseq"], case["kv"]
    lens = _lens(case)
    if kind == "append":
        tokens = sum(_counts(case))
        row = 8 * case["hd"]  # fp32 K and V
        back = row + _entry_bytes(case) if case["dtype"] == "e4m3" else 0
        return {"bytes": float(tokens * kv * (row + _entry_bytes(case) + back)), "flops": 0.0}
    if kind == "attend":
        seen = sum(min(x, case["window"]) if case["window"] else x for x in lens)
        ends = 8 * n * case["heads"] * case["hd"]
        track = 8 * sum(lens) * kv if case["track"] else 0
        return {"bytes": float(seen * kv * _entry_bytes(case) + ends + track),
                "flops": 4.0 * seen * case["heads"] * case["hd"]}
    keep = [min(x, case["budget"]) for x in lens]
    if kind == "choose":
        return {"bytes": 4.0 * kv * (sum(lens) * (2 if case["moved"] else 1) + n * case["budget"]),
                "flops": 0.0}
    # of the entries that go, those below the budget are filled again
    moved = sum((x - k) * k / max(1, x) for x, k in zip(lens, keep))
    return {"bytes": kv * (moved * (2 * _entry_bytes(case) + 16) + 4.0 * n * case["budget"]),
            "flops": 0.0}


# ---------------------------------------------------------------- inputs ---
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)


def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std


def _int32(values):
    return torch.tensor(values, device="cuda", dtype=torch.int32)


def _weights(g, case):
    """Running sums as softmax weights leave them, the newest still zero."""
    n, kv, cap = case["nseq"], case["kv"], case["cap"]
    w = torch.exp(_normal(g, n, kv, cap, std=2.0)) * 1e-3
    late = torch.arange(cap, device="cuda") >= cap - cap // 64
    return torch.where(late, torch.zeros_like(w), w)


def _capacity(case):
    """Entries that a row of the page table covers."""
    page = case.get("page", 16)
    return -(-case["cap"] // page) * page


def _wide(t, case, fill):
    """Per-entry values padded to the table's capacity."""
    return torch.nn.functional.pad(t, (0, _capacity(case) - t.shape[-1]), value=fill).contiguous()


def _inputs(case, seed):
    g, kind, n, kv = _gen(seed), case["kind"], case["nseq"], case["kv"]
    v = {"lens": _int32(_lens(case))}
    if kind != "choose":
        pages = _capacity(case) // case["page"]
        order = torch.randperm(n * pages + 3, generator=g, device="cuda")
        v["table"] = order[:n * pages].to(torch.int32).view(n, pages)
        v["pool_pages"] = n * pages + 3
    else:
        v["table"] = torch.arange(n * (_capacity(case) // 16), device="cuda",
                                  dtype=torch.int32).view(n, -1)
    if kind == "append":
        v["counts"] = _int32(_counts(case))
        v["k"], v["v"] = (_normal(g, n, case["rows"], kv, case["hd"]) for _ in range(2))
    elif kind != "choose":
        v["k"], v["v"] = (_normal(g, n, case["cap"], kv, case["hd"]) for _ in range(2))
    if kind == "attend":
        v["q"] = _normal(g, n, case["heads"], case["hd"], std=2.0)
        if case["track"]:
            v["weight"] = _wide(_weights(g, case), case, 0.0)
    elif kind == "choose":
        v["weight"] = _wide(_weights(g, case), case, 0.0)
        if case["moved"]:
            # positions of what is left after earlier evictions, in slot order
            # but for the slots that were filled again
            pos = torch.arange(case["cap"], device="cuda", dtype=torch.int32) * 2
            swap = torch.rand(n, kv, case["cap"], generator=g, device="cuda").argsort(-1)
            some = torch.rand(n, kv, case["cap"], generator=g, device="cuda") < 0.7
            pos = torch.where(some, pos.expand(n, kv, -1), pos[swap])
            v["pos"] = _wide(pos, case, 0)
            v["next"] = v["lens"] * 2
    elif kind == "compact":
        v["weight"] = _wide(_weights(g, case), case, 0.0)
        pos = torch.arange(case["cap"], device="cuda", dtype=torch.int32).expand(n, kv, -1)
        v["pos"] = _wide(pos, case, 0)
        score = torch.rand(n, kv, case["cap"], generator=g, device="cuda")
        v["src"] = _pairs(score, v["lens"], case["budget"])
    return v


# ------------------------------------------------------------ plain forms ---
def _pairs(key, lens, budget):
    """src [n][kv][budget]: the entry that each slot below the budget holds
    after the `budget` highest of key[..., :len] are kept (ties to the lowest
    index): its own, or the next one kept from behind; -1 past the length."""
    n, kv, cap = key.shape
    at = torch.arange(cap, device="cuda")
    held = at < lens[:, None, None]
    key = torch.where(held, key.float(), torch.full_like(key, -math.inf))
    order = torch.sort(key, dim=-1, descending=True, stable=True).indices
    m = min(budget, cap)
    keep = torch.zeros(n, kv, cap, device="cuda", dtype=torch.bool)
    keep.scatter_(-1, order[..., :m], True)
    keep &= held
    below = torch.arange(m, device="cuda").expand(n, kv, m)
    hole = ~keep[..., :m] & held[..., :m]
    tail = torch.sort((~keep[..., m:]).to(torch.uint8), dim=-1, stable=True).indices + m
    if tail.shape[-1]:
        rank = (hole.cumsum(-1) - 1).clamp(0, tail.shape[-1] - 1)
        below = torch.where(hole, tail.gather(-1, rank), below)
    src = torch.where(held[..., :m].expand(n, kv, m), below, torch.full_like(below, -1))
    return torch.nn.functional.pad(src, (0, budget - m), value=-1).to(torch.int32).contiguous()


def _e4m3(x):
    """Codes (as float8 values) and scales [..., 1] of rows of x: the scale is
    the row's largest magnitude over 240, at least 2^-96, 1 for a row of zeros;
    values round to the nearest code, ties away from zero, and those below the
    least normal one are zero."""
    # (64 bits: 32 would put values next to a tie between codes on its other side)
    s = (x.abs().amax(-1, keepdim=True).double() / 240.0).float()
    s = torch.where(s == 0, torch.ones_like(s), s.clamp(min=2.0 ** -96))
    v = (x.double() / s.double()).float()
    bits = v.abs().contiguous().view(torch.int32)
    field = (bits >> 20) + ((bits >> 19) & 1) - (120 << 3)
    mag = ((field << 20) + (120 << 23)).view(torch.float32)
    # the least normal code is 2^-6; magnitudes below it are decoded as zero
    mag = torch.where((bits >> 23) >= 121, mag, torch.zeros_like(mag))
    return (mag * torch.sign(v)).to(torch.float8_e4m3fn), s


def _store(x, dtype):
    """Rows as a cache holds them: values, and scales for E4M3."""
    if dtype == "e4m3":
        return _e4m3(x)
    return (x.bfloat16() if dtype == "bf16" else x), None


def _slots(table, page, at):
    """Pool rows of entries `at` [n][m] of every sequence."""
    return table.long().gather(1, at // page) * page + at % page


def _plain_append(st):
    case, n, r = st["case"], st["case"]["nseq"], st["case"]["rows"]
    i = torch.arange(r, device="cuda").expand(n, r)
    ok = i < st["counts"][:, None]
    at = torch.where(ok, st["lens"][:, None] + i, st["lens"][:, None].long())
    slot = _slots(st["table"], case["page"], at)
    which, back = slot[ok], []
    for name in ("k", "v"):
        val, s = _store(st[name], case["dtype"])
        pool = st["pool_" + name]
        if s is None:
            pool[which] = val[ok]
            back.append(_by_page(pool, case))
        else:
            pool.view(torch.uint8)[which] = val.view(torch.uint8)[ok]
            st["scale_" + name][which] = s[ok]
            got = pool[slot].float() * st["scale_" + name][slot]
            back.append(torch.where(ok[:, :, None, None], got, torch.zeros_like(got)))
    return back


def _gather(st, name, at):
    """Entries at [n][m] in fp32: [n][kv][m][hd]."""
    slot = _slots(st["table"], st["case"]["page"], at)
    x = st["pool_" + name][slot].float()
    if st["case"]["dtype"] == "e4m3":
        x = x * st["scale_" + name][slot]
    return x.permute(0, 2, 1, 3).contiguous()


def _slopes(heads, dtype):
    j = torch.arange(1, heads + 1, device="cuda", dtype=torch.float64)
    return torch.exp2(-8.0 * j / heads).to(dtype)


def _plain_attend(st):
    case = st["case"]
    n, H, kv, hd, cap = (case[x] for x in ("nseq", "heads", "kv", "hd", "cap"))
    at = torch.arange(cap, device="cuda")
    lens = st["lens"][:, None]
    held = at < lens
    ahead = lens - 1 - at  # distance of the query from an entry
    seen = held & (ahead < case["window"]) if case["window"] else held
    k = _gather(st, "k", torch.where(held, at, torch.zeros_like(at)))
    q = st["q"].view(n, kv, H // kv, hd)
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * (1.0 / math.sqrt(hd))
    del k
    if case["alibi"]:
        slope = _slopes(H, torch.float32).view(1, kv, H // kv, 1)
        s = s - slope * ahead.float()[:, None, None, :]
    s = s.masked_fill(~seen[:, None, None, :], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - top)
    total = p.sum(-1, keepdim=True)
    p, lse = p / total, (top + torch.log(total)).reshape(n, H)
    v = _gather(st, "v", torch.where(held, at, torch.zeros_like(at)))
    out = torch.matmul(p, v).reshape(n, H * hd)
    if not case["track"]:
        return [out, lse]
    st["weight"][..., :cap] += p.sum(2)
    return [out, lse, st["weight"]]


def _plain_choose(st):
    case = st["case"]
    at = torch.arange(case["cap"], device="cuda")
    pos = st["pos"][..., :case["cap"]] if "pos" in st else at.expand(case["nseq"], case["kv"], -1)
    end = st["next"] if "next" in st else st["lens"]
    first = (pos < case["sinks"]) | (pos >= end[:, None, None] - case["recent"])
    w = st["weight"][..., :case["cap"]]
    return [_pairs(torch.where(first, torch.full_like(w, math.inf), w), st["lens"], case["budget"])]


def _plain_compact(st):
    case, src = st["case"], st["src"].long()
    n, kv, m = src.shape
    m = min(m, case["cap"])
    src = src[..., :m]
    at = torch.arange(m, device="cuda").expand(n, kv, m)
    b, h, j = torch.nonzero((src >= 0) & (src != at), as_tuple=True)
    s = src[b, h, j]
    slots = [_slots_of(st["table"], case["page"], b, e) for e in (s, j)]
    for name in ("k", "v"):
        pool = st["pool_" + name]
        raw = pool.view(torch.uint8) if case["dtype"] == "e4m3" else pool
        raw[slots[1], h] = raw[slots[0], h]
        if case["dtype"] == "e4m3":
            st["scale_" + name][slots[1], h] = st["scale_" + name][slots[0], h]
    for name in ("weight", "pos"):
        st[name][b, h, j] = st[name][b, h, s]
    out = [st["weight"], st["pos"]]
    if case["dtype"] == "e4m3":
        every = torch.arange(m, device="cuda").expand(n, m)
        ok = (every < st["lens"][:, None])[:, :, None, None]
        for name in ("k", "v"):
            x = _gather(st, name, every).transpose(1, 2)
            out.append(torch.where(ok, x, torch.zeros_like(x)))
        return out
    return out + [_by_page(st["pool_" + name], case) for name in ("k", "v")]


def _slots_of(table, page, b, e):
    return table[b, e // page].long() * page + e % page


def _by_page(pool, case):
    return pool.view(-1, case["page"], case["kv"], case["hd"])


# --------------------------------------------------------------- prepare ---
_STREAM = None


def _stream():
    """The one stream that a program queues its passes on."""
    global _STREAM
    if _STREAM is None:
        _STREAM = torch.cuda.Stream()
    return _STREAM.cuda_stream


def _binding():
    # the binding lives in a folder whose name is no Python package name
    path = os.path.join(os.getcwd(), "welvet.cuda_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import pywelvet

    return pywelvet


class _Raw:
    """Device memory of the cache as torch sees it. A tensor made of this keeps
    it, and it keeps the cache: the memory lives as long as the tensor does."""

    def __init__(self, cache, ptr, shape, typestr):
        self.cache = cache
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": shape, "strides": None,
                                         "typestr": typestr, "version": 2}


def _pool_view(case, cache, ptr, pages):
    """The pool as [page][entry][kv][hd] in the cache's type (F32 and BF16)."""
    pitch = cache.buffers().pitch
    shape = (pages, case["kv"], case["page"], pitch)
    t = torch.as_tensor(_Raw(cache, ptr, shape, "<f4" if case["dtype"] == "f32" else "<i2"), device="cuda")
    t = t if case["dtype"] == "f32" else t.view(torch.bfloat16)
    return t[..., :case["hd"]].permute(0, 2, 1, 3)


def prepare(case, seed):
    v = _inputs(case, seed)
    st = {"case": dict(case), **{x: t for x, t in v.items() if x not in ("k", "v")}}
    kind, n = case["kind"], case["nseq"]
    if kind == "append":
        st["k"], st["v"] = v["k"], v["v"]
    if not own:
        if kind == "choose":
            return st
        page, slots = case["page"], v["pool_pages"] * case["page"]
        dt = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.uint8}[case["dtype"]]
        for name in ("k", "v"):
            pool = torch.zeros(slots, case["kv"], case["hd"], device="cuda", dtype=dt)
            if case["dtype"] == "e4m3":
                pool = pool.view(torch.float8_e4m3fn)
                st["scale_" + name] = torch.ones(slots, case["kv"], 1, device="cuda")
            if kind != "append":
                at = torch.arange(case["cap"], device="cuda").expand(n, -1)
                ok = at < v["lens"][:, None]
                which = _slots(v["table"], page, at)[ok]
                val, s = _store(v[name], case["dtype"])
                if s is None:
                    pool[which] = val[ok]
                else:
                    pool.view(torch.uint8)[which] = val.view(torch.uint8)[ok]
                    st["scale_" + name][which] = s[ok]
            st["pool_" + name] = pool
        return st
    pw = _binding()
    st["stream"], page = _stream(), case.get("page", 16)
    table = v["table"]
    st["cache"] = cache = pw.KVCache(
        DTYPES[case.get("dtype", "bf16")], v.get("pool_pages", 1), page, case["heads"], case["kv"],
        case.get("hd", 16), n, table.shape[1])

    def ptr(name):
        return st[name].data_ptr() if name in st else None

    st["seqs"] = pw.KVSeqs(n, table.data_ptr(), v["lens"].data_ptr(), ptr("next"), ptr("pos"),
                           ptr("weight"))
    zero = torch.zeros_like(v["lens"])
    torch.cuda.synchronize()  # the inputs were made on another stream than the calls' own
    if kind in ("attend", "compact"):
        cache.append(pw.KVSeqs(n, table.data_ptr(), zero.data_ptr()), case["cap"],
                     v["k"].data_ptr(), v["v"].data_ptr(), v["lens"].data_ptr(), stream=st["stream"])
        torch.cuda.synchronize()
    if kind == "attend":
        st["out"] = torch.empty(n, case["heads"] * case["hd"], device="cuda")
        st["lse"] = torch.empty(n, case["heads"], device="cuda")
    elif kind == "choose":
        st["src"] = torch.empty(n, case["kv"], case["budget"], device="cuda", dtype=torch.int32)
    elif case["dtype"] == "e4m3":
        m = case["rows"] if kind == "append" else min(case["budget"], case["cap"])
        st["back"] = [torch.empty(n, m, case["kv"], case["hd"], device="cuda") for _ in range(2)]
        st["read_first"] = v["lens"] if kind == "append" else None
        st["read_count"] = v["counts"] if kind == "append" else v["lens"]
    else:
        b = cache.buffers()
        st["pools"] = [_pool_view(case, cache, p, v["pool_pages"]) for p in (b.k, b.v)]
    return st


# ------------------------------------------------------------------- run ---
def run(st):
    kind = st["case"]["kind"]
    if not own:
        return {"append": _plain_append, "attend": _plain_attend, "choose": _plain_choose,
                "compact": _plain_compact}[kind](st)
    case, cache, seqs, q = st["case"], st["cache"], st["seqs"], st["stream"]
    if kind == "append":
        cache.append(seqs, case["rows"], st["k"].data_ptr(), st["v"].data_ptr(),
                     st["counts"].data_ptr(), stream=q)
    elif kind == "attend":
        cache.attend(seqs, st["q"].data_ptr(), st["out"].data_ptr(), window=case["window"],
                     alibi=case["alibi"], lse=st["lse"].data_ptr(), stream=q)
        return [st["out"], st["lse"]] + ([st["weight"]] if case["track"] else [])
    elif kind == "choose":
        cache.choose(seqs, case["budget"], case["sinks"], case["recent"], st["src"].data_ptr(),
                     stream=q)
        return [st["src"]]
    else:
        cache.compact(seqs, case["budget"], st["src"].data_ptr(), stream=q)
    own_state = [st["weight"], st["pos"]] if kind == "compact" else []
    if case["dtype"] != "e4m3":
        return own_state + st["pools"]
    k, v = st["back"]
    first, count = st["read_first"], st["read_count"]
    cache.read(seqs, k.shape[1], k.data_ptr(), v.data_ptr(),
               None if first is None else first.data_ptr(), count.data_ptr(), stream=q)
    return own_state + st["back"]


# ----------------------------------------------------------------- exact ---
def _value64(x, dtype):
    """What a cache's entry stands for, in 64 bits."""
    x = x.double()
    if dtype == "f32":
        return x
    if dtype == "bf16":
        return x.float().bfloat16().double()
    s = (x.abs().amax(-1, keepdim=True) / 240.0).float().double().clamp(min=2.0 ** -96)
    m, e = torch.frexp((x / s).float().double().abs())
    # four significant bits, half away from zero; below 2^-6 zero
    r = torch.floor(m * 16.0 + 0.5) / 16.0 * torch.exp2(e.double())
    r = torch.where(m * torch.exp2(e.double()) < 2.0 ** -6, torch.zeros_like(r), r)
    return r * torch.sign(x) * s


def _exact_append(case, v):
    """The entries read back (E4M3), or the pool that they were written to."""
    n, r, out = case["nseq"], case["rows"], []
    ok = torch.arange(r, device="cuda") < v["counts"][:, None]
    at = v["lens"][:, None] + torch.arange(r, device="cuda")
    for name in ("k", "v"):
        x = _value64(v[name], case["dtype"]) * ok[:, :, None, None]
        if case["dtype"] != "e4m3":
            pool = torch.zeros(v["pool_pages"], case["page"], case["kv"], case["hd"], device="cuda",
                               dtype=torch.float64)
            b = torch.arange(n, device="cuda")[:, None].expand(n, r)[ok]
            e = at[ok]
            pool[v["table"][b, e // case["page"]].long(), e % case["page"]] = x[ok]
            x = pool
        out.append(x)
    return out


def _exact_compact(case, v):
    """Every sequence's entries in their order after the moves."""
    n, kv, page = case["nseq"], case["kv"], case["page"]
    src = v["src"].long()[..., :case["cap"]]
    m = src.shape[-1]
    now = torch.arange(case["cap"], device="cuda").repeat(n, kv, 1)
    now[..., :m] = torch.where(src >= 0, src, now[..., :m])
    out = [v["weight"].double(), None]  # (the positions are whole numbers)
    out[0][..., :case["cap"]] = out[0].gather(-1, now)
    held = torch.arange(case["cap"], device="cuda") < v["lens"][:, None]
    for name in ("k", "v"):
        x = _value64(v[name], case["dtype"]) * held[:, :, None, None]
        x = x.gather(1, now.transpose(1, 2)[..., None].expand_as(x))
        if case["dtype"] == "e4m3":
            out.append(x[:, :m])
            continue
        pool = torch.zeros(v["pool_pages"] * page, kv, case["hd"], device="cuda", dtype=torch.float64)
        b, e = torch.nonzero(held, as_tuple=True)
        pool[v["table"][b, e // page].long() * page + e % page] = x[b, e]
        out.append(pool.view(-1, page, kv, case["hd"]))
    return out


def exact(case, seed):
    if case["kind"] == "choose":
        return None  # whole numbers
    v = _inputs(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, v)
    if case["kind"] == "compact":
        return _exact_compact(case, v)
    n, H, kv, hd = (case[x] for x in ("nseq", "heads", "kv", "hd"))
    group = H // kv
    out = torch.zeros(n, H, hd, device="cuda", dtype=torch.float64)
    lse = torch.zeros(n, H, device="cuda", dtype=torch.float64)
    weight = v["weight"].double() if case["track"] else None
    slope = torch.tensor([2.0 ** (-8.0 * (j + 1) / H) for j in range(H)], device="cuda",
                         dtype=torch.float64)
    for b, length in enumerate(_lens(case)):
        lo = max(0, length - case["window"]) if case["window"] else 0
        back = torch.arange(length - 1 - lo, -1, -1, device="cuda", dtype=torch.float64)
        for h in range(kv):
            K = _value64(v["k"][b, lo:length, h], case["dtype"])
            V = _value64(v["v"][b, lo:length, h], case["dtype"])
            j = slice(h * group, (h + 1) * group)
            s = (K @ v["q"][b, j].double().T.contiguous()).T / math.sqrt(hd)
            if case["alibi"]:
                s = s - slope[j, None] * back
            p = torch.softmax(s, 1)
            out[b, j], lse[b, j] = p @ V, torch.logsumexp(s, 1)
            if weight is not None:
                weight[b, h, lo:length] += p.sum(0)
    return [out.view(n, H * hd), lse] + ([weight] if weight is not None else [])
