"""The paged KV cache held in 8 bits (gmoe_kv_create_q8, gmoe_kv_append, gmoe_kv_read,
gmoe_kv_truncate and gmoe_attention over it) against the float64 restatement in
oracle/attention8.py: head layouts and widths, block and page borders, prompts and decode
steps in any cut, windows, refusals, non-finite input, streams, and a run of them together."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

import garuda_amd as G
from garuda_amd.attention import KvCache
from oracle.attention8 import BLOCK, Kv8Oracle
from tests.test_gpu_dense import _hip
from tests.test_gpu_parity import bits, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    d = G.Device(0, slab_bytes=64 << 20)
    yield d
    d.close()


class Gpu:
    """Device buffers and a stream of the caller's, through the runtime that the library links."""

    def __init__(self):
        self.hip, self.bufs, self.st = _hip(), [], C.c_void_p()
        assert self.hip.hipStreamCreate(C.byref(self.st)) == 0
        self.stream = self.st.value

    def empty(self, nbytes):
        b = C.c_void_p()
        assert self.hip.hipMalloc(C.byref(b), nbytes) == 0
        self.bufs.append(b)
        return b.value

    def up(self, x):
        at = self.empty(x.nbytes)
        assert self.hip.hipMemcpy(at, x.ctypes.data, x.nbytes, 1) == 0
        return at

    def down(self, at, shape):
        x = np.empty(shape, np.float32)
        assert self.hip.hipMemcpy(x.ctypes.data, at, x.nbytes, 2) == 0
        return x

    def wait(self):
        assert self.hip.hipStreamSynchronize(self.st) == 0

    def __enter__(self):
        return self

    def __exit__(self, *a):
        self.hip.hipStreamSynchronize(self.st)
        self.hip.hipStreamDestroy(self.st)
        for b in self.bufs:
            self.hip.hipFree(b)


def draw(rng, n, nh, nkv, hd):
    return tuple(rng.normal(size=(n, w * hd)).astype(np.float32) for w in (nh, nkv, nkv))


def check(got, want, mag, span, hd, vmax, what):
    """A score is a sum of hd products, each of a query element held to 2^-22 of the head's largest (twice, for the pair's
    two roundings) and summed in f32: off by at most (hd + 8) 2^-23 of its products' magnitudes, plus two
    roundings of its own. A weight is off by that (relative), and its exponential by 2^-21; the mean by
    twice the weights' errors and 2^-24 a term, of the largest value."""
    ds = (hd + 10) * 2.0 ** -23 * max(mag, 1.0)
    bound = vmax * (2 * ds + 2.0 ** -20 + min(span, 4096) * 2.0 ** -24)
    err = np.abs(got - want)
    assert np.isfinite(got).all() and err.max() <= bound, f"{what}: max err {err.max():.3g}, bound {bound:.3g}"


def precise(got, want, what):
    """In the 2-norm, for scores of order 1 to 10: a score of up to 16 (in base 2) is rounded to 2^-21 a few
    times, and everything else is smaller."""
    rel = np.linalg.norm(got - want) / np.linalg.norm(want)
    assert rel < 2e-6, f"{what}: {rel:.3g}"


def run(kv, o, layer, seqs, qkv, what):
    q, k, v = qkv
    say(what)
    got = kv.attention(layer, seqs, q, k, v)
    want, mag = o.attention(layer, seqs, q, k, v)
    span = max(o.seq_len(int(s), layer) for s in seqs)
    vmax = max(np.abs(o.of(int(s), layer).given[1]).max() for s in seqs)
    check(got, want, mag, span, kv.hd, vmax, what)
    precise(got, want, what)


def same_rows(kv, o, layer, seqs, what):
    for s in set(int(s) for s in seqs):
        n = kv.seq_len(s, layer)
        assert n == o.seq_len(s, layer), what
        if n:
            got, want = (c.read(layer, [s] * n, range(n)) for c in (kv, o))
            for g, w, name in zip(got, want, ("keys", "values")):
                assert np.array_equal(g, w), f"{what}: {name} of sequence {s} differ at {np.argwhere(g != w)[:3]}"


HEADS = [(8, 2, 64), (32, 8, 128), (4, 4, 32), (16, 1, 128), (8, 1, 256), (12, 4, 80), (6, 2, 96), (3, 1, 20), (2, 1, 4),
         (5, 5, 36), (32, 2, 192), (7, 1, 132), (2, 2, 252)]


@pytest.mark.parametrize("nh,nkv,hd", HEADS)
def test_steps_and_prompts_of_every_head_layout(dev, nh, nkv, hd):
    rng = np.random.default_rng(hd + nh)
    kw = dict(max_positions=400, rope_theta=1e4)
    with KvCache(dev, 2, nh, nkv, hd, block_size=16, max_seqs=3, bits=8, **kw) as kv:
        o = Kv8Oracle(2, nh, nkv, hd, **kw)
        seqs = [kv.open_seq() for _ in range(3)]
        mk = lambda n: draw(rng, n, nh, nkv, hd)
        run(kv, o, 1, [seqs[0]] * 21, mk(21), f"{nh}/{nkv}/{hd}: prompt of 21")
        run(kv, o, 1, [seqs[1]] * 150 + [seqs[2]] * 16, mk(166), f"{nh}/{nkv}/{hd}: prompts of 150 and 16")
        for step in range(14):
            run(kv, o, 1, seqs, mk(3), f"{nh}/{nkv}/{hd}: step {step}")
        run(kv, o, 1, [seqs[0]] * 3 + [seqs[2]] * 2, mk(5), f"{nh}/{nkv}/{hd}: drafts")
        same_rows(kv, o, 1, seqs, "after")
        assert kv.seq_len(seqs[0], 0) == 0


def in_tiles(nh, nkv, hd, spans, window=0):
    """Whether a call of runs (start, end) of 160 rows or more goes in tiles: as groups of 16 rows and splits of
    their spans it would make more than 1536 workgroups, of heads wider than 128 more than 512."""
    g = nh // nkv
    assert all((e - s) * g >= 160 for s, e in spans)
    first = [max(0, e - window) // BLOCK * BLOCK if window else 0 for _, e in spans]
    wgs = sum(-(-(e - s) // (16 // g)) * (1 + -(-((e - 1) // BLOCK * BLOCK - f) // 512)) * nkv for (s, e), f in zip(spans, first))
    return wgs > (1536 if hd <= 128 else 512)


@pytest.mark.parametrize("nh,nkv,hd,bs,window,sizes", [
    (8, 2, 64, 16, 0, [300] * 8), (32, 8, 128, 16, 0, [150, 400]), (4, 4, 32, 32, 0, [520] * 8),
    (16, 1, 128, 16, 0, [600, 500]), (12, 4, 80, 16, 100, [330] * 4), (6, 2, 96, 48, 0, [440] * 6),
    (3, 1, 20, 16, 0, [650] * 8), (7, 1, 36, 16, 33, [700] * 3), (32, 32, 4, 16, 1, [790]), (32, 8, 112, 16, 16, [170, 360]),
    (8, 1, 256, 16, 0, [500, 500, 300]), (4, 2, 160, 32, 50, [440] * 6), (16, 16, 192, 16, 0, [530]),
    (5, 1, 252, 16, 0, [650] * 3), (12, 3, 132, 16, 1, [300] * 6),
])
def test_prompts_in_tiles(dev, nh, nkv, hd, bs, window, sizes):
    # prompts from their beginning, then more of each from an odd position, beside a step of another
    rng = np.random.default_rng(nh * hd)
    kw = dict(max_positions=2 * max(sizes), sliding_window=window)
    with KvCache(dev, 1, nh, nkv, hd, block_size=bs, max_seqs=len(sizes) + 1, bits=8, **kw) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, **kw)
        seqs = [kv.open_seq() for _ in sizes]
        other = kv.open_seq()
        for call, add in enumerate((0, -37)):
            spans = [(o.seq_len(s), o.seq_len(s) + n + add) for s, n in zip(seqs, sizes)]
            assert in_tiles(nh, nkv, hd, spans, window) or call
            ids = [s for s, (a, b) in zip(seqs, spans) for _ in range(b - a)] + [other] * call
            q, k, v = draw(rng, len(ids), nh, nkv, hd)
            what = f"tiles {nh}/{nkv}/{hd} bs {bs} window {window}, call {call}"
            say(what)
            got = kv.attention(0, ids, q, k, v)
            o.append(0, ids, k, v)
            at = 0
            for s, (a, b) in zip(seqs + [other] * call, spans + [(0, 1)]):
                mine = slice(at, at + b - a)
                want, mag = o.attend_run(0, s, a, q[mine])
                check(got[mine], want, mag, b, hd, np.abs(v).max() + 5, what)
                precise(got[mine], want, what)
                at += b - a
        same_rows(kv, o, 0, seqs + [other], "tiles")


@pytest.mark.parametrize("bs,window", [(16, 0), (32, 0), (64, 7), (16, 16), (16, 1), (48, 100), (16, 250)])
def test_pages_and_windows(dev, bs, window):
    nh, nkv, hd = 8, 2, 64
    rng = np.random.default_rng(bs + window)
    kw = dict(max_positions=640, sliding_window=window)
    with KvCache(dev, 1, nh, nkv, hd, block_size=bs, max_seqs=2, bits=8, **kw) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, **kw)
        a, b = kv.open_seq(), kv.open_seq()
        mk = lambda n: draw(rng, n, nh, nkv, hd)
        run(kv, o, 0, [a] * 300 + [b] * 5, mk(305), f"bs {bs} window {window}: prompts")
        for step in range(40):
            run(kv, o, 0, [a, b], mk(2), f"bs {bs} window {window}: step {step}")
        run(kv, o, 0, [b] * 70, mk(70), f"bs {bs} window {window}: prompt of 70 at 45")
        same_rows(kv, o, 0, [a, b], "after")


def test_long_spans_join_their_splits(dev):
    # several thousand positions: many splits of the keys, one sequence long and one short
    nh, nkv, hd = 8, 2, 64
    rng = np.random.default_rng(5)
    with KvCache(dev, 1, nh, nkv, hd, block_size=64, max_positions=6000, max_seqs=2, bits=8) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, max_positions=6000)
        a, b = kv.open_seq(), kv.open_seq()
        k, v = (rng.normal(size=(4990, nkv * hd)).astype(np.float32) for _ in range(2))
        kv.append(0, [a] * 4990, k, v)
        o.append(0, [a] * 4990, k, v)
        for step in range(4):
            run(kv, o, 0, [a, b], draw(rng, 2, nh, nkv, hd), f"long spans, step {step}")
        run(kv, o, 0, [a] * 40 + [b], draw(rng, 41, nh, nkv, hd), "long spans, prompt beside a step")
        # 320 tokens in tiles, their keys in many splits, the own blocks by themselves
        assert in_tiles(nh, nkv, hd, [(5034, 5354)])
        q, k, v = draw(rng, 321, nh, nkv, hd)
        got = kv.attention(0, [b] + [a] * 320, q, k, v)
        o.append(0, [b] + [a] * 320, k, v)
        want, mag = o.attend_run(0, a, 5034, q[1:])
        check(got[1:], want, mag, 5354, hd, 6.0, "long spans, tiles")
        precise(got[1:], want, "long spans, tiles")


@pytest.mark.parametrize("order", ["interleaved", "mixed", "twice"])
def test_entries_in_any_order(dev, order):
    nh, nkv, hd = 8, 2, 32
    rng = np.random.default_rng(7)
    with KvCache(dev, 1, nh, nkv, hd, max_positions=300, max_seqs=4, bits=8) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, max_positions=300)
        s = [kv.open_seq() for _ in range(4)]
        ids = {"interleaved": [s[0], s[1]] * 40, "mixed": [s[2]] + [s[0]] * 60 + [s[1]] + [s[3]] * 7 + [s[0]] * 30,
               "twice": [s[0], s[1], s[2], s[1]]}[order]
        for call in range(3):
            run(kv, o, 0, ids, draw(rng, len(ids), nh, nkv, hd), f"{order} {call}")
        same_rows(kv, o, 0, s, order)


@pytest.mark.parametrize("n", [64, 65, 130])
def test_wide_decode_batches(dev, n):
    # more sequences than ride in the kernel arguments
    nh, nkv, hd = 4, 1, 32
    rng = np.random.default_rng(n)
    with KvCache(dev, 1, nh, nkv, hd, max_positions=64, max_seqs=n, bits=8) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, max_positions=64)
        seqs = [kv.open_seq() for _ in range(n)]
        for i, s in enumerate(seqs):
            if i % 20:
                k, v = draw(rng, i % 20, nh, nkv, hd)[1:]
                kv.append(0, [s] * (i % 20), k, v)
                o.append(0, [s] * (i % 20), k, v)
        for step in range(3):
            run(kv, o, 0, seqs, draw(rng, n, nh, nkv, hd), f"batch of {n}, step {step}")
        same_rows(kv, o, 0, seqs, "batch")


def test_a_step_does_not_depend_on_its_batch(dev):
    nh, nkv, hd = 8, 2, 128
    rng = np.random.default_rng(8)
    with KvCache(dev, 1, nh, nkv, hd, max_positions=2000, max_seqs=9, bits=8) as kv:
        seqs = [kv.open_seq() for _ in range(9)]
        k, v = (rng.normal(size=(1500, nkv * hd)).astype(np.float32) for _ in range(2))
        for s in seqs:
            kv.append(0, [s] * 1500, k, v)
        q, k, v = draw(rng, 1, nh, nkv, hd)
        alone = kv.attention(0, seqs[:1], q, k, v)
        rep = lambda x: np.repeat(x, 8, 0)
        many = kv.attention(0, seqs[1:], rep(q), rep(k), rep(v))
        assert all(np.array_equal(bits(m), bits(alone[0])) for m in many)


@pytest.mark.parametrize("bits_", [32, 8])
def test_append_leaves_the_cache_as_attention_does(dev, bits_):
    nh, nkv, hd = 4, 2, 64
    rng = np.random.default_rng(9)
    with KvCache(dev, 1, nh, nkv, hd, max_positions=200, max_seqs=2, bits=bits_) as A, \
            KvCache(dev, 1, nh, nkv, hd, max_positions=200, max_seqs=2, bits=bits_) as B:
        a, b = A.open_seq(), B.open_seq()
        for n in (1, 20, 3, 70, 9, 1):
            q, k, v = draw(rng, n, nh, nkv, hd)
            A.attention(0, [a] * n, q, k, v)
            B.append(0, [b] * n, k, v)
        n = A.seq_len(a)
        assert n == B.seq_len(b) == 104 and A.free_pages() == B.free_pages()
        for x, y in zip(A.read(0, [a] * n, range(n)), B.read(0, [b] * n, range(n))):
            assert np.array_equal(bits(x), bits(y))
        q, k, v = draw(rng, 1, nh, nkv, hd)
        assert np.array_equal(bits(A.attention(0, [a], q, k, v)), bits(B.attention(0, [b], q, k, v)))


@pytest.mark.parametrize("bits_,bs", [(32, 5), (32, 100), (8, 16), (8, 64)])
def test_read_in_any_order(dev, bits_, bs):
    nkv, hd = 2, 36
    rng = np.random.default_rng(10)
    with KvCache(dev, 1, 4, nkv, hd, block_size=bs, max_positions=300, max_seqs=2, bits=bits_) as kv:
        a, b = kv.open_seq(), kv.open_seq()
        for s, n in ((a, 211), (b, 37)):
            kv.append(0, [s] * n, *draw(rng, n, 4, nkv, hd)[1:])
        ids = np.array([a] * 211 + [b] * 37)
        pos = np.concatenate([np.arange(211), np.arange(37)])
        k, v = kv.read(0, ids, pos)
        if bits_ == 32:  # the values as they were given
            assert np.isfinite(k).all() and np.abs(v).max() > 1
        at = rng.integers(0, ids.size, 700)  # rows several times
        k2, v2 = kv.read(0, ids[at], pos[at])
        assert np.array_equal(k2, k[at]) and np.array_equal(v2, v[at])


@pytest.mark.parametrize("bits_", [32, 8])
def test_truncate(dev, bits_):
    nh, nkv, hd = 4, 2, 64
    rng = np.random.default_rng(11)
    with KvCache(dev, 2, nh, nkv, hd, block_size=16, max_positions=200, max_seqs=3, bits=bits_) as kv:
        o = Kv8Oracle(2, nh, nkv, hd, max_positions=200) if bits_ == 8 else None
        s = [kv.open_seq() for _ in range(3)]
        free = kv.free_pages()

        def put(layer, ids):
            q, k, v = draw(rng, len(ids), nh, nkv, hd)
            if o:
                run(kv, o, layer, ids, (q, k, v), f"truncate: {len(ids)} tokens")
            else:
                kv.attention(layer, ids, q, k, v)

        def cut(ids, lens):
            kv.truncate(ids, lens)
            if o:
                o.truncate(ids, lens)
                for l in range(2):
                    same_rows(kv, o, l, s, f"cut to {lens}")

        for l in range(2):
            put(l, [s[0]] * 100 + [s[1]] * 30)
        assert kv.free_pages() == free - 2 * (7 + 2)
        cut([s[0], s[1]], [98, 40])           # inside the last block; longer than it is: stays
        put(0, [s[0]] * 2 + [s[1]])
        cut([s[0]], [41])                     # into an earlier block
        assert kv.free_pages() == free - 2 * (3 + 2)
        put(0, [s[0]] * 3)                    # layer 0: 44, layer 1: 41
        put(1, [s[0]] * 30)
        cut([s[0], s[0], s[1]], [60, 33, 16])  # one sequence twice, and to a block's start
        cut([s[1], s[2]], [5, 0])
        for l in range(2):
            put(l, s)
            put(l, [s[1]] * 50)
        cut([s[0], s[1], s[2]], [0, 0, 0])
        assert kv.free_pages() == free and kv.seq_len(s[0]) == 0
        put(0, s)


def test_truncate_restores_more_sequences_than_one_launch_takes(dev):
    nkv, hd, n = 1, 8, 70
    rng = np.random.default_rng(12)
    with KvCache(dev, 2, 2, nkv, hd, max_positions=64, max_seqs=n, bits=8) as kv:
        o = Kv8Oracle(2, 2, nkv, hd, max_positions=64)
        s = [kv.open_seq() for _ in range(n)]
        for l in range(2):
            ids = [x for x in s for _ in range(33)]
            k, v = draw(rng, len(ids), 2, nkv, hd)[1:]
            kv.append(l, ids, k, v)
            o.append(l, ids, k, v)
        lens = [3 + i % 13 for i in range(n)]
        kv.truncate(s, lens)
        o.truncate(s, lens)
        for l in range(2):
            same_rows(kv, o, l, s, "restored")
            run(kv, o, l, s, draw(rng, n, 2, nkv, hd), "after")


@pytest.mark.parametrize("tiles", [0, 8, 132], ids=["rows", "tiles", "tiles-wide"])
@pytest.mark.parametrize("what", ["nan_k", "inf_k", "nan_v", "nan_q", "inf_q", "huge_q", "huge_k", "zero", "tiny", "scales"])
def test_unusual_values(dev, what, tiles):
    """Non-finite input stands for NaN in its block; uniform weights where a score is not below +inf;
    values of very different size from block to block, and none but zeros."""
    nh, nkv, hd = (32, 32, tiles) if tiles else (4, 2, 32)
    assert not tiles or in_tiles(nh, nkv, hd, [(22, 562)])
    rng = np.random.default_rng(13)
    with KvCache(dev, 1, nh, nkv, hd, max_positions=700, max_seqs=1, bits=8) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, max_positions=700)
        s = kv.open_seq()
        for call, n in enumerate((20, 1, 1, 540 if tiles else 60, 1, 15, 1, 1)):
            q, k, v = draw(rng, n, nh, nkv, hd)
            if what == "zero":
                k[:], v[:] = 0, 0
            elif what == "tiny":
                k, v = k * np.float32(1e-30), v * np.float32(1e-30)
            elif what == "huge_k":
                k, q = k * np.float32(1e30), q * np.float32(1e-30)
            elif what == "scales":
                v *= np.float32(10.0) ** rng.integers(-3, 4)
                k *= np.float32(2.0) ** rng.integers(-3, 2)
            elif call == 3:
                x = {"nan_k": k, "inf_k": k, "nan_v": v, "nan_q": q, "inf_q": q, "huge_q": q}[what]
                x[7, 5] = {"nan": np.nan, "inf": np.inf, "huge": 3e38}[what[:-2]]
                if what == "huge_q":
                    x[7] = 3e38  # scores beyond f32
            say(f"{what}, call {call}")
            got = kv.attention(0, [s] * n, q, k, v)
            want, mag = o.attention(0, [s] * n, q, k, v)
            fine = np.isfinite(want)
            assert np.array_equal(np.isnan(got), np.isnan(want)), what
            if fine.any():
                vmax = np.nanmax(np.abs(np.where(np.isfinite(o.of(s, 0).given[1]), o.of(s, 0).given[1], 0)))
                check(got[fine], want[fine], mag, o.seq_len(s), hd, vmax, what)
        n = kv.seq_len(s)
        for g, w in zip(kv.read(0, [s] * n, range(n)), o.read(0, [s] * n, range(n))):
            assert np.array_equal(g, w, equal_nan=True)


def test_refusals_change_nothing(dev):
    nh, nkv, hd = 4, 2, 16
    rng = np.random.default_rng(14)
    mk = lambda n: draw(rng, n, nh, nkv, hd)
    with pytest.raises(G.ModelError):
        KvCache(dev, 1, nh, nkv, hd, block_size=8, bits=8)
    with pytest.raises(G.ModelError):
        KvCache(dev, 1, nh, nkv, 260, bits=8)
    with pytest.raises(G.ModelError):
        KvCache(dev, 1, 34, 2, hd, bits=8)
    for bits_ in (8, 32):
        with KvCache(dev, 1, nh, nkv, hd, block_size=16, max_positions=40, max_seqs=2, max_pages=3, bits=bits_) as kv:
            a, b = kv.open_seq(), kv.open_seq()
            kv.append(0, [a] * 30, *mk(30)[1:])
            for bad in ([b] * 17, [a] * 11, [a, b, a, b] * 8):  # pages, window, both
                with pytest.raises(G.CacheError):
                    kv.append(0, bad, *mk(len(bad))[1:])
                with pytest.raises(G.CacheError):
                    kv.attention(0, bad, *mk(len(bad)))
            for call in (lambda: kv.append(1, [a], *mk(1)[1:]), lambda: kv.append(0, [7], *mk(1)[1:]),
                         lambda: kv.append(0, [], *mk(0)[1:]), lambda: kv.read(0, [a], [30]), lambda: kv.read(0, [b], [0]),
                         lambda: kv.read(1, [a], [0]), lambda: kv.read(0, [9], [0]), lambda: kv.read(0, [], []),
                         lambda: kv.truncate([a, 5], [0, 0]), lambda: kv.truncate([], [])):
                with pytest.raises(G.InferenceError):
                    call()
            for call in (lambda: kv.read(0, [a], [0, 1]), lambda: kv.truncate([a], [0, 1])):
                with pytest.raises(ValueError):
                    call()
            assert (kv.seq_len(a), kv.seq_len(b), kv.free_pages()) == (30, 0, 1)
            kv.attention(0, [a] * 2 + [b] * 3, *mk(5))
            kv.close_seq(a)
            with pytest.raises(G.InferenceError):
                kv.truncate([a], [0])
            assert kv.free_pages() == 2


@pytest.mark.parametrize("bits_", [8, 32])
@pytest.mark.parametrize("more", [dict(max_pages=2**60), dict(max_pages=2**33), dict(block_size=2**31, max_pages=2**31),
                                  dict(max_positions=2**32 - 1, max_seqs=2**31, max_pages=1)])
def test_sizes_that_no_card_has(dev, bits_, more):
    # their products pass 64 bits, or a page's number 32
    with pytest.raises(G.ConfigError):
        KvCache(dev, 1, 4, 2, 16, bits=bits_, **more)


def test_a_call_that_no_grid_holds(dev):
    # one head of 4, 256 rows a tile: one tile more than a grid's 65535; refused before a position is taken
    n = 65535 * 256 + 1
    with KvCache(dev, 1, 1, 1, 4, block_size=1 << 16, max_positions=n, max_seqs=1, bits=8) as kv, Gpu() as gpu:
        s, free = kv.open_seq(), kv.free_pages()
        x = gpu.up(np.zeros(4 * n, np.float32))
        with pytest.raises(G.InferenceError, match="one launch"):
            kv.attention_async(0, np.full(n, s, np.uint32), x, x, x, gpu.up(np.zeros(4 * n, np.float32)), gpu.stream)
        assert kv.seq_len(s) == 0 and kv.free_pages() == free
        kv.append_async(0, np.full(1000, s, np.uint32), x, x, gpu.stream)
        gpu.wait()
        assert kv.seq_len(s) == 1000


def test_capture_is_refused(dev):
    with KvCache(dev, 1, 4, 2, 32, max_positions=64, max_seqs=1, bits=8) as kv, Gpu() as gpu:
        s = kv.open_seq()
        x, hip, graph = gpu.up(np.ones(128, np.float32)), gpu.hip, C.c_void_p()
        kv.append_async(0, [s], x, x, gpu.stream)
        gpu.wait()
        assert hip.hipStreamBeginCapture(gpu.st, 1) == 0  # thread-local capture mode
        try:
            for call in (lambda: kv.attention_async(0, [s], x, x, x, x, gpu.stream),
                         lambda: kv.append_async(0, [s], x, x, gpu.stream),
                         lambda: kv.read_async(0, [s], [0], x, x, gpu.stream),
                         lambda: kv.truncate([s], [0], gpu.stream)):
                with pytest.raises(G.InferenceError, match="captured"):
                    call()
        finally:
            assert hip.hipStreamEndCapture(gpu.st, C.byref(graph)) == 0  # the refusals have not broken it
            hip.hipGraphDestroy(graph)
        assert kv.seq_len(s) == 1


def test_offsets_past_32_bits(dev):
    # pages of a million positions: the second sequence's page, and the last kv head of each,
    # lie more than 4 GB into the pool
    nh, nkv, hd = 16, 8, 256
    rng = np.random.default_rng(15)
    with KvCache(dev, 1, nh, nkv, hd, block_size=1 << 20, max_positions=1 << 20, max_seqs=2, max_pages=2, bits=8) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, max_positions=1 << 20)
        a, b = kv.open_seq(), kv.open_seq()
        for n in (40, 1):
            run(kv, o, 0, [a] * n + [b] * n, draw(rng, 2 * n, nh, nkv, hd), f"far pages, {n}")
        same_rows(kv, o, 0, [a, b], "far pages")


def test_far_positions_turn_exactly(dev):
    # at position 100000 an angle formed in f32 is off by up to 0.004; here by less than a
    # rounding of the rotated key
    nh, nkv, hd, n = 2, 1, 64, 100000
    rng = np.random.default_rng(16)
    with KvCache(dev, 1, nh, nkv, hd, block_size=1024, max_positions=n + 40, max_seqs=1, bits=8, rope_theta=1e6) as kv:
        from oracle.attention8 import hold, rope64
        s = kv.open_seq()
        kv.append(0, [s] * n, *draw(rng, n, nh, nkv, hd)[1:])
        k, v = draw(rng, 37, nh, nkv, hd)[1:]
        kv.append(0, [s] * 37, k, v)
        got, _ = kv.read(0, [s] * 37, range(n, n + 37))
        want = np.stack([rope64(k[i].reshape(1, hd), n + i, 1e6) for i in range(37)])
        held = np.concatenate([hold(want[:16]), hold(want[16:32]), want[32:]])
        assert np.array_equal(got, held[:, 0])


def test_more_parts_than_a_pass_joins(dev):
    # heads of 256: four threads' groups of 16 parts of 512 positions are 32768 positions
    nh, nkv, hd, n = 2, 1, 256, 40005
    rng = np.random.default_rng(18)
    with KvCache(dev, 1, nh, nkv, hd, block_size=64, max_positions=n + 40, max_seqs=2, bits=8) as kv:
        o = Kv8Oracle(1, nh, nkv, hd, max_positions=n + 40)
        a, b = kv.open_seq(), kv.open_seq()
        for s, m in ((a, n), (b, 700)):
            k, v = draw(rng, m, nh, nkv, hd)[1:]
            kv.append(0, [s] * m, k, v)
            o.append(0, [s] * m, k, v)
        run(kv, o, 0, [a, b], draw(rng, 2, nh, nkv, hd), "many parts, a step")
        run(kv, o, 0, [b, a, a, a], draw(rng, 4, nh, nkv, hd), "many parts, drafts")


def test_streams_and_a_run_of_them_together(dev):
    """A prompt shared by three sequences, appended once each without attention; decode steps on a
    stream of the caller's; drafted tokens checked in one call and half of them taken back; the
    rows read on the device. All queued without waiting, against the restatement."""
    nh, nkv, hd, n = 8, 2, 64, 3
    rng = np.random.default_rng(17)
    with KvCache(dev, 2, nh, nkv, hd, block_size=32, max_positions=300, max_seqs=n, bits=8) as kv, Gpu() as gpu:
        o = Kv8Oracle(2, nh, nkv, hd, max_positions=300)
        seqs = [kv.open_seq() for _ in range(n)]
        outs = []

        def attend(layer, ids):
            q, k, v = draw(rng, len(ids), nh, nkv, hd)
            out = gpu.empty(q.nbytes)
            kv.attention_async(layer, ids, *(gpu.up(x) for x in (q, k, v)), out, gpu.stream)
            want, mag = o.attention(layer, ids, q, k, v)
            outs.append((out, want, mag))

        for l in range(2):
            for s in seqs:
                k, v = draw(np.random.default_rng(99 + l), 83, nh, nkv, hd)[1:]
                kv.append_async(l, [s] * 83, gpu.up(k), gpu.up(v), gpu.stream)
                o.append(l, [s] * 83, k, v)
        for rnd in range(6):
            for l in range(2):
                attend(l, seqs)
            for l in range(2):
                attend(l, [s for s in seqs for _ in range(5)])
            lens = [o.seq_len(s) - 2 - i for i, s in enumerate(seqs)]
            kv.truncate(seqs, lens, gpu.stream)
            o.truncate(seqs, lens)
        rows = [(s, p) for s in seqs for p in range(o.seq_len(s))]
        ids, pos = zip(*rows)
        kr, vr = (gpu.empty(len(rows) * nkv * hd * 4) for _ in range(2))
        kv.read_async(1, ids, pos, kr, vr, gpu.stream)
        gpu.wait()
        for i, (out, want, mag) in enumerate(outs):
            check(gpu.down(out, want.shape), want, mag, 300, hd, 6.0, f"call {i}")
        for g, w in zip((kr, vr), o.read(1, ids, pos)):
            assert np.array_equal(gpu.down(g, w.shape), w)


@pytest.mark.parametrize("n,past", [(3, 100), (2, 20), (40, 33)])
def test_context_over_its_queries(dev, n, past):
    # the output may be the query buffer, as with a cache in f32
    nh, nkv, hd = 8, 2, 64
    rng = np.random.default_rng(18)
    with KvCache(dev, 1, nh, nkv, hd, max_positions=300, max_seqs=n, bits=8) as kv, Gpu() as gpu:
        o = Kv8Oracle(1, nh, nkv, hd, max_positions=300)
        seqs = [kv.open_seq() for _ in range(3)] if n > 2 else [kv.open_seq()]
        ids = seqs * (n // len(seqs)) + seqs[:n % len(seqs)]
        for s in seqs:
            k, v = draw(rng, past, nh, nkv, hd)[1:]
            kv.append(0, [s] * past, k, v)
            o.append(0, [s] * past, k, v)
        q, k, v = draw(rng, n, nh, nkv, hd)
        at = gpu.up(np.concatenate([x.reshape(-1) for x in (q, k, v)]))
        kv.attention_async(0, ids, at, at + q.nbytes, at + q.nbytes + k.nbytes, at, gpu.stream)
        gpu.wait()
        want, mag = o.attention(0, ids, q, k, v)
        check(gpu.down(at, q.shape), want, mag, past + n, hd, 6.0, "over its queries")
