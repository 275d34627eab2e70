"""A model over a KV cache held in 8 bits (garuda_amd.DecodeModel on KvCache(bits=8)).

Teacher-forced, as tests/test_gpu_model.py: the device's own q, k and v go through
oracle/attention8.py's cache, and the model's contexts must match it within that file's bar
(rtol 1e-3, atol 1e-4 of the values' size), across the ends of blocks and pages. All else is
bit for bit: replayed graphs against eager launches, a prompt in one call against the same
chunks in two, and a step, prompt or draft that failed or was taken back against a model
that never made it."""
from __future__ import annotations

import numpy as np
import pytest

import garuda_amd as G
from garuda_amd.attention import KvCache
from oracle.attention8 import Kv8Oracle
from tests.test_gpu_model import close, release
from tests.test_gpu_parity import say
from tests.test_model_oracle import tiny_model

pytestmark = pytest.mark.gpu

VOCAB, NL, NH, NKV, HD = 256, 2, 8, 2, 32


@pytest.fixture(scope="module")
def dev():
    d = G.Device(0, slab_bytes=256 << 20)
    yield d
    d.close()


@pytest.fixture(scope="module")
def weights():
    return tiny_model(29, n_layers=NL, d=256, nh=NH, nkv=NKV, hd=HD, f=256, ne=8, k=2, vocab=VOCAB)


def model8(dev, w, max_positions=64, max_seqs=4, window=0):
    layers, out, onorm, embd, (nh, nkv, hd) = w
    kv = KvCache(dev, len(layers), nh, nkv, hd, block_size=32, max_positions=max_positions, max_seqs=max_seqs,
                 sliding_window=window, bits=8)
    moe, dense = [], {n: [] for n in ("wq", "wk", "wv", "wo")}
    for L in layers:
        m = L["moe"]
        moe.append(G.MoeLayer(dev, m["d"], m["f"], m["ne"], m["k"], m["router"], m["gate"], m["up"], m["down"],
                              m["qtypes"]))
        for n in dense:
            qt, raw, r, c = L[n]
            dense[n].append(G.DenseWeight(dev, qt, r, c, raw))
    qt, raw, r, c = out
    head = G.DenseWeight(dev, qt, r, c, raw)
    model = G.DecodeModel(dev, kv, moe, dense["wq"], dense["wk"], dense["wv"], dense["wo"], head,
                          np.stack([L["attn_norm"] for L in layers]), np.stack([L["ffn_norm"] for L in layers]),
                          onorm, embd)
    return model, kv, moe, dense, head


def bits(x):
    return np.asarray(x, np.float32).view(np.uint32)


def same_step(step, a, b):
    assert np.array_equal(a[0], b[0]), f"step {step}: next tokens differ"
    assert np.array_equal(bits(a[1]), bits(b[1])), f"step {step}: logits differ"


def same_cache(kva, sa, kvb, sb, n):
    pos = np.arange(n)
    for l in range(NL):
        assert kva.seq_len(sa, l) == kvb.seq_len(sb, l) == n
        for x, y in zip(kva.read(l, [sa] * n, pos), kvb.read(l, [sb] * n, pos)):
            assert np.array_equal(bits(x), bits(y)), f"layer {l}: rows differ"


@pytest.mark.parametrize("window", [0, 20])
def test_contexts_teacher_forced(dev, weights, window):
    parts = model8(dev, weights, window=window)
    model, kv = parts[0], parts[1]
    orc = Kv8Oracle(NL, NH, NKV, HD, max_positions=64, sliding_window=window)
    try:
        seqs = [kv.open_seq() for _ in range(3)]
        toks = np.array([3, 77, 200], np.uint32)
        for step in range(36):
            live = [0, 1, 2] if step % 5 else [0, 2]  # the lengths drift apart
            say(f"8-bit model step {step}, window {window}")
            gn, _, tr, _ = model.decode_step_trace([seqs[i] for i in live], toks[live])
            for l, T in enumerate(tr):
                ctx, _ = orc.attention(l, [seqs[i] for i in live], T["q"], T["k"], T["v"])
                close(f"step {step} layer {l}: context", T["context"], ctx)
            toks[live] = gn
    finally:
        release(*parts)


@pytest.mark.parametrize("prompt,max_positions", [(0, 64), (505, 32768)], ids=["short", "long-window"])
def test_graph_steps_equal_eager_steps(dev, weights, prompt, max_positions):
    """The batch drifts over sizes, the contexts pass ends of blocks, pages, and (long-window)
    of the positions that one part of a row attends to."""
    a, b = model8(dev, weights, max_positions), model8(dev, weights, max_positions)
    ma, kva, mb, kvb = a[0], a[1], b[0], b[1]
    try:
        ma.set_graphs(False)
        sa, sb = [kva.open_seq() for _ in range(3)], [kvb.open_seq() for _ in range(3)]
        rng = np.random.default_rng(5)
        toks = rng.integers(0, VOCAB, 3).astype(np.uint32)
        if prompt:
            p = rng.integers(0, VOCAB, prompt).astype(np.uint32)
            for i in (0, 2):
                same_step(f"prompt {i}", ma.prefill(sa[i], p, want_logits=True), mb.prefill(sb[i], p, want_logits=True))
        pattern, replays = [3, 2, 3, 1, 3, 2, 2, 3, 1, 1], 0
        for step in range(40):
            n = pattern[step % len(pattern)]
            live = list(range(n))
            replays += mb.graph_ready(n)
            say(f"8-bit graph step {step}, batch {n}")
            ra = ma.decode_step([sa[i] for i in live], toks[live], want_logits=True)
            rb = mb.decode_step([sb[i] for i in live], toks[live], want_logits=True)
            same_step(step, ra, rb)
            toks[live] = ra[0]
        assert replays >= 30, f"{replays} steps replayed from a graph"
        for i in range(3):
            same_cache(kva, sa[i], kvb, sb[i], kva.seq_len(sa[i]))
    finally:
        release(*a)
        release(*b)


def test_a_prompt_in_two_calls_of_the_same_chunks(dev, weights):
    """300 tokens run as chunks of 256 and 44: the same bits as two calls of 256 and 44, and
    from the steps that follow. The keys are those that single steps leave: the sums of the
    batched projections differ in order only, so that a held value differs by their
    rounding (1e-3 of its block's largest) and by one step of its code at most."""
    a, b = model8(dev, weights, 512), model8(dev, weights, 512)
    ma, kva, mb, kvb = a[0], a[1], b[0], b[1]
    try:
        prompt = np.random.default_rng(8).integers(0, VOCAB, 300).astype(np.uint32)
        s, t = kva.open_seq(), kvb.open_seq()
        ra = ma.prefill(s, prompt, n_last=3, want_logits=True)
        mb.prefill(t, prompt[:256])
        rb = mb.prefill(t, prompt[256:], n_last=3, want_logits=True)
        same_step("prompt", ra, rb)
        toks = ra[0][-1:]
        for step in range(20):
            ra = ma.decode_step([s], toks, want_logits=True)
            same_step(step, ra, mb.decode_step([t], toks, want_logits=True))
            toks = ra[0]
        same_cache(kva, s, kvb, t, 320)
        u = kvb.open_seq()
        for i in prompt[:40]:
            mb.decode_step([u], [i])
        for x, y in zip(kva.read(0, [s] * 32, np.arange(32)), kvb.read(0, [u] * 32, np.arange(32))):
            for blk in (slice(0, 16), slice(16, 32)):
                xb, yb = x[blk].reshape(16, NKV, HD), y[blk].reshape(16, NKV, HD)
                m = np.abs(yb).max(axis=(0, 2), keepdims=True)
                assert np.all(np.abs(xb - yb) <= (1 / 127 + 1e-3) * m)
    finally:
        release(*a)
        release(*b)


@pytest.mark.parametrize("fail", ["prompt", "step"])
def test_a_late_failure_leaves_the_cache_as_it_was(dev, weights, fail):
    """The output head is gone, so that the call fails after its last layer has written its
    rows: lengths, pages and rows, the open block's among them, come back, and the cache
    answers on like one that never saw the call."""
    a, b = model8(dev, weights, 128), model8(dev, weights, 128)
    ma, kva, mb, kvb = a[0], a[1], b[0], b[1]
    try:
        rng = np.random.default_rng(9)
        for n in (21, 31, 32, 1):
            prompt = rng.integers(0, VOCAB, n).astype(np.uint32)
            s, t = kva.open_seq(), kvb.open_seq()
            same_step("prompt", ma.prefill(s, prompt, want_logits=True), mb.prefill(t, prompt, want_logits=True))
        ma.set_graphs(False)
        a[4].release()
        free = kva.free_pages()
        for s, n in enumerate((21, 31, 32, 1)):
            say(f"a {fail} that fails at position {n}")
            with pytest.raises(G.GarudaError):
                if fail == "prompt":
                    ma.prefill(s, rng.integers(0, VOCAB, 40).astype(np.uint32))
                else:
                    ma.decode_step([s], [7])
            same_cache(kva, s, kvb, s, n)
        assert kva.free_pages() == free
        for step in range(20):  # over the end of each one's open block
            q = rng.normal(size=(4, NH * HD)).astype(np.float32)
            k, v = (rng.normal(size=(4, NKV * HD)).astype(np.float32) for _ in range(2))
            for l in range(NL):
                x, y = kva.attention(l, range(4), q, k, v), kvb.attention(l, range(4), q, k, v)
                assert np.array_equal(bits(x), bits(y)), (step, l)
    finally:
        a[0].close()
        for m in a[2]:
            m.release()
        for ws in a[3].values():
            for w in ws:
                w.release()
        kva.close()
        release(*b)


def test_drafts_taken_back(dev, weights):
    """Draft tokens decoded and taken back, as speculation does: within the open block the
    next steps are those of a model that never drafted, bit for bit. Cut back into a complete
    block, its kept rows are what they are held as."""
    a, b = model8(dev, weights, 128), model8(dev, weights, 128)
    ma, kva, mb, kvb = a[0], a[1], b[0], b[1]
    try:
        rng = np.random.default_rng(10)
        sa, sb = [kva.open_seq() for _ in range(2)], [kvb.open_seq() for _ in range(2)]
        toks = np.array([1, 2], np.uint32)
        free = kva.free_pages()
        for step in range(34):
            if step % 16 in (2, 7, 9):  # drafts of 4 stay in the block
                kept = [kva.seq_len(s) for s in sa]
                for _ in range(4):
                    ma.decode_step(sa, rng.integers(0, VOCAB, 2).astype(np.uint32))
                kva.truncate(sa, kept)
                assert all(kva.seq_len(s, l) == k for s, k in zip(sa, kept) for l in range(NL))
            ra = ma.decode_step(sa, toks, want_logits=True)
            same_step(step, ra, mb.decode_step(sb, toks, want_logits=True))
            toks = ra[0]
        for s, t in zip(sa, sb):
            same_cache(kva, s, kvb, t, 34)
        held = [kva.read(l, [sa[0]] * 32, np.arange(32)) for l in range(NL)]
        kva.truncate(sa, [21, 0])
        for l in range(NL):
            for x, y in zip(kva.read(l, [sa[0]] * 21, np.arange(21)), held[l]):
                assert np.array_equal(bits(x), bits(y[:21]))
        ma.decode_step(sa, toks)
        assert [kva.seq_len(s, NL - 1) for s in sa] == [22, 1]
        kva.truncate(sa, [0, 0])
        assert kva.free_pages() == free
    finally:
        release(*a)
        release(*b)


def test_refusals_leave_the_sequences_unchanged(dev, weights):
    parts = model8(dev, weights, max_positions=33)
    model, kv = parts[0], parts[1]
    try:
        a, b = kv.open_seq(), kv.open_seq()
        model.prefill(a, np.arange(32, dtype=np.uint32))
        for bad in ([a, a], [a, 99]):
            with pytest.raises(G.InferenceError):
                model.decode_step(bad, [1, 2])
        with pytest.raises(G.CacheError):
            model.prefill(a, [1, 2])
        model.decode_step([a, b], [3, 4])
        with pytest.raises(G.CacheError):  # a's window of 33 positions is full
            model.decode_step([a, b], [6, 7])
        kv.fail_reserves(1)  # a new batch size: its scratch is reserved before anything commits
        with pytest.raises(G.DeviceError):
            model.decode_step([b], [5])
        assert [(kv.seq_len(a, l), kv.seq_len(b, l)) for l in range(NL)] == [(33, 1)] * NL
        model.decode_step([b], [5])
        assert kv.seq_len(b, NL - 1) == 2
    finally:
        release(*parts)
