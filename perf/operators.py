"""Timed operators of the KV cache held in 8 bits, through the library's public entry points.

A cache of `bits=8` (`KvCache(..., bits=8)`) holds keys and values in blocks of 16
positions. For one sequence, layer and kv head, a complete block of keys (or values) is held
as integers in [-127, 127] and one f32 scale; the block that a sequence's last position is
in, while it is incomplete, is held in f32. Keys are held rotated by their position, with
the angle formed in 64 bits and the rotated key rounded once to f32.

  * `step`: one call of attention over the cache (`KvCache.attention_async`): the tokens' keys
    and values are appended and each token attends to its sequence up to itself, to the
    positions of its own block as they were given and to earlier ones as held in 8 bits. The
    rows that the call appended are read back (`KvCache.read_async`);
  * `append`: keys and values appended without attention (`KvCache.append_async`), as when
    a prompt's projections are known and only its cache is wanted, and read back.

Each pass first takes the sequences back to the length they had (`KvCache.truncate`), as a
program does with drafted tokens that were not accepted, or when an answer is asked for again.

`own` says whether `run` makes these calls or computes the same in elementary torch operations
over a cache of the same content.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

BLOCK = 16
#: query heads, kv heads, head width, rope theta
HEADS = {
    "32x8x128": (32, 8, 128, 1e6),   # the Mixtral shape
    "8x2x32": (8, 2, 32, 1e4),       # the synthetic engine
    "16x16x64": (16, 16, 64, 1e4),   # a kv head for each query head
    "8x1x256": (8, 1, 256, 1e4),     # one wide kv head
    "12x4x80": (12, 4, 80, 1e4),     # a width that is no multiple of 32, groups of three
}


def listed():
    return [
        # the smallest call: the synthetic engine's heads, one sequence, three blocks; launches
        dict(name="step_1_short", kind="step", heads="8x2x32", seqs=1, tokens=1, past=40, ragged=False, window=0),
        # single-user decode at a usual context: few workgroups, latency and the join of the splits
        dict(name="step_1_4000", kind="step", heads="32x8x128", seqs=1, tokens=1, past=4000, ragged=False, window=0),
        # a small decode batch; the token completes a block, which is then held in 8 bits
        dict(name="step_8_2047", kind="step", heads="32x8x128", seqs=8, tokens=1, past=2047, ragged=False, window=0),
        # continuous batching: sequences of all ages
        dict(name="step_48_ragged", kind="step", heads="32x8x128", seqs=48, tokens=1, past=16000, ragged=True, window=0),
        # the largest decode step: long documents, bound by the cache's bytes
        dict(name="step_8_65000", kind="step", heads="32x8x128", seqs=8, tokens=1, past=65000, ragged=False, window=0),
        # a sliding window over sequences that have outgrown it, a kv head for each query head
        dict(name="step_16_window", kind="step", heads="16x16x64", seqs=16, tokens=1, past=5003, ragged=False, window=1000),
        # wide heads, one kv head for eight query heads
        dict(name="step_32_wide", kind="step", heads="8x1x256", seqs=32, tokens=1, past=6000, ragged=True, window=0),
        # five drafted tokens of each sequence checked in one call
        dict(name="drafts_6x5", kind="step", heads="32x8x128", seqs=6, tokens=5, past=6000, ragged=True, window=0),
        # one chunk of a prompt, as the model's prefill cuts it
        dict(name="prompt_256_1280", kind="step", heads="32x8x128", seqs=1, tokens=256, past=1280, ragged=False, window=0),
        # a long chunk of a long prompt: bound by the products
        dict(name="prompt_1024_8192", kind="step", heads="32x8x128", seqs=1, tokens=1024, past=8192, ragged=False, window=0),
        # one row of each of 64 sequences, without attention
        dict(name="append_64x1", kind="append", heads="32x8x128", seqs=64, tokens=1, past=300, ragged=True, window=0),
        # two prompts of odd length from their beginning, without attention
        dict(name="append_2x1999", kind="append", heads="32x8x128", seqs=2, tokens=1999, past=0, ragged=False, window=0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("decode", "decode", "decode", "drafts", "prompt", "prompt", "append"))
    heads = rng.choice(("32x8x128", "32x8x128") + tuple(sorted(HEADS)))
    window = rng.choice((0, 0, _log_int(rng, 20, 4000)))
    if kind == "decode":
        past = _log_int(rng, 1, 65000)
        seqs = _log_int(rng, 1, max(1, min(64, 500000 // past)))
        return dict(kind="step", heads=heads, seqs=seqs, tokens=1, past=past, ragged=rng.random() < 0.5, window=window)
    if kind == "drafts":
        return dict(kind="step", heads=heads, seqs=_log_int(rng, 1, 16), tokens=rng.randint(2, 12),
                    past=_log_int(rng, 10, 16000), ragged=rng.random() < 0.5, window=window)
    tokens = _log_int(rng, 17, 1024)
    if kind == "prompt":
        past = rng.choice((0, _log_int(rng, 16, 8192)))
        seqs = _log_int(rng, 1, max(1, min(8, 9000000 // (tokens * (past + tokens)))))
        return dict(kind="step", heads=heads, seqs=seqs, tokens=tokens, past=past, ragged=rng.random() < 0.5, window=window)
    return dict(kind="append", heads=heads, seqs=_log_int(rng, 1, 16), tokens=rng.choice((1, tokens, 2 * tokens - 1)),
                past=_log_int(rng, 1, 2000), ragged=rng.random() < 0.5, window=0)


# ---- sizes and inputs ----

def _pasts(case):
    """Each sequence's length before the call. Drafts sit inside one block, and prompts begin at a
    block's start (a shared prefix ends there), so that a sequence taken back holds what it held."""
    n, t = case["seqs"], case["tokens"]
    got = []
    for i in range(n):
        p = case["past"]
        if case["ragged"] and p > 0:
            p = 1 + int((p - 1) * ((i + 1) * 0.6180339887498949 % 1.0))
        if t > BLOCK:
            p -= p % BLOCK
        elif t > 1:
            p = p - p % BLOCK + p % (BLOCK + 1 - t)
        got.append(p)
    return got


def _starts(case, p):
    """The first position that a token at position p attends to."""
    return max(0, p + 1 - case["window"]) if case["window"] else 0


def _dev():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _gen(seed, *tag):
    h = int(seed) & 0xFFFFFFFF
    for t in tag:
        h = (h * 1000003 + int(t) + 12345) & 0xFFFFFFFFFFFF
    return torch.Generator(device=_dev()).manual_seed(h)


def _rows(case, seed, n, tag):
    """n tokens' keys and values; a key's channels differ in size, as a projection's do."""
    _, nkv, hd, _ = HEADS[case["heads"]]
    size = torch.exp(0.5 * torch.randn(nkv * hd, generator=_gen(seed, 1), device=_dev()))
    k = torch.randn(n, nkv * hd, generator=_gen(seed, 2, tag), device=_dev()) * size
    return k, torch.randn(n, nkv * hd, generator=_gen(seed, 3, tag), device=_dev())


def _inputs(case, seed):
    nh, _, hd, _ = HEADS[case["heads"]]
    n = case["seqs"] * case["tokens"]
    q = torch.randn(n, nh * hd, generator=_gen(seed, 4), device=_dev())
    return (q, *_rows(case, seed, n, 1000000))


# ---- the plain form ----

def _rotate(x, pos, theta):
    """x [..., hd] by the positions pos (that broadcast to x's leading axes), in 64 bits, rounded once."""
    hd = x.shape[-1]
    f = float(theta) ** (-torch.arange(0, hd, 2, device=x.device, dtype=torch.float64) / hd)
    a = pos.double()[..., None] * f
    c, s = torch.cos(a), torch.sin(a)
    x = x.double()
    x, y = x[..., 0::2], x[..., 1::2]
    return torch.stack((x * c - y * s, x * s + y * c), -1).flatten(-2).float()


def _quantise(x):
    """x [..., 16, hd]: codes, and a scale for each block."""
    top = x.abs().amax((-1, -2)).double()
    inv = torch.where(top > 0, 127.0 / top, torch.zeros_like(top))
    return (x.double() * inv[..., None, None]).round().to(torch.int8), (top / 127.0).float()


def _held(codes, scale):
    return codes.float() * scale[..., None, None]


class _Plain:
    """A cache's content as tensors: codes and scales of complete blocks, [seqs, nkv, blocks, 16, hd]
    and [seqs, nkv, blocks], and the open block's rows in f32, [seqs, nkv, 16, hd]."""

    def __init__(self, case, seed):
        _, nkv, hd, theta = HEADS[case["heads"]]
        pasts = _pasts(case)
        n, nb = len(pasts), max(p // BLOCK for p in pasts)
        dev = _dev()
        self.first = min(_starts(case, p) // BLOCK for p in pasts)  # no token attends to a block before it
        self.first = min(self.first, nb)
        self.codes = [torch.zeros(n, nkv, nb, BLOCK, hd, dtype=torch.int8, device=dev) for _ in range(2)]
        self.scale = [torch.zeros(n, nkv, nb, device=dev) for _ in range(2)]
        self.open = [torch.zeros(n, nkv, BLOCK, hd, device=dev) for _ in range(2)]
        for s, p in enumerate(pasts):
            if p == 0:
                continue
            k, v = (x.view(p, nkv, hd) for x in _rows(case, seed, p, s))
            k = _rotate(k, torch.arange(p, device=dev)[:, None], theta)
            b = p // BLOCK
            for j, x in enumerate((k, v)):
                if b:
                    c, sc = _quantise(x[:b * BLOCK].view(b, BLOCK, nkv, hd).permute(2, 0, 1, 3))
                    self.codes[j][s, :, :b], self.scale[j][s, :, :b] = c, sc
                if p % BLOCK:
                    self.open[j][s, :, :p % BLOCK] = x[b * BLOCK:].transpose(0, 1)
        self.past = torch.tensor(pasts, device=dev)
        rem = max(p % BLOCK for p in pasts)
        self.blocks = -(-(rem + case["tokens"]) // BLOCK)  # that the call's positions, from their block's start on, take


def _plain_append(st):
    """The call's positions from the start of their block on: f32 rows and what they are held as,
    [2][seqs, nkv, blocks * 16, hd], each row's index there, and the rows' values read back."""
    c, t = st.plain, st.case["tokens"]
    _, nkv, hd, theta = HEADS[st.case["heads"]]
    n, rem = c.past.numel(), c.past % BLOCK
    at = torch.arange(c.blocks * BLOCK, device=rem.device)
    src = at - rem[:, None]  # the call's token at a place, negative: an earlier one of the block
    pos = c.past[:, None] + torch.arange(t, device=rem.device)
    new = (_rotate(st.k.view(n, t, nkv, hd), pos[..., None], theta), st.v.view(n, t, nkv, hd))
    given, held, back = [], [], []
    whole = (torch.arange(1, c.blocks + 1, device=rem.device) * BLOCK <= rem[:, None] + t)[:, None, :, None, None]
    to = (rem[:, None] + torch.arange(t, device=rem.device))[:, None, :, None].expand(n, nkv, t, hd)
    for x, old in zip(new, c.open):
        x = x.transpose(1, 2).gather(2, src.clamp(0, t - 1)[:, None, :, None].expand(n, nkv, at.numel(), hd))
        old = old[:, :, at.clamp(max=BLOCK - 1)]
        x = torch.where((src < 0)[:, None, :, None], old, x) * (src < t)[:, None, :, None]
        b = x.view(n, nkv, c.blocks, BLOCK, hd)
        q = torch.where(whole, _held(*_quantise(b)), b).view_as(x)
        given.append(x)
        held.append(q)
        back.append(q.gather(2, to).transpose(1, 2).reshape(n * t, nkv * hd))
    return given, held, pos, back


def _plain_step(st):
    given, held, pos, back = _plain_append(st)
    c, t = st.plain, st.case["tokens"]
    nh, nkv, hd, theta = HEADS[st.case["heads"]]
    n, g = c.past.numel(), nh // nkv
    q = _rotate(st.q.view(n, t, nh, hd), pos[..., None], theta)
    q = q.view(n, t, nkv, g, hd).permute(0, 2, 3, 1, 4).reshape(n, nkv, g * t, hd) * hd ** -0.5
    old = [_held(x[:, :, c.first:], s[:, :, c.first:]).flatten(2, 3) for x, s in zip(c.codes, c.scale)]
    keys = (old[0], held[0], given[0])
    s = torch.cat([torch.matmul(q, x.transpose(-1, -2)) for x in keys], -1).view(n, nkv, g, t, -1)
    base = c.past - c.past % BLOCK  # the call's first block
    begin = (pos + 1 - st.case["window"]).clamp(min=0) if st.case["window"] else torch.zeros_like(pos)
    p0 = c.first * BLOCK + torch.arange(old[0].shape[2], device=pos.device).expand(n, -1)
    p1 = base[:, None] + torch.arange(held[0].shape[2], device=pos.device)
    block, begin, at = pos[..., None] // BLOCK, begin[..., None], pos[..., None]
    ok = torch.cat(((p0 < base[:, None])[:, None] & (p0[:, None] >= begin),
                    (p1[:, None] // BLOCK < block) & (p1[:, None] >= begin),
                    (p1[:, None] // BLOCK == block) & (p1[:, None] <= at) & (p1[:, None] >= begin)), -1)
    s = s.masked_fill(~ok[:, None, None], -math.inf)
    w = torch.exp(s - s.amax(-1, keepdim=True))
    w = (w / w.sum(-1, keepdim=True)).view(n, nkv, g * t, -1)
    parts = w.split([x.shape[2] for x in keys], -1)
    out = sum(torch.matmul(x, y) for x, y in zip(parts, (old[1], held[1], given[1])))
    out = out.view(n, nkv, g, t, hd).permute(0, 3, 1, 2, 4).reshape(n * t, nh * hd)
    return [out, *back]


# ---- the framework's calls ----

_lib = None


def _library():
    """The program's device and its stream."""
    global _lib
    if _lib is None:
        import garuda_amd as G
        _lib = (G.Device(0, slab_bytes=1 << 20), torch.cuda.Stream())
    return _lib


class _State:
    kv = None

    def __del__(self):
        if self.kv is not None:
            self.kv.close()


def _cache(st, case, seed):
    from garuda_amd.attention import KvCache
    nh, nkv, hd, theta = HEADS[case["heads"]]
    dev, stream = _library()
    pasts, t = _pasts(case), case["tokens"]
    st.kv = KvCache(dev, 1, nh, nkv, hd, block_size=BLOCK, max_positions=max(pasts) + t, sliding_window=case["window"],
                    max_seqs=len(pasts), max_pages=sum(-(-(p + t) // BLOCK) for p in pasts), rope_theta=theta, bits=8)
    st.seqs = np.array([st.kv.open_seq() for _ in pasts], np.uint32)
    st.lens = np.array(pasts, np.uint32)
    for s, p in enumerate(pasts):
        if p:
            k, v = _rows(case, seed, p, s)
            torch.cuda.synchronize()
            st.kv.append_async(0, np.full(p, st.seqs[s], np.uint32), k.data_ptr(), v.data_ptr(), stream.cuda_stream)
            stream.synchronize()
    st.ids = np.repeat(st.seqs, t)
    st.pos = (st.lens[:, None] + np.arange(t, dtype=np.uint32)).reshape(-1)
    st.stream = stream.cuda_stream
    st.out, st.k_back, st.v_back = torch.empty_like(st.q), torch.empty_like(st.k), torch.empty_like(st.v)


def _own_run(st):
    st.kv.truncate(st.seqs, st.lens, st.stream)
    if st.case["kind"] == "step":
        st.kv.attention_async(0, st.ids, st.q.data_ptr(), st.k.data_ptr(), st.v.data_ptr(), st.out.data_ptr(), st.stream)
    else:
        st.kv.append_async(0, st.ids, st.k.data_ptr(), st.v.data_ptr(), st.stream)
    st.kv.read_async(0, st.ids, st.pos, st.k_back.data_ptr(), st.v_back.data_ptr(), st.stream)
    return [st.out, st.k_back, st.v_back] if st.case["kind"] == "step" else [st.k_back, st.v_back]


# ---- what the tools call ----

def prepare(case, seed):
    st = _State()
    st.case = case
    st.q, st.k, st.v = _inputs(case, seed)
    if own:
        _cache(st, case, seed)
    else:
        st.plain = _Plain(case, seed)
    return st


def run(st):
    if own:
        return _own_run(st)
    return _plain_step(st) if st.case["kind"] == "step" else _plain_append(st)[3]


def work(case):
    """Codes and scales of the complete blocks attended to, the open blocks' f32 rows, the call's rows in and
    its context out; the appended rows written, and read back in f32. Two products of the span a head."""
    nh, nkv, hd, _ = HEADS[case["heads"]]
    t, row = case["tokens"], 4 * nkv * hd
    total = flops = 0
    for p in _pasts(case):
        done = (p + t) // BLOCK - p // BLOCK  # blocks that the call completes
        rem = p % BLOCK
        total += 2 * row * t + 2 * row * t  # k and v in, and back out
        total += done * nkv * (2 * BLOCK * hd + 8) + 2 * row * (((p + t) % BLOCK) if done else t)
        total += 2 * row * rem if done or case["kind"] == "step" else 0
        if case["kind"] == "step":
            total += 8 * nh * hd * t + max(0, p // BLOCK - _starts(case, p) // BLOCK) * nkv * (2 * BLOCK * hd + 8)
            flops += sum(4 * nh * hd * (i + 1 - _starts(case, i)) for i in range(p, p + t))
    return {"bytes": total, "flops": flops}


def exact(case, seed):
    """Sequence by sequence in 64 bits: every key and value as it was given (the held f32 row) and as
    its block holds it, a token taking the one for its own block and the other for earlier ones."""
    nh, nkv, hd, theta = HEADS[case["heads"]]
    t, g, dev = case["tokens"], nh // nkv, _dev()
    q_all, k_all, v_all = _inputs(case, seed)
    freq = torch.tensor([float(theta) ** (-2.0 * i / hd) for i in range(hd // 2)], dtype=torch.float64, device=dev)

    def turned(x, first):  # [rows, heads, hd] at positions first, first + 1, ...
        pairs = torch.view_as_complex(x.double().reshape(*x.shape[:2], hd // 2, 2))
        ang = torch.arange(first, first + x.shape[0], dtype=torch.float64, device=dev)[:, None, None] * freq
        return torch.view_as_real(pairs * torch.polar(torch.ones_like(ang), ang)).flatten(-2)

    def as_held(x):  # [rows, nkv, hd] f32, from position 0 on
        whole = x.shape[0] // BLOCK * BLOCK
        b = x[:whole].double().reshape(whole // BLOCK, BLOCK, nkv, hd)
        top = b.abs().amax(dim=(1, 3), keepdim=True)
        scale = (top / 127).float().double()
        codes = torch.round(b * torch.where(top > 0, 127 / top, 0.0))
        return torch.cat([(codes * scale).reshape(whole, nkv, hd), x[whole:].double()])

    ctx, kb, vb = [], [], []
    for s, p in enumerate(_pasts(case)):
        mine = slice(s * t, (s + 1) * t)
        k, v = k_all[mine], v_all[mine]
        if p:
            k0, v0 = _rows(case, seed, p, s)
            k, v = torch.cat([k0, k]), torch.cat([v0, v])
        given = [turned(k.view(-1, nkv, hd), 0).float(), v.view(-1, nkv, hd)]
        held = [as_held(x) for x in given]
        kb.append(held[0][p:].reshape(t, -1))
        vb.append(held[1][p:].reshape(t, -1))
        if case["kind"] != "step":
            continue
        q = turned(q_all[mine].view(t, nh, hd), p).float().double()
        at, key = torch.arange(p, p + t, device=dev)[:, None], torch.arange(p + t, device=dev)[None]
        low = (at + 1 - case["window"]).clamp(min=0) if case["window"] else 0
        seen, near = (key <= at) & (key >= low), key // BLOCK == at // BLOCK
        rows = []
        for h in range(nh):
            kh, vh, kg, vg = held[0][:, h // g], held[1][:, h // g], given[0][:, h // g].double(), given[1][:, h // g].double()
            sc = torch.where(near, q[:, h] @ kg.T, q[:, h] @ kh.T) / math.sqrt(hd)
            w = torch.softmax(sc.masked_fill(~seen, -math.inf), -1)
            rows.append((w * near) @ vg + (w * ~near) @ vh)
        ctx.append(torch.stack(rows, 1).reshape(t, nh * hd))
    back = [torch.cat(kb), torch.cat(vb)]
    return [torch.cat(ctx), *back] if case["kind"] == "step" else back
