"""CPU restatement of the KV cache held in 8 bits, from its definition.

TEST INFRASTRUCTURE ONLY: imported by tests/ as the checker of gmoe_kv_create_q8's caches
(garuda_amd/csrc/gmoe_attn8.hip, gmoe_kv.cpp). The product never loads it.

Sequences and layers as oracle/attention.py's KvOracle. Keys are rotated with the angle in
float64 and rounded once to float32. A complete block of 16 positions of one kv head is held
as codes rint(x * 127 / m), m = max |x|, and a float32 scale m / 127; a token attends to its
own block's rows as they were given and to earlier ones as held. Sums are float64.
"""
from __future__ import annotations

import numpy as np

BLOCK = 16


def rope64(x: np.ndarray, pos: int, theta: float) -> np.ndarray:
    """One token's heads [heads, hd], rotated in float64, rounded once."""
    hd = x.shape[-1]
    ang = pos * np.float64(theta) ** (-np.arange(0, hd, 2, dtype=np.float64) / hd)
    c, s = np.cos(ang), np.sin(ang)
    a, b = x[..., 0::2].astype(np.float64), x[..., 1::2].astype(np.float64)
    out = np.empty(x.shape, np.float32)
    with np.errstate(invalid="ignore", over="ignore"):
        out[..., 0::2] = a * c - b * s
        out[..., 1::2] = a * s + b * c
    return out


def hold(x: np.ndarray) -> np.ndarray:
    """A block's rows [16, heads, hd] (f32) as what they are held as (f32)."""
    out = np.empty_like(x)
    for h in range(x.shape[1]):
        m = np.abs(x[:, h]).max()
        if not np.isfinite(m):
            out[:, h] = np.nan
        elif m == 0:
            out[:, h] = 0
        else:
            codes = np.rint(x[:, h].astype(np.float64) * (127.0 * (1.0 / np.float64(m))))
            out[:, h] = codes.astype(np.float32) * np.float32(np.float64(m) / 127.0)
    return out


class _Rows:
    def __init__(self, nkv, hd):
        self.given = [np.zeros((0, nkv, hd), np.float32) for _ in range(2)]  # keys, values as given
        self.held = [np.zeros((0, nkv, hd), np.float32) for _ in range(2)]   # complete blocks
        self.open_block = 0


class Kv8Oracle:
    def __init__(self, n_layers, n_heads, n_kv_heads, head_dim, max_positions=2048, sliding_window=0,
                 rope_theta=10000.0):
        self.nl, self.nh, self.nkv, self.hd = n_layers, n_heads, n_kv_heads, head_dim
        self.maxpos, self.win, self.theta = max_positions, sliding_window, rope_theta
        self.rows = {}

    def of(self, seq, layer):
        return self.rows.setdefault((seq, layer), _Rows(self.nkv, self.hd))

    def seq_len(self, seq, layer=0):
        return len(self.of(seq, layer).given[0])

    def append_one(self, layer, seq, k, v):
        r = self.of(seq, layer)
        pos = len(r.given[0])
        if pos >= self.maxpos:
            raise ValueError("context window exhausted")
        new = (rope64(np.asarray(k, np.float32).reshape(self.nkv, self.hd), pos, self.theta),
               np.asarray(v, np.float32).reshape(self.nkv, self.hd))
        for j in range(2):
            r.given[j] = np.concatenate([r.given[j], new[j][None]])
            if (pos + 1) % BLOCK == 0:
                r.held[j] = np.concatenate([r.held[j], hold(r.given[j][-BLOCK:])])
        r.open_block = pos // BLOCK
        return pos

    def seen(self, layer, seq, pos):
        """(start, keys, values) that the token at `pos` attends to, float64."""
        r = self.of(seq, layer)
        own = pos // BLOCK * BLOCK
        start = max(0, pos + 1 - self.win) if self.win else 0
        return (start, *(np.concatenate([r.held[j][:own], r.given[j][own:pos + 1]])[start:].astype(np.float64)
                         for j in range(2)))

    def attend_one(self, layer, seq, pos, q):
        """(context, a bound on the magnitude of its scores' products): float64."""
        q = rope64(np.asarray(q, np.float32).reshape(self.nh, self.hd), pos, self.theta).astype(np.float64)
        _, K, V = self.seen(layer, seq, pos)
        g, out, mag = self.nh // self.nkv, np.empty((self.nh, self.hd)), 0.0
        with np.errstate(invalid="ignore", over="ignore"):
            for h in range(self.nh):
                k = K[:, h // g]
                s = k @ q[h] / np.sqrt(self.hd)
                s32 = s.astype(np.float32)  # beyond f32 a score is infinite
                if np.isnan(s32).any() or np.isposinf(s32).any() or np.isneginf(s32).all():
                    w = np.full(s.size, 1.0 / s.size)
                else:
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    mag = max(mag, float(np.max(np.abs(k) @ np.abs(q[h])) / np.sqrt(self.hd)))
                out[h] = w @ V[:, h // g]
        return out.reshape(-1), mag

    def append(self, layer, seqs, k, v):
        """Entries in order; returns their positions."""
        seqs = [int(s) for s in seqs]
        at, pos = 0, []
        while at < len(seqs):
            n = at + 1
            while n < len(seqs) and seqs[n] == seqs[at]:
                n += 1
            pos += self._append_run(layer, seqs[at], k[at:n], v[at:n])
            at = n
        return pos

    def _append_run(self, layer, seq, k, v):
        r = self.of(seq, layer)
        p0, n = len(r.given[0]), len(k)
        if p0 + n > self.maxpos:
            raise ValueError("context window exhausted")
        k = np.asarray(k, np.float32).reshape(n, self.nkv, self.hd)
        new = (np.stack([rope64(k[i], p0 + i, self.theta) for i in range(n)]),
               np.asarray(v, np.float32).reshape(n, self.nkv, self.hd))
        for j in range(2):
            r.given[j] = np.concatenate([r.given[j], new[j]])
            done = range(len(r.held[j]), (p0 + n) // BLOCK * BLOCK, BLOCK)
            r.held[j] = np.concatenate([r.held[j], *(hold(r.given[j][b:b + BLOCK]) for b in done)])
        r.open_block = (p0 + n - 1) // BLOCK
        return list(range(p0, p0 + n))

    def attention(self, layer, seqs, q, k, v):
        """Entries in order: contexts [n, nh * hd], and the bound of attend_one over all."""
        pos = self.append(layer, seqs, k, v)
        out, mag = [], 0.0
        for i, s in enumerate(seqs):
            c, m = self.attend_one(layer, int(s), pos[i], q[i])
            out.append(c)
            mag = max(mag, m)
        return np.stack(out), mag

    def attend_run(self, layer, seq, pos0, q):
        """attend_one of consecutive positions from pos0 on, all input finite and its scores within f32."""
        n, g, r = len(q), self.nh // self.nkv, self.of(seq, layer)
        q = np.stack([rope64(np.asarray(q[i], np.float32).reshape(self.nh, self.hd), pos0 + i, self.theta)
                      for i in range(n)]).astype(np.float64)
        end = pos0 + n
        at, key = np.arange(pos0, end)[:, None], np.arange(end)[None]
        near, seen = key // BLOCK == at // BLOCK, key <= at
        if self.win:
            seen &= key > at - self.win
        given = [x[:end].astype(np.float64) for x in r.given]
        held = [np.concatenate([h[:end], g_[len(h):end]]).astype(np.float64) for h, g_ in zip(r.held, r.given)]
        out, mag = np.empty((n, self.nh, self.hd)), 0.0
        for h in range(self.nh):
            kg, kh, vg, vh = given[0][:, h // g], held[0][:, h // g], given[1][:, h // g], held[1][:, h // g]
            s = np.where(near, q[:, h] @ kg.T, q[:, h] @ kh.T) / np.sqrt(self.hd)
            s = np.where(seen, s, -np.inf)
            w = np.exp(s - s.max(1, keepdims=True))
            w /= w.sum(1, keepdims=True)
            out[:, h] = (w * near) @ vg + (w * ~near) @ vh
            mag = max(mag, float((np.abs(q[:, h]) @ np.abs(kg).T).max() / np.sqrt(self.hd)))
        return out.reshape(n, -1), mag

    def read(self, layer, seqs, positions):
        out = [[], []]
        for s, p in zip(seqs, positions):
            r = self.of(int(s), layer)
            for j in range(2):
                out[j].append((r.held if p < len(r.held[j]) else r.given)[j][p].reshape(-1))
        return np.stack(out[0]), np.stack(out[1])

    def truncate(self, seqs, lens):
        for s, n in zip(seqs, lens):
            for layer in range(self.nl):
                r = self.of(int(s), layer)
                if len(r.given[0]) <= n:
                    continue
                b = int(n) // BLOCK
                reopened = n % BLOCK and r.open_block != b
                for j in range(2):
                    kept = r.given[j][:n].copy()
                    if reopened:
                        kept[b * BLOCK:] = r.held[j][b * BLOCK:n]
                    r.given[j] = kept
                    r.held[j] = r.held[j][:b * BLOCK]
                if reopened:
                    r.open_block = b
