"""The restatement of the KV cache held in 8 bits (oracle/attention8.py) against closed forms
and the f32 cache's restatement. No GPU."""
from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from garuda_amd import _lib
from garuda_amd.attention import GmoeKvDesc, KvCache
from oracle.attention import KvOracle, rope
from oracle.attention8 import BLOCK, Kv8Oracle, hold, rope64


def test_rotation_is_the_f32_cache_s_up_to_its_angle():
    rng = np.random.default_rng(0)
    x = rng.normal(size=(1, 64)).astype(np.float32)
    for pos in (0, 1, 7, 100):
        # the f32 angle is off by at most 2^-23 of it (frequency and product rounded), the turned pair by two roundings
        bound = np.hypot(x[0, 0::2], x[0, 1::2]).repeat(2) * (pos * 2.0 ** -22 + 2.0 ** -22)
        assert (np.abs(rope64(x, pos, 1e4)[0] - rope(x[0], pos, 1e4)) <= bound).all()
    assert np.array_equal(rope64(x, 0, 1e4), x)


def test_held_rows_are_within_half_a_step():
    rng = np.random.default_rng(1)
    x = rng.normal(size=(BLOCK, 3, 32)).astype(np.float32)
    x[:, 1] = 0
    step = np.abs(x).max(axis=(0, 2), keepdims=True) / 127
    assert (np.abs(hold(x) - x) <= step * (0.5 + 2.0 ** -16)).all()
    assert (hold(x)[:, 1] == 0).all()
    x[3, 2, 5] = np.inf
    assert np.isnan(hold(x)[:, 2]).all() and np.isfinite(hold(x)[:, :2]).all()


@pytest.mark.parametrize("window", [0, 5, 40])
def test_first_block_is_the_f32_cache(window):
    nh, nkv, hd = 4, 2, 16
    rng = np.random.default_rng(2)
    a, b = Kv8Oracle(1, nh, nkv, hd, sliding_window=window), KvOracle(1, nh, nkv, hd, sliding_window=window)
    for _ in range(BLOCK):
        q, k, v = (rng.normal(size=(1, w * hd)) for w in (nh, nkv, nkv))
        assert np.allclose(a.attention(0, [0], q, k, v)[0], b.attention(0, [0], q, k, v), rtol=1e-4, atol=1e-5)


def test_equal_values_come_back_and_truncation_reopens():
    nh, nkv, hd = 2, 1, 8
    o = Kv8Oracle(1, nh, nkv, hd)
    rng = np.random.default_rng(3)
    v = np.ones((1, hd), np.float32)
    for _ in range(40):
        got, _ = o.attention(0, [0], rng.normal(size=(1, nh * hd)), rng.normal(size=(1, hd)), v)
        assert np.allclose(got, 1.0, atol=1e-6)  # a weighted mean of equal values (127 * (1 / 127) in f32)
    k20 = o.read(0, [0], [20])[0]
    given = o.of(0, 0).given[0][20].copy()
    o.truncate([0], [21])
    assert np.array_equal(o.read(0, [0], [20])[0], k20) and not np.array_equal(k20[0], given.reshape(-1))
    o.truncate([0], [16])
    assert o.seq_len(0) == 16 and len(o.of(0, 0).held[0]) == 16


@pytest.mark.parametrize("window", [0, 30])
def test_runs_are_the_tokens_one_by_one(window):
    nh, nkv, hd = 4, 2, 16
    rng = np.random.default_rng(4)
    a, b = (Kv8Oracle(1, nh, nkv, hd, sliding_window=window) for _ in range(2))
    at = 0
    for n in (21, 1, 50, 9):
        q, k, v = (rng.normal(size=(n, w * hd)).astype(np.float32) for w in (nh, nkv, nkv))
        one, _ = a.attention(0, [0] * n, q, k, v)
        for i in range(n):
            assert b.append_one(0, 0, k[i], v[i]) == at + i
        run, _ = b.attend_run(0, 0, at, q)
        assert np.allclose(run, one, rtol=1e-12, atol=1e-12)
        at += n
    for x, y in zip(a.read(0, [0] * at, range(at)), b.read(0, [0] * at, range(at))):
        assert np.array_equal(x, y)


def test_null_arguments_are_refused_without_a_device():
    lib = _lib.lib()
    x = np.zeros(4, np.float32)
    f = x.ctypes.data_as(C.POINTER(C.c_float))
    ids = np.zeros(1, np.uint32)
    out = C.c_void_p()
    d = GmoeKvDesc()
    assert lib.gmoe_kv_create_q8(None, C.byref(d), C.byref(out)) == 2
    assert lib.gmoe_kv_append(None, 0, ids.ctypes.data, 1, f, f) == 2
    assert lib.gmoe_kv_append_async(None, 0, ids.ctypes.data, 1, x.ctypes.data, x.ctypes.data, None) == 2
    assert lib.gmoe_kv_read(None, 0, ids.ctypes.data, ids.ctypes.data, 1, f, f) == 2
    assert lib.gmoe_kv_read_async(None, 0, ids.ctypes.data, ids.ctypes.data, 1, x.ctypes.data, x.ctypes.data, None) == 2
    assert lib.gmoe_kv_truncate(None, ids.ctypes.data, ids.ctypes.data, 1, None) == 2
    assert b"null" in lib.gmoe_last_error()
    with pytest.raises(ValueError):
        KvCache(None, 1, 1, 1, 16, bits=4)
