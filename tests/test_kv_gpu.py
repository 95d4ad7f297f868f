"""The cached-attention operators on the GPU against the float64 oracle: norms and rotation, the 8-bit cache written
and read (bit for bit), attention over it, and a run of them together, eager and captured."""

from __future__ import annotations

import ctypes
from ctypes import byref, c_int, c_void_p

import numpy as np
import pytest

from kv_cases import Cached, Rows, Sequences, attend, scattered_table, starts
from oracle import kv as ok
from supra_attn import _lib

pytestmark = pytest.mark.gpu

TYPES = ["F32", "F16", "BF16"]


def near(got, want, tol, what=""):
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan, err_msg=f"{what}: NaN in other places")
    bad = ~nan & ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, worst {np.max(np.where(bad, np.abs(got - want) / tol, 0)):.3g} of the bound"


# ---- norms and rotation

def rope_call(dev, rng, T, H, Hkv, D, rot, near_pairs, dtype, norm=1, weights=True, far=4096, off=0, pad=0, in_place=False, rope_scale=0.0):
    width = (H + 2 * Hkv) * D
    ld = width + pad
    x = ok.to_type(rng.standard_normal((T, width)) * np.exp(rng.standard_normal(width)), dtype)
    packed = Rows(dev, T, width, dtype, off, ld, x)
    wq, wk = (1 + 0.3 * rng.standard_normal(D)).astype(np.float32), (1 + 0.3 * rng.standard_normal(D)).astype(np.float32)
    freq = 10000.0 ** (-np.arange(0, max(rot, 2), 2) / max(rot, 2))
    pos = rng.integers(-5, far, T).astype(np.int32)
    dw = [dev.from_array(a) for a in (wq, wk, freq, pos)]
    outs = [packed, packed] if in_place else [Rows(dev, T, H * D, dtype, off), Rows(dev, T, Hkv * D, dtype, off)]
    a = _lib.QkRopeArgs(dtype=_lib.SA_DT[dtype], T=T, H=H, Hkv=Hkv, D=D, rotary_dim=rot, pairs=int(near_pairs), norm=norm, eps=1e-6,
                        rope_scale=rope_scale, q=packed.buf.ptr, k=packed.buf.ptr, q_off=off, k_off=off + H * D, ldq=ld, ldk=ld,
                        q_out=outs[0].buf.ptr, k_out=outs[1].buf.ptr, qo_off=off, ko_off=off + H * D if in_place else off,
                        ldqo=ld if in_place else 0, ldko=ld if in_place else 0, q_weight=dw[0].ptr if weights else None,
                        k_weight=dw[1].ptr if weights else None, inv_freq=dw[2].ptr, positions=dw[3].ptr)
    _lib.qk_norm_rope(a, dev.stream)
    xv = ok.values(x, dtype)
    if in_place:
        got = packed.read((T, width))
        got_q, got_k = got[:, :H * D].reshape(T, H, D), got[:, H * D:(H + Hkv) * D].reshape(T, Hkv, D)
        np.testing.assert_array_equal(packed.raw[:, (H + Hkv) * D:], x[:, (H + Hkv) * D:], err_msg="the v columns changed")
    else:
        got_q, got_k = outs[0].read((T, H, D)), outs[1].read((T, Hkv, D))
    for got, at, n, w in ((got_q, 0, H, wq), (got_k, H * D, Hkv, wk)):
        y, size = ok.norm_rope(xv[:, at:at + n * D].reshape(T, n, D), w if weights else None, 1e-6, norm, pos, freq, rot, near_pairs, rope_scale or 1.0)
        near(got, y, ok.rope_tolerance(y, size, D, dtype), f"heads at {at}")
    for b in [packed, *outs[:0 if in_place else 2], *dw]:
        b.release()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("near_pairs", [False, True])
@pytest.mark.parametrize("T,H,Hkv,D,rot", [(1, 32, 8, 128, 128), (5, 9, 9, 64, 32), (33, 3, 1, 256, 64), (7, 2, 2, 80, 80), (3, 5, 1, 2, 2),
                                           (2, 1, 1, 512, 512), (4, 2, 1, 96, 20), (2, 0, 3, 64, 64), (2, 3, 0, 64, 0), (300, 4, 2, 128, 128)])
def test_norm_rope(dev, dtype, near_pairs, T, H, Hkv, D, rot):
    rope_call(dev, np.random.default_rng(T * 1000 + D + rot), T, H, Hkv, D, rot, near_pairs, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kw", [dict(off=1), dict(pad=3), dict(off=8, pad=16), dict(norm=0), dict(weights=False), dict(norm=0, weights=False),
                                dict(far=1 << 30), dict(in_place=True), dict(in_place=True, off=3, pad=5), dict(rope_scale=1.25)], ids=str)
def test_norm_rope_forms(dev, dtype, kw):
    for near_pairs in (False, True):
        rope_call(dev, np.random.default_rng(7), 19, 6, 2, 128, 64, near_pairs, dtype, **kw)


def test_norm_rope_many_tokens(dev):
    """More waves than a token's heads give work: the run of all heads in one wave, and the cut ones, agree bit for bit."""
    rng = np.random.default_rng(3)
    H, Hkv, D = 7, 2, 64
    T = 5000
    x = ok.to_type(rng.standard_normal((T, (H + Hkv) * D)), "BF16")
    pos, freq = np.arange(T, dtype=np.int32), 10000.0 ** (-np.arange(0, D, 2) / D)
    b = [dev.from_array(a) for a in (x, pos, freq)]
    out = dev.empty(x.shape, np.uint16)

    def call(t0, n):
        _lib.qk_norm_rope(_lib.QkRopeArgs(dtype=_lib.SA_DT["BF16"], T=n, H=H, Hkv=Hkv, D=D, rotary_dim=D, norm=1, eps=1e-6, q=b[0].ptr, k=b[0].ptr,
                                          q_off=t0 * x.shape[1], k_off=t0 * x.shape[1] + H * D, ldq=x.shape[1], ldk=x.shape[1], q_out=out.ptr, k_out=out.ptr,
                                          qo_off=t0 * x.shape[1], ko_off=t0 * x.shape[1] + H * D, ldqo=x.shape[1], ldko=x.shape[1], inv_freq=b[2].ptr,
                                          positions=b[1].ptr + 4 * t0), dev.stream)
        return out.read()[t0:t0 + n]

    whole = call(0, T)
    for t0, n in ((0, 1), (17, 100), (4990, 10)):
        np.testing.assert_array_equal(call(t0, n), whole[t0:t0 + n])


# ---- the cache

def same_cache(got: ok.Cache, want: ok.Cache, what=""):
    np.testing.assert_array_equal(got.exp, want.exp, err_msg=f"{what}: exponents")
    a, b = got.codes.copy(), want.codes.copy()
    a[a & 127 == 127] = b[b & 127 == 127] = 127  # any NaN code
    np.testing.assert_array_equal(a, b, err_msg=f"{what}: codes")


def write_call(dev, cached, seqs, k, v, dtype, off=0, pad=0):
    T, width = seqs.oracle.T, cached.oracle.Hkv * cached.oracle.D
    ld = width + pad if pad else 0
    rk, rv = (Rows(dev, T, width, dtype, off, ld, x) for x in (k, v))
    _lib.kv_write(_lib.KvRowsArgs(dtype=_lib.SA_DT[dtype], cache=cached.desc, seqs=seqs.desc, k=rk.buf.ptr, v=rv.buf.ptr, k_off=off, v_off=off,
                                  ldk=ld, ldv=ld), dev.stream)
    dev.sync()
    rk.release()
    rv.release()


def read_call(dev, cached, seqs, dtype, off=0, pad=0):
    T, width = seqs.oracle.T, cached.oracle.Hkv * cached.oracle.D
    ld = width + pad if pad else 0
    rk, rv = (Rows(dev, T, width, dtype, off, ld) for _ in range(2))
    _lib.kv_read(_lib.KvRowsArgs(dtype=_lib.SA_DT[dtype], cache=cached.desc, seqs=seqs.desc, k=rk.buf.ptr, v=rv.buf.ptr, k_off=off, v_off=off,
                                 ldk=ld, ldv=ld), dev.stream)
    shape = (T, cached.oracle.Hkv, cached.oracle.D)
    return rk.read(shape), rv.read(shape), rk, rv


def rows_data(rng, T, Hkv, D, dtype, wild):
    x = rng.standard_normal((T, Hkv, D)) * np.exp2(rng.integers(-6, 7, (T, 1, 1)))
    if wild and x.size:
        x *= np.exp2(rng.integers(-12, 4, x.shape))
        flat = x.reshape(-1)
        for val in (np.nan, np.inf, -np.inf, 0.0, -0.0, 448.0, 448.0 * (1 + 2.0 ** -7), 2.0 ** -10, 3 * 2.0 ** -10):
            flat[rng.integers(0, flat.size, 2)] = val
    return ok.to_type(x.reshape(T, Hkv * D), dtype)


SEQUENCES = {  # rows and lengths of the sequences of one call
    "tokens": ([1, 1, 1, 1, 1, 1], [1, 2, 32, 33, 64, 100]),
    "prompts": ([5, 0, 32, 33, 64, 71], [5, 40, 32, 40, 95, 71]),
    "inside": ([1, 3, 30, 34, 2], [31, 20, 63, 65, 34]),
    "long": ([300, 1], [317, 450]),
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("form", list(SEQUENCES))
def test_write_and_read(dev, dtype, D, form):
    """Codes, exponents and untouched bytes equal the oracle's; so do the values read back, over a cache full of old
    bytes (pages are used again)."""
    rng = np.random.default_rng(D + len(form))
    rows, lens = SEQUENCES[form]
    Hkv, T = 3, sum(rows) + 2
    pages = sum(-(-n // 32) for n in lens) + 3
    cache = ok.Cache(pages, Hkv, D, rng)
    cache.exp = rng.integers(118, 132, cache.exp.shape).astype(np.uint8)  # old scales near the new ones: some grow, some not
    cached = Cached(dev, cache)
    seqs = Sequences(dev, ok.Seqs(lens, scattered_table(rng, lens, pages), T, max(rows), starts(rows)))
    k, v = (rows_data(rng, T, Hkv, D, dtype, True) for _ in range(2))
    write_call(dev, cached, seqs, k, v, dtype)
    cache.write(seqs.oracle, *(ok.values(x, dtype).reshape(T, Hkv, D) for x in (k, v)))
    same_cache(cached.now(), cache, form)
    whole = Sequences(dev, ok.Seqs(lens, seqs.oracle.table, sum(lens) + 1, max(lens), starts(lens)))
    gk, gv, rk, rv = read_call(dev, cached, whole, dtype)
    wk, wv, mine = cache.read(whole.oracle, whole.oracle.T)
    for got, want, r in ((gk, wk, rk), (gv, wv, rv)):
        np.testing.assert_array_equal(got[mine], ok.values(ok.to_type(want[mine], dtype), dtype))
        assert r.untouched(~mine)
    for x in (cached, seqs, whole, rk, rv):
        x.release()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("off,pad", [(1, 0), (0, 7), (8, 8), (3, 5)])
def test_write_and_read_any_alignment(dev, dtype, off, pad):
    rng = np.random.default_rng(off * 10 + pad)
    rows, lens, Hkv, D = [40, 3], [50, 3], 2, 64
    cache = ok.Cache(5, Hkv, D)
    cached = Cached(dev, cache)
    seqs = Sequences(dev, ok.Seqs(lens, scattered_table(rng, lens, 5), 43, 40, starts(rows)))
    k, v = (rows_data(rng, 43, Hkv, D, dtype, False) for _ in range(2))
    write_call(dev, cached, seqs, k, v, dtype, off, pad)
    cache.write(seqs.oracle, *(ok.values(x, dtype).reshape(43, Hkv, D) for x in (k, v)))
    same_cache(cached.now(), cache)
    gk, gv, rk, rv = read_call(dev, cached, seqs, dtype, off, pad)
    wk, wv, mine = cache.read(seqs.oracle, 43)
    np.testing.assert_array_equal(gk[mine], ok.values(ok.to_type(wk[mine], dtype), dtype))
    np.testing.assert_array_equal(gv[mine], ok.values(ok.to_type(wv[mine], dtype), dtype))
    for x in (cached, seqs, rk, rv):
        x.release()


def test_token_by_token_is_the_oracle_token_by_token(dev):
    """A page filled one token at a time, its scale growing and not: every state on the way."""
    rng = np.random.default_rng(5)
    Hkv, D = 2, 64
    cache = ok.Cache(2, Hkv, D, rng)
    cached = Cached(dev, cache)
    for n in range(1, 36):
        seqs = Sequences(dev, ok.Seqs([n], [[1, 0]], 1, 1))
        k, v = (ok.to_type(rng.standard_normal((1, Hkv * D)) * 2.0 ** rng.integers(-8, 6), "BF16") for _ in range(2))
        write_call(dev, cached, seqs, k, v, "BF16")
        cache.write(seqs.oracle, *(ok.values(x, "BF16").reshape(1, Hkv, D) for x in (k, v)))
        same_cache(cached.now(), cache, f"after {n} tokens")
        seqs.release()
    cached.release()


@pytest.mark.parametrize("scale", [2.0 ** -149, 2.0 ** -130, 2.0 ** -119, 2.0 ** 100, 2.0 ** 127, 0.0])
def test_extreme_magnitudes(dev, scale):
    rng = np.random.default_rng(2)
    cache = ok.Cache(2, 1, 64, rng)
    cached = Cached(dev, cache)
    seqs = Sequences(dev, ok.Seqs([40], [[1, 0]], 40, 40))
    k, v = ((rng.uniform(-1.9, 1.9, (40, 64)) * scale).astype(np.float32) for _ in range(2))
    write_call(dev, cached, seqs, k, v, "F32")
    cache.write(seqs.oracle, *(x.astype(np.float64).reshape(40, 1, 64) for x in (k, v)))
    same_cache(cached.now(), cache)
    gk, gv, rk, rv = read_call(dev, cached, seqs, "F32")
    wk, wv, _ = cache.read(seqs.oracle, 40)
    np.testing.assert_array_equal(gk, wk)
    np.testing.assert_array_equal(gv, wv)
    for x in (cached, seqs, rk, rv):
        x.release()


def test_bounds_of_the_device_arrays(dev):
    """Pages outside the cache, negative and too large lengths, rows past T, rows at negative positions: what they say
    is dropped, read as zeros or passed over, and nothing outside the arrays changes."""
    rng = np.random.default_rng(9)
    Hkv, D, pages, T = 2, 64, 6, 90
    lens = [70, 33, -4, 1000, 10, 5]
    table = np.array([[3, 1 << 30, 5], [-1, 0, 2], [1, 1, 1], [4, -(1 << 31), 6], [1, -7, 9], [2, 9, 9]], np.int32)
    row_start = np.array([5, 0, 20, 25, 60, 85, 200], np.int32)  # the first: backwards; the last: past T
    seqs = Sequences(dev, ok.Seqs(lens, table, T, 36, row_start))
    cache = ok.Cache(pages, Hkv, D, rng)
    cache.exp = rng.integers(120, 130, cache.exp.shape).astype(np.uint8)
    cached = Cached(dev, cache)
    k, v = (rows_data(rng, T, Hkv, D, "F32", False) for _ in range(2))
    write_call(dev, cached, seqs, k, v, "F32")
    cache.write(seqs.oracle, *(ok.values(x, "F32").reshape(T, Hkv, D) for x in (k, v)))
    same_cache(cached.now(), cache)
    gk, gv, rk, rv = read_call(dev, cached, seqs, "F32")
    wk, wv, mine = cache.read(seqs.oracle, T)
    np.testing.assert_array_equal(gk[mine], wk[mine])
    np.testing.assert_array_equal(gv[mine], wv[mine])
    assert rk.untouched(~mine) and rv.untouched(~mine)
    for causal in (False, True):
        q = ok.to_type(rng.standard_normal((T, 4 * D)), "F32")
        got, ro, _ = attend(dev, cached, seqs, q, 4, "F32", D ** -0.5, causal)
        o, size, reach, count, mine = cache.attention(seqs.oracle, q.astype(np.float64).reshape(T, 4, D), D ** -0.5, causal)
        near(got[mine], o[mine], ok.attention_tolerance(o, size, reach, count, D, "F32")[mine], f"causal {causal}")
        assert ro.untouched(~mine)
        ro.release()
    for x in (cached, seqs, rk, rv):
        x.release()


# ---- attention

def filled(rng, dev, lens, Hkv, D, spread=2, pages=None, extra=1):
    """A cache with random codes (NaN codes in every place that no sequence holds) and page scales 2^spread apart."""
    pages = pages or sum(-(-max(n, 0) // 32) for n in lens) + 2
    cache = ok.Cache(pages, Hkv, D, rng)
    cache.codes[cache.codes & 127 == 127] = 0x30
    cache.codes = np.where(rng.random(cache.codes.shape) < 0.5, cache.codes & 0x87 | 0x30, cache.codes & 0xBF)
    cache.exp = rng.integers(124 - spread, 125 + spread, cache.exp.shape).astype(np.uint8)
    table = scattered_table(rng, lens, pages, extra)
    held = np.zeros((pages, ok.BLOCK), bool)
    for b, n in enumerate(lens):
        for j in range(max(n, 0)):
            held[table[b, j // 32], j % 32] = True
    cache.codes[:, ~held[:, None].repeat(Hkv, 1)] = 0xFF
    return cache, table


def check_attention(dev, rng, rows, lens, H, Hkv, D, dtype, causal, T=None, spread=2, q_scale=1.0, max_len=0, uniform=False, extra=1, **kw):
    cache, table = filled(rng, dev, lens, Hkv, D, spread, extra=extra)
    cached = Cached(dev, cache)
    T = T or sum(rows) + 1
    seqs = Sequences(dev, ok.Seqs(lens, table, T, max(rows), None if uniform else starts(rows)))
    q = ok.to_type(rng.standard_normal((T, H * D)) * q_scale, dtype)
    scale = float(np.float32(D ** -0.5))
    got, ro, splits = attend(dev, cached, seqs, q, H, dtype, scale, causal, max_len, **kw)
    o, size, reach, count, mine = cache.attention(seqs.oracle, ok.values(q, dtype).reshape(T, H, D), scale, causal)
    near(got[mine], o[mine], ok.attention_tolerance(o, size, reach, count, D, dtype)[mine])
    assert ro.untouched(~mine)
    for x in (cached, seqs, ro):
        x.release()
    return splits


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("H,Hkv", [(3, 3), (8, 2), (7, 1)])
def test_attention_tokens(dev, dtype, D, H, Hkv):
    """A decoding step: lengths of none, one and the edges of pages."""
    check_attention(dev, np.random.default_rng(D + H), [1] * 8, [0, 1, 2, 31, 32, 33, 100, 290], H, Hkv, D, dtype, True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_prompts(dev, dtype, D, causal):
    """Ragged rows, more rows than keys among them (rows at negative positions attend to nothing when causal)."""
    check_attention(dev, np.random.default_rng(D), [5, 0, 40, 33, 70, 1], [5, 40, 33, 97, 130, 64], 4, 2, D, dtype, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_attention_many_rows(dev, dtype, causal):
    """Enough rows for whole workgroups of them, past a cached prefix, and one head per key head."""
    check_attention(dev, np.random.default_rng(1), [150, 260], [300, 260], 2, 2, 64, dtype, causal)
    check_attention(dev, np.random.default_rng(2), [130], [450], 4, 1, 128, dtype, causal)


def test_attention_splits_and_their_merge(dev):
    """Few rows and many keys: the keys are split over workgroups; max_len shapes that and changes nothing else."""
    rng = np.random.default_rng(4)
    for dtype in TYPES:
        assert check_attention(dev, rng, [1, 2], [2500, 40], 4, 2, 64, dtype, True) > 1
    assert check_attention(dev, rng, [1], [2500], 2, 1, 128, "BF16", True, max_len=2500) > 1
    assert check_attention(dev, rng, [1], [2500], 2, 1, 128, "BF16", True, max_len=1) == 1
    lens = [int(n) for n in rng.integers(1, 500, 20)]
    assert check_attention(dev, rng, [1] * 20, lens, 8, 4, 64, "F16", True, max_len=500) == 1  # eight waves a workgroup
    assert check_attention(dev, rng, [1] * 20, lens, 8, 4, 64, "F16", True, extra=70) > 1
    assert check_attention(dev, rng, [3] * 20, [n + 3 for n in lens], 32, 4, 64, "F32", True, extra=70) == 1  # two groups of 16 rows
    assert check_attention(dev, rng, [5] * 33, [n % 97 + 300 for n in range(33)], 32, 8, 64, "F32", True, max_len=400) > 1  # 32 rows
    assert check_attention(dev, rng, [5] * 33, [n % 97 + 300 for n in range(33)], 32, 8, 128, "BF16", True, max_len=400) > 1
    assert check_attention(dev, rng, [9] * 10, [n % 7 + 300 for n in range(10)], 32, 8, 128, "F16", True, max_len=400) == 1  # in eight waves
    assert check_attention(dev, rng, [1] * 10, lens[:10], 4, 4, 128, "BF16", True, max_len=500) == 1  # few pages in eight waves
    assert check_attention(dev, rng, [1] * 10, [n + 900 for n in lens[:10]], 4, 4, 128, "BF16", True, max_len=1400) > 1  # four waves
    assert check_attention(dev, rng, [1] * 10, lens[:10], 4, 4, 256, "BF16", True, max_len=500) > 1  # wide heads
    assert check_attention(dev, rng, [5, 1], [300, 290], 8, 2, 64, "F32", True, max_len=300) == 1  # two groups in eight waves
    assert check_attention(dev, rng, [1, 1], [256, 257], 2, 1, 128, "F16", True, max_len=257) == 1  # nine pages
    assert check_attention(dev, rng, [100], [600], 2, 1, 64, "F16", True) == 1
    for dtype in TYPES:
        assert check_attention(dev, rng, [100], [600], 2, 1, 256, dtype, True) > 1  # 128 rows each
    assert check_attention(dev, rng, [35, 7, 34], [600, 3000, 41], 9, 1, 64, "BF16", True) > 1  # groups of 16 rows of three sequences


@pytest.mark.parametrize("B", [2, 3, 33, 64, 65])
@pytest.mark.parametrize("G,causal", [(1, True), (3, True), (2, False)])
def test_attention_of_ragged_prompts(dev, B, G, causal):
    """Prompts of many lengths in one call, whose workgroups are taken by their pages (up to 64 sequences): without rows,
    of one, all of a sequence's tokens, more rows than tokens, no tokens, the same length twice, longer than max_len says."""
    rng = np.random.default_rng(23 + B)
    rows = [int(r) for r in rng.integers(0, 60 if B > 3 else 400, B)]
    lens = [int(n) for n in rng.integers(1, 1300, B)]
    rows[0], lens[0], rows[1], lens[1] = 300, 1290, 260, 260
    if B > 6:
        rows[2], rows[3], rows[4], lens[4], rows[5], lens[5], lens[6] = 0, 1, 45, 20, 33, 0, lens[7]
    for dtype, D, max_len in (("BF16", 64, 0), ("F16", 128, 1100), ("F32", 64, 1024)):
        check_attention(dev, rng, rows, lens, G, 1, D, dtype, causal, max_len=max_len)
    if B == 3:
        check_attention(dev, rng, rows, lens, 2 * G, 2, 256, "BF16", causal, extra=40)  # the keys split too


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_forms(dev, dtype):
    """Uniform rows without row_start; odd offsets and strides of q and o; large and tiny queries; scales far apart."""
    rng = np.random.default_rng(6)
    check_attention(dev, rng, [3, 3, 3], [50, 3, 64], 4, 2, 64, dtype, True, uniform=True, T=10)
    for off, ld, o_off, ldo in ((1, 0, 0, 0), (0, 259, 0, 0), (0, 0, 3, 0), (0, 0, 0, 261), (5, 263, 7, 257)):
        check_attention(dev, rng, [3, 2], [50, 33], 4, 2, 64, dtype, True, off=off, ld=ld, o_off=o_off, ldo=ldo)
    check_attention(dev, rng, [2, 40], [100, 70], 4, 2, 64, dtype, False, q_scale=2.0 ** -12)
    check_attention(dev, rng, [2, 40], [100, 70], 4, 2, 64, dtype, False, q_scale=4.0)
    check_attention(dev, rng, [2, 40], [100, 70], 2, 1, 64, dtype, True, spread=8, q_scale=2.0 ** -6)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_nan_where_it_is_not_attended(dev, dtype):
    """NaN codes at tokens behind a row's position leave the row alone, and reach the rows that attend to them."""
    rng = np.random.default_rng(8)
    for D in (64, 128, 256):
        cache, table = filled(rng, dev, [70], 1, D)
        cache.codes[1, table[0, 1], 0, 20, 3] = 0x7F   # V of token 52
        cache.codes[0, table[0, 2], 0, 2, 5] = 0xFF    # K of token 66
        cached = Cached(dev, cache)
        seqs = Sequences(dev, ok.Seqs([70], table, 70, 70, [0, 70]))
        q = ok.to_type(rng.standard_normal((70, 2 * D)), dtype)
        got, ro, _ = attend(dev, cached, seqs, q, 2, dtype, D ** -0.5, True)
        o, size, reach, count, mine = cache.attention(seqs.oracle, ok.values(q, dtype).reshape(70, 2, D), D ** -0.5, True)
        assert np.isfinite(o[:52]).all() and np.isnan(o[52:, :, 3]).all() and np.isfinite(o[52:66, :, 4]).all() and np.isnan(o[66:]).all()
        near(got, o, ok.attention_tolerance(o, size, reach, count, D, dtype), f"D {D}")
        for x in (cached, seqs, ro):
            x.release()
        # a few rows, in tiles of 16
        seqs = Sequences(dev, ok.Seqs([70], table, 20, 20, [0, 20]))
        cached = Cached(dev, cache)
        got, ro, _ = attend(dev, cached, seqs, q[:20, :D], 1, dtype, D ** -0.5, True)
        o, size, reach, count, mine = cache.attention(seqs.oracle, ok.values(q[:20, :D], dtype).reshape(20, 1, D), D ** -0.5, True)
        assert np.isfinite(o[:2]).all() and np.isnan(o[2:, :, 3]).all() and np.isfinite(o[2:16, :, 4]).all() and np.isnan(o[16:]).all()
        near(got, o, ok.attention_tolerance(o, size, reach, count, D, dtype), f"D {D}, 20 rows")
        for x in (cached, seqs, ro):
            x.release()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_queries_of_every_size(dev, dtype):
    """Elements of a row from 2^-9 to 2^5 of each other, rows of zeros, infinities and NaN, a negative scale."""
    rng = np.random.default_rng(13)
    D, n, H = 128, 90, 2
    cache, table = filled(rng, dev, [100], 1, D)
    cached = Cached(dev, cache)
    for rows in (n, 7):
        x = rng.standard_normal((rows, H * D)) * np.exp2(rng.integers(-9, 6, (rows, H * D))) / 4
        x[1], x[2, 5], x[3, D + 7], x[4, 3] = 0, np.inf, np.nan, -np.inf
        q = ok.to_type(x, dtype)
        seqs = Sequences(dev, ok.Seqs([100], table, rows, rows))
        for scale in (0.0625, -0.0625, 0.0):
            got, ro, _ = attend(dev, cached, seqs, q, H, dtype, scale, True)
            qv = ok.values(q, dtype).reshape(rows, H, D)
            with np.errstate(invalid="ignore"):
                o, size, reach, count, _ = cache.attention(seqs.oracle, qv, scale, True)
            o[~np.isfinite(qv).all(-1)] = np.nan  # inf - inf, or 0 * inf, in the scores
            near(got, o, ok.attention_tolerance(o, size, reach, count, D, dtype), f"rows {rows} scale {scale}")
            ro.release()
        seqs.release()
    cached.release()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("sign", [1, -1])
def test_attention_of_infinite_scores(dev, dtype, D, sign):
    """An infinity in a row makes each of its scores infinite, here all of one sign: the row is NaN, whichever it is (the
    differences of equal infinities), where it attends to anything; the other rows are as ever."""
    rng = np.random.default_rng(19)
    for rows, n in ((1, 40), (3, 40), (20, 40), (90, 40), (1, 2500)):
        cache, table = filled(rng, dev, [n], 1, D)
        cache.codes[0, :, :, :, 0] = 0xB8  # K's first element: -1, in every place
        cached = Cached(dev, cache)
        x = rng.standard_normal((rows, 2 * D))
        x[rows // 2, D] = sign * np.inf
        q = ok.to_type(x, dtype)
        for causal in (False, True):
            seqs = Sequences(dev, ok.Seqs([n], table, rows, rows))
            got, ro, _ = attend(dev, cached, seqs, q, 2, dtype, 0.125, causal)
            qv = ok.values(q, dtype).reshape(rows, 2, D)
            with np.errstate(invalid="ignore"):
                o, size, reach, count, _ = cache.attention(seqs.oracle, qv, 0.125, causal)
            o[(~np.isfinite(qv).all(-1)) & (count > 0)[:, None]] = np.nan
            near(got, o, ok.attention_tolerance(o, size, reach, count, D, dtype), f"rows {rows} of {n} causal {causal}")
            ro.release()
            seqs.release()
        cached.release()


class Wider(ok.Seqs):
    """The same sequences under a bound of many more rows, which gives them to the kernel of 128 rows a workgroup."""

    def __init__(self, seq_len, table, T, max_rows, row_start=None):
        if row_start is None:
            row_start = np.minimum(np.arange(len(seq_len) + 1) * max_rows, T)
        super().__init__(seq_len, table, T, 80000, row_start)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_few_rows_as_of_many(dev, dtype, monkeypatch):
    """The kernel of many rows on the rows, masks, NaN codes and queries that the other tests give the kernel of few."""
    monkeypatch.setattr(ok, "Seqs", Wider)
    for D in (64, 128, 256):
        test_attention_tokens(dev, dtype, D, 7, 1)
        for causal in (True, False):
            test_attention_prompts(dev, dtype, D, causal)
        test_attention_of_infinite_scores(dev, dtype, D, -1)
    test_attention_forms(dev, dtype)
    test_attention_nan_where_it_is_not_attended(dev, dtype)
    test_attention_queries_of_every_size(dev, dtype)


@pytest.mark.parametrize("B", [3, 64])
@pytest.mark.parametrize("G,causal", [(1, True), (3, True), (2, False)])
def test_attention_of_ragged_prompts_as_of_many(dev, B, G, causal, monkeypatch):
    """Their workgroups by their pages: the order is the kernel of many rows' alone."""
    monkeypatch.setattr(ok, "Seqs", Wider)
    test_attention_of_ragged_prompts(dev, B, G, causal)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_of_many_rows_in_many_heads(dev, dtype, causal):
    """More than 512 workgroups of 128 rows by the call's own sizes."""
    rng = np.random.default_rng(29)
    check_attention(dev, rng, [131], [200], 257, 257, 64, dtype, causal)
    check_attention(dev, rng, [65, 2], [70, 40], 258, 129, 128, dtype, causal)


def test_without_pages_and_with_shared_ones(dev):
    """No column in the block table: rows of zeros. One page in the tables of 70000 sequences: the same row for each."""
    rng = np.random.default_rng(17)
    D = 64
    cache, _ = filled(rng, dev, [32], 1, D)
    cache.codes[cache.codes & 127 == 127] = 0x30
    cached = Cached(dev, cache)
    q = ok.to_type(rng.standard_normal((3, D)), "BF16")
    for rows in (1, 3):
        none = Sequences(dev, ok.Seqs([50] * (3 // rows), np.zeros((3 // rows, 0), np.int32), 3, rows))
        none.desc.max_blocks = 0
        got, ro, _ = attend(dev, cached, none, q, 1, "BF16", 0.125, False)
        assert (got == 0).all()
        gk, gv, rk, rv = read_call(dev, cached, none, "BF16")
        assert (gk == 0).all() and (gv == 0).all()
        write_call(dev, cached, none, q, q, "BF16")  # nowhere to
        same_cache(cached.now(), cache)
        for x in (none, ro, rk, rv):
            x.release()
    B = 70000
    many = Sequences(dev, ok.Seqs([20] * B, np.zeros((B, 1), np.int32), B, 1))
    got, ro, _ = attend(dev, cached, many, np.repeat(q[:1], B, 0), 1, "BF16", 0.125, True)
    assert (got == got[:1]).all()
    o, size, reach, count, _ = cache.attention(ok.Seqs([20], [[0]], 1, 1), ok.values(q[:1], "BF16").reshape(1, 1, D), 0.125, True)
    near(got[:1], o, ok.attention_tolerance(o, size, reach, count, D, "BF16"))
    gk, gv, rk, rv = read_call(dev, cached, many, "F32")
    wk, wv, _ = cache.read(ok.Seqs([20], [[0]], 1, 1), 1)
    assert (gk == wk).all() and (gv == wv).all()
    for x in (cached, many, ro, rk, rv):
        x.release()


def test_pages_beyond_32_bit_offsets(dev):
    """A cache of more than 4 GiB for K and for V: its last pages are written, read and attended to."""
    rng = np.random.default_rng(11)
    Hkv, D, n = 8, 256, 70
    pages = (1 << 32) // (Hkv * 32 * D) + 4
    k, v = (dev.empty([_lib.kv_cache_bytes(pages, Hkv, D)], np.uint8) for _ in range(2))
    ks, vs = (dev.empty([pages * Hkv], np.uint8) for _ in range(2))
    desc = _lib.KvCache(pages=pages, Hkv=Hkv, D=D, k=k.ptr, v=v.ptr, k_scale=ks.ptr, v_scale=vs.ptr)
    far = [pages - 1, pages - 2, pages - 4]
    seqs = Sequences(dev, ok.Seqs([n], [far], n, n))
    small = ok.Cache(3, Hkv, D)
    kk, vv = (rows_data(rng, n, Hkv, D, "BF16", False) for _ in range(2))
    small.write(ok.Seqs([n], [[0, 1, 2]], n, n), *(ok.values(x, "BF16").reshape(n, Hkv, D) for x in (kk, vv)))
    big = type("Big", (), dict(desc=desc, oracle=small))()
    write_call(dev, big, seqs, kk, vv, "BF16")
    gk, gv, rk, rv = read_call(dev, big, seqs, "BF16")
    wk, wv, _ = small.read(ok.Seqs([n], [[0, 1, 2]], n, n), n)
    np.testing.assert_array_equal(gk, wk)
    np.testing.assert_array_equal(gv, wv)
    q = ok.to_type(rng.standard_normal((n, Hkv * D)) / 64, "BF16")
    got, ro, _ = attend(dev, big, seqs, q, Hkv, "BF16", D ** -0.5, True)
    o, size, reach, count, _ = small.attention(ok.Seqs([n], [[0, 1, 2]], n, n), ok.values(q, "BF16").reshape(n, Hkv, D), D ** -0.5, True)
    near(got, o, ok.attention_tolerance(o, size, reach, count, D, "BF16"))
    for x in (k, v, ks, vs, seqs, rk, rv, ro):
        x.release()


# ---- a run of them together

def _hip():
    hip = ctypes.CDLL("libamdhip64.so.7")  # the runtime libsupra_attn.so links
    for name, args in (("hipStreamBeginCapture", [c_void_p, c_int]), ("hipStreamEndCapture", [c_void_p, c_void_p]),
                       ("hipGraphInstantiate", [c_void_p, c_void_p, c_void_p, c_void_p, ctypes.c_size_t]),
                       ("hipGraphLaunch", [c_void_p, c_void_p]), ("hipGraphExecDestroy", [c_void_p]), ("hipGraphDestroy", [c_void_p])):
        fn = getattr(hip, name)
        fn.restype = c_int
        fn.argtypes = args
    return hip


class Layer:
    """q|k|v projection, norms and rotation in place, cache write, attention: one layer's first half, over B sequences."""

    def __init__(self, dev, rng, B, H, Hkv, D, C, pages, max_blocks, table, T, max_rows, max_len):
        W = (H + 2 * Hkv) * D
        f = lambda *s, std=1.0: (rng.standard_normal(s) * std).astype(np.float32)
        self.dev, self.dims = dev, (B, H, Hkv, D, C, W)
        self.w, self.b = f(W, C, std=C ** -0.5), f(W, std=0.1)
        self.wq, self.wk = 1 + f(D, std=0.2), 1 + f(D, std=0.2)
        self.freq = 10000.0 ** (-np.arange(0, D, 2) / D)
        self.cache = ok.Cache(pages, Hkv, D, rng)
        self.cached = Cached(dev, self.cache)
        up = dev.from_array
        self.dw = [up(x) for x in (self.w, self.b, self.wq, self.wk, self.freq)]
        self.x, self.qkv, self.o = dev.empty((T, C)), dev.empty((T, W)), dev.empty((T, H * D))
        self.pos, self.len, self.start = dev.empty([T], np.int32), dev.empty([B], np.int32), dev.empty([B + 1], np.int32)
        self.table_host, self.table = table, up(table)
        self.T = T
        seqs = _lib.KvSeqs(B=B, T=T, max_rows=max_rows, max_blocks=max_blocks, row_start=self.start.ptr, seq_len=self.len.ptr, block_table=self.table.ptr)
        f32 = _lib.SA_DT["F32"]
        p = self.qkv.ptr
        self.lin = _lib.LinearArgs(M=T, N=W, K=C, x=self.x.ptr, w=self.dw[0].ptr, bias=self.dw[1].ptr, y=p)
        self.rope = _lib.QkRopeArgs(dtype=f32, T=T, H=H, Hkv=Hkv, D=D, rotary_dim=D, norm=1, eps=1e-6, q=p, k=p, k_off=H * D, ldq=W, ldk=W, q_out=p,
                                    k_out=p, ko_off=H * D, ldqo=W, ldko=W, q_weight=self.dw[2].ptr, k_weight=self.dw[3].ptr, inv_freq=self.dw[4].ptr,
                                    positions=self.pos.ptr)
        self.write = _lib.KvRowsArgs(dtype=f32, cache=self.cached.desc, seqs=seqs, k=p, v=p, k_off=H * D, v_off=(H + Hkv) * D, ldk=W, ldv=W)
        self.attn = _lib.KvAttnArgs(dtype=f32, cache=self.cached.desc, seqs=seqs, H=H, causal=1, scale=D ** -0.5, max_len=max_len, q=p, ldq=W, o=self.o.ptr)
        need = _lib.kv_attention_workspace_bytes(self.attn)
        self.ws = dev.empty([max(need, 16)], np.uint8)
        self.attn.workspace, self.attn.workspace_bytes = self.ws.ptr, need

    def inputs(self, x, lens, rows):
        self.x.upload(x)
        self.len.upload(np.asarray(lens, np.int32))
        self.start.upload(starts(rows))
        pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)] + [np.zeros(self.T - sum(rows), np.int64)])
        self.pos.upload(pos.astype(np.int32))
        return pos

    def launch(self):
        s = self.dev.stream
        _lib.linear(self.lin, s)
        _lib.qk_norm_rope(self.rope, s)
        _lib.kv_write(self.write, s)
        _lib.kv_attention(self.attn, s)

    def release(self):
        for b in (*self.dw, self.x, self.qkv, self.o, self.pos, self.len, self.start, self.table, self.ws, self.cached):
            b.release()

    def expect(self, x, lens, rows):
        """The oracle's result and bound for the rows, its cache left as after the call. The device's own projected and
        rotated rows (checked against float64 first) are what enters the cache: a rounding of them may move a code."""
        B, H, Hkv, D, C, W = self.dims
        pos = np.concatenate([np.arange(n - r, n) for n, r in zip(lens, rows)])
        n = len(pos)
        y = x[:n].astype(np.float64) @ self.w.T.astype(np.float64) + self.b
        lin_tol = (C + 4) * 2.0 ** -24 * (np.abs(x[:n]).astype(np.float64) @ np.abs(self.w.T).astype(np.float64) + np.abs(self.b))
        got = self.qkv.read()[:n].astype(np.float64)
        for at, heads, wt in ((0, H, self.wq), (H * D, Hkv, self.wk)):
            part, tol = y[:, at:at + heads * D].reshape(n, heads, D), lin_tol[:, at:at + heads * D].reshape(n, heads, D)
            want, size = ok.norm_rope(part, wt, 1e-6, 1, pos, self.freq, D, False)
            # an error of the projection passes through the norm (divided by the rms, twice at most) and the rotation
            rms = np.sqrt((part ** 2).mean(-1, keepdims=True))
            through = 4 * tol.max(-1, keepdims=True) / rms * np.abs(wt).max()
            near(got[:, at:at + heads * D].reshape(n, heads, D), want, ok.rope_tolerance(want, size, D, "F32") + through, "rotated rows")
        seqs = ok.Seqs(lens, self.table_host, self.T, max(rows), starts(rows))
        pad = np.zeros((self.T, W))
        pad[:n] = got
        self.cache.write(seqs, pad[:, H * D:(H + Hkv) * D].reshape(self.T, Hkv, D), pad[:, (H + Hkv) * D:].reshape(self.T, Hkv, D))
        o, size, reach, count, mine = self.cache.attention(seqs, pad[:, :H * D].reshape(self.T, H, D), D ** -0.5, True)
        return o, ok.attention_tolerance(o, size, reach, count, D, "F32"), mine


def test_prompt_then_tokens_together(dev):
    """Two prompts, then tokens one by one: every step's attention and the whole cache against the oracle."""
    rng = np.random.default_rng(21)
    B, H, Hkv, D, C = 2, 6, 2, 64, 96
    table = np.array([[4, 0, 2], [1, 5, 3]], np.int32)
    layer = Layer(dev, rng, B, H, Hkv, D, C, 6, 3, table, 80, 64, 96)
    lens = [40, 29]
    for step, rows in enumerate([[40, 29]] + [[1, 1]] * 5):
        if step:
            lens = [n + 1 for n in lens]
        x = rng.standard_normal((layer.T, C)).astype(np.float32)
        layer.inputs(x, lens, rows)
        layer.launch()
        o, tol, mine = layer.expect(x, lens, rows)
        near(layer.o.read().reshape(layer.T, H, D)[mine], o[mine], tol[mine], f"step {step}")
        same_cache(layer.cached.now(), layer.cache, f"step {step}")
    layer.release()


def test_a_decoding_step_in_a_graph(dev):
    """The four calls captured once; replays with new inputs, lengths and pages in the same buffers equal eager calls."""
    rng = np.random.default_rng(22)
    B, H, Hkv, D, C = 3, 4, 1, 128, 64
    table = rng.permutation(3 * 80).reshape(3, 80).astype(np.int32)
    layer = Layer(dev, rng, B, H, Hkv, D, C, 240, 80, table, B, 1, 0)
    assert layer.attn.workspace_bytes > 0  # the keys are split: two launches and a workspace in the graph
    rows, lens = [1, 1, 1], [300, 33, 1]
    x = rng.standard_normal((B, C)).astype(np.float32)
    layer.inputs(x, lens, rows)
    layer.launch()
    layer.expect(x, lens, rows)
    hip, s = _hip(), c_void_p(dev.stream)
    graph, exe = c_void_p(), c_void_p()
    dev.sync()
    assert hip.hipStreamBeginCapture(s, 0) == 0
    try:
        layer.launch()
    finally:
        rc = hip.hipStreamEndCapture(s, byref(graph))
    assert rc == 0 and graph.value
    assert hip.hipGraphInstantiate(byref(exe), graph, None, None, 0) == 0
    try:
        for rep in range(5):
            lens = [n + 1 for n in lens]
            x = rng.standard_normal((B, C)).astype(np.float32)
            layer.inputs(x, lens, rows)
            layer.ws.fill_bytes(0xFF)
            layer.o.fill_bytes(0xFF)
            dev.sync()
            assert hip.hipGraphLaunch(exe, s) == 0
            got = layer.o.read()
            o, tol, mine = layer.expect(x, lens, rows)
            near(got.reshape(B, H, D)[mine], o[mine], tol[mine], f"replay {rep}")
            same_cache(layer.cached.now(), layer.cache, f"replay {rep}")
            layer.launch()  # eager, the same inputs and state (a token written again is the same token)
            np.testing.assert_array_equal(layer.o.read(), got)
    finally:
        hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)
    layer.release()


def test_two_streams_with_a_workspace_each(dev):
    """Calls in flight at once on two streams, over one cache that both only read."""
    rng = np.random.default_rng(23)
    D, H, lens = 128, 2, [3000]
    cache, table = filled(rng, dev, lens, 1, D)
    cached = Cached(dev, cache)
    seqs = Sequences(dev, ok.Seqs(lens, table, 1, 1))
    other = c_void_p()
    _lib.check(_lib.load().sa_stream_create(byref(other)))
    calls = []
    for stream in (dev.stream, other.value):
        q = ok.to_type(rng.standard_normal((1, H * D)), "F16")
        rq, ro = Rows(dev, 1, H * D, "F16", data=q), Rows(dev, 1, H * D, "F16")
        a = _lib.KvAttnArgs(dtype=_lib.SA_DT["F16"], cache=cached.desc, seqs=seqs.desc, H=H, causal=1, scale=D ** -0.5, q=rq.buf.ptr, o=ro.buf.ptr)
        ws = dev.empty([_lib.kv_attention_workspace_bytes(a)], np.uint8)
        a.workspace, a.workspace_bytes = ws.ptr, ws.nbytes
        calls.append((stream, q, rq, ro, a, ws))
    dev.sync()
    for _ in range(20):
        for stream, _, _, _, a, _ in calls:
            _lib.kv_attention(a, stream)
    _lib.check(_lib.load().sa_device_sync())
    for _, q, rq, ro, a, ws in calls:
        o, size, reach, count, _ = cache.attention(seqs.oracle, q.astype(np.float64).reshape(1, H, D), D ** -0.5, True)
        near(ro.read((1, H, D)), o, ok.attention_tolerance(o, size, reach, count, D, "F16"))
        for x in (rq, ro, ws):
            x.release()
    _lib.check(_lib.load().sa_stream_destroy(other))
    cached.release()
    seqs.release()
