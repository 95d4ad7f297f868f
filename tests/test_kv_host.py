"""The cached-attention boundary on the CPU: struct layouts, the cache's layout and bounds as host code (the header the
kernels share), calls that are refused before any launch, and calls with nothing to do."""

from __future__ import annotations

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest

from oracle import kv as ok
from supra_attn import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")
FAKE = 0x7F0000000000  # device-looking addresses: validation only compares them
F32, F16, BF16 = (_lib.SA_DT[t] for t in ("F32", "F16", "BF16"))

no_device = pytest.mark.skipif(_lib.device_count() > 0, reason="made-up device addresses: run on a host without a GPU")


@pytest.mark.parametrize("cls,ctype", [(_lib.QkRopeArgs, "sa_qk_rope_args"), (_lib.KvCache, "sa_kv_cache"), (_lib.KvSeqs, "sa_kv_seqs"),
                                       (_lib.KvRowsArgs, "sa_kv_rows_args"), (_lib.KvAttnArgs, "sa_kv_attn_args")])
def test_struct_layout_matches_c(tmp_path, cls, ctype):
    fields = [f[0] for f in cls._fields_]
    src = tmp_path / "layout.c"
    body = "\n".join(f'  printf("{f} %zu\\n", offsetof({ctype}, {f}));' for f in fields)
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "supra_kv.h"\nint main(void) {\n'
                   f'  printf("sizeof %zu\\n", sizeof({ctype}));\n{body}\n  return 0;\n}}\n')
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{INCLUDE}", str(src), "-o", str(exe)], check=True)
    lines = dict(ln.split() for ln in subprocess.run([str(exe)], capture_output=True, text=True).stdout.splitlines())
    assert int(lines["sizeof"]) == ctypes.sizeof(cls)
    for f in fields:
        assert int(lines[f]) == getattr(cls, f).offset, f


def test_constants():
    text = open(os.path.join(INCLUDE, "supra_kv.h")).read()
    for name in ("SA_NORM_NONE", "SA_NORM_RMS", "SA_ROPE_HALF", "SA_ROPE_NEAR", "SA_KV_BLOCK"):
        assert int(re.search(rf"#define {name} (\d+)", text).group(1)) == getattr(_lib, name)


def test_layout_and_bounds_of_the_kernels_header(tmp_path):
    """kv_layout.h as host code: V's slots, K's places, exponents of every kind of magnitude, powers of two, pages, and
    the bounds of sequences whose arrays say anything."""
    src = tmp_path / "layout.cpp"
    src.write_text('''
#include <stdio.h>
#include <string.h>
#include <stdlib.h>
#include "kv_layout.h"
int main(int argc, char** argv) {
  for (int t = 0; t < 32; ++t) printf("%d ", sa::kv_v_slot(t));
  printf("\\n");
  for (int t = 0; t < 32; ++t) for (int d = 0; d < 64; ++d) printf("%d ", sa::kv_k_place(t, d));
  printf("\\n");
  FILE* f = fopen(argv[1], "rb");
  unsigned u;
  while (fread(&u, 4, 1, f) == 1) printf("%d ", sa::kv_exponent(u));
  printf("\\n");
  for (int n = -140; n <= 127; ++n) { unsigned b = sa::kv_pow2_bits(n); float x; memcpy(&x, &b, 4); printf("%a ", x); }
  printf("\\n");
  const int ids[] = {-2147483647 - 1, -1, 0, 5, 6, 2147483647};
  for (int id : ids) printf("%d ", (int)sa::kv_page_ok(id, 6));
  printf("%lld\\n", (long long)sa::kv_tile(1 << 22, 8, 7, 256));
  int n;
  f = fopen(argv[2], "r");
  while (fscanf(f, "%d", &n) == 1) {
    int T, max_rows, max_blocks, uniform, start[2], len;
    if (fscanf(f, "%d %d %d %d %d %d", &T, &max_rows, &max_blocks, &uniform, &start[0], &start[1]) != 6) return 1;
    len = n;
    sa_kv_seqs s = {1, T, max_rows, max_blocks, uniform ? NULL : start, &len, NULL};
    sa::KvSeq q = sa::kv_seq(s, 0);
    printf("%d %d %d %d ", q.len, q.rows, q.row0, q.first);
  }
  printf("\\n");
  return 0;
}
''')
    rng = np.random.default_rng(1)
    mags = np.concatenate([np.array([0, 2.0 ** -149, 2.0 ** -126, 2.0 ** -119, 448, 449, 3.4e38, 1.75, 1.7500001, 1.7499999]),
                           rng.uniform(1, 2, 3000) * 2.0 ** rng.integers(-126, 127, 3000)]).astype(np.float32)
    (tmp_path / "m.bin").write_bytes(mags.tobytes())
    big = 2 ** 31 - 1
    cases = [(70, 90, 36, 3, 0, 10, 20), (-5, 90, 36, 3, 0, 0, 20), (1000, 90, 36, 3, 0, 80, 120), (10, 90, 36, 3, 0, 30, 29), (10, 90, 36, 3, 0, -1, 4),
             (10, 90, 36, 3, 0, 90, 95), (10, 90, 36, 3, 0, -big - 1, big), (10, 90, 36, 3, 0, big, -big), (5, 36, 36, 3, 1, 0, 0), (big, big, big, 1 << 25, 0, 0, big),
             (0, 90, 36, 0, 0, 0, 5), (96, 90, 36, 3, 0, 0, 50)]
    (tmp_path / "s.txt").write_text("\n".join(" ".join(map(str, c)) for c in cases))
    exe = tmp_path / "layout"
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover", f"-I{INCLUDE}",
                    f"-I{ROOT}/supra2-img-web_amd/csrc", str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe), str(tmp_path / "m.bin"), str(tmp_path / "s.txt")], capture_output=True, text=True, check=True).stdout.split("\n")
    slots = [int(x) for x in out[0].split()]
    assert slots == [ok.v_slot(t) for t in range(32)] and sorted(slots) == list(range(32))
    assert [int(x) for x in out[1].split()] == [(d // 32) * 1024 + t * 32 + d % 32 for t in range(32) for d in range(64)]
    np.testing.assert_array_equal([int(x) for x in out[2].split()], ok.exponent(mags.astype(np.float64)))
    assert [float.fromhex(x) for x in out[3].split()] == [0.0 if n < -126 else 2.0 ** n for n in range(-140, 128)]
    assert out[4].split() == ["0", "0", "1", "1", "0", "0", str(((1 << 22) * 8 + 7) * 32 * 256)]
    got = [int(x) for x in out[5].split()]
    for i, (n, T, max_rows, max_blocks, uniform, r0, r1) in enumerate(cases):
        cap, start, r = 32 * max_blocks, r0, r1 - r0
        n = min(max(n, 0), cap)
        if uniform:
            start, r = 0, max_rows
        if r < 0 or start < 0 or start >= T:
            r = 0
        first = max(n - r, -(1 << 30))
        rows = max(0, min(r, max_rows, T - start))
        length, grows, row0, gfirst = got[4 * i:4 * i + 4]
        assert (length, grows, gfirst) == (n, rows, first) and (rows == 0 or row0 == start), cases[i]
        assert 0 <= grows and (grows == 0 or 0 <= row0 and row0 + grows <= T)


def cache(**over):
    kw = dict(pages=10, Hkv=2, D=64, k=FAKE, v=FAKE + (1 << 32), k_scale=FAKE + (2 << 32), v_scale=FAKE + (3 << 32))
    kw.update(over)
    return _lib.KvCache(**kw)


def seqs(**over):
    kw = dict(B=3, T=12, max_rows=4, max_blocks=5, row_start=FAKE + (4 << 32), seq_len=FAKE + (5 << 32), block_table=FAKE + (6 << 32))
    kw.update(over)
    return _lib.KvSeqs(**kw)


def rows_args(c=None, s=None, **over):
    kw = dict(dtype=BF16, cache=c or cache(), seqs=s or seqs(), k=FAKE + (7 << 32), v=FAKE + (8 << 32))
    kw.update(over)
    return _lib.KvRowsArgs(**kw)


def attn_args(c=None, s=None, **over):
    kw = dict(dtype=BF16, cache=c or cache(), seqs=s or seqs(), H=4, causal=1, scale=0.125, q=FAKE + (7 << 32), o=FAKE + (8 << 32))
    kw.update(over)
    return _lib.KvAttnArgs(**kw)


def rope_args(**over):
    kw = dict(dtype=BF16, T=10, H=4, Hkv=2, D=64, rotary_dim=64, norm=1, eps=1e-6, q=FAKE, k=FAKE + (1 << 32), q_out=FAKE + (2 << 32),
              k_out=FAKE + (3 << 32), inv_freq=FAKE + (4 << 32), positions=FAKE + (5 << 32))
    kw.update(over)
    return _lib.QkRopeArgs(**kw)


INVALID, UNSUPPORTED, ALIAS = _lib.SA_ERR_INVALID, _lib.SA_ERR_UNSUPPORTED, _lib.SA_ERR_ALIAS

SHARED = [  # (status, cache fields, sequence fields): every call over a cache refuses them
    (INVALID, dict(pages=0), {}), (INVALID, dict(Hkv=0), {}), (INVALID, dict(pages=-1), {}), (INVALID, dict(reserved=1), {}),
    (UNSUPPORTED, dict(D=96), {}), (UNSUPPORTED, dict(D=512), {}), (INVALID, dict(D=0), {}), (UNSUPPORTED, dict(Hkv=4097), {}),
    (INVALID, dict(k=None), {}), (INVALID, dict(v=None), {}), (INVALID, dict(k_scale=None), {}), (INVALID, dict(v_scale=None), {}),
    (INVALID, dict(k=FAKE + 8), {}), (INVALID, dict(v=FAKE + 1), {}), (ALIAS, dict(v=FAKE + 16), {}), (ALIAS, dict(v_scale=FAKE + (2 << 32) + 3), {}),
    (ALIAS, dict(k_scale=FAKE + 100), {}),
    (INVALID, {}, dict(B=-1)), (INVALID, {}, dict(T=-1)), (INVALID, {}, dict(max_rows=-1)), (INVALID, {}, dict(max_blocks=-1)),
    (UNSUPPORTED, {}, dict(max_blocks=(1 << 25) + 1)), (UNSUPPORTED, {}, dict(B=(1 << 20) + 1)), (INVALID, {}, dict(seq_len=None)),
    (INVALID, {}, dict(block_table=None)), (INVALID, {}, dict(row_start=None, T=11)),
]


@no_device
@pytest.mark.parametrize("status,c,s", SHARED, ids=str)
def test_refusals_of_the_cache_and_sequences(status, c, s):
    lib = _lib.load()
    for fn, args in ((lib.sa_kv_write, rows_args(cache(**c), seqs(**s))), (lib.sa_kv_read, rows_args(cache(**c), seqs(**s))),
                     (lib.sa_kv_attention, attn_args(cache(**c), seqs(**s)))):
        assert fn(ctypes.byref(args), None) == status and lib.sa_last_status() == status and lib.sa_last_error()
    assert lib.sa_kv_attention_workspace_bytes(ctypes.byref(attn_args(cache(**c), seqs(**s)))) == status


@no_device
@pytest.mark.parametrize("status,over", [
    (UNSUPPORTED, dict(dtype=_lib.SA_DT["F64"])), (UNSUPPORTED, dict(dtype=_lib.SA_DT["F8_E4M3"])), (INVALID, dict(dtype=0)), (INVALID, dict(dtype=99)),
    (INVALID, dict(struct_size=8)), (INVALID, dict(k=None)), (INVALID, dict(v=None)), (INVALID, dict(k=FAKE + (7 << 32) + 1)), (INVALID, dict(k_off=-1)),
    (INVALID, dict(v_off=1 << 40)), (INVALID, dict(ldk=127)), (INVALID, dict(ldv=1 << 40)), (INVALID, dict(ldk=-1)), (ALIAS, dict(k=FAKE + 64)),
    (ALIAS, dict(v=FAKE + (3 << 32))),
])
def test_refusals_of_rows(status, over):
    lib = _lib.load()
    for fn in (lib.sa_kv_write, lib.sa_kv_read):
        assert fn(ctypes.byref(rows_args(**over)), None) == status


@no_device
def test_refusals_of_reads_alone():
    lib = _lib.load()
    read = lambda **over: lib.sa_kv_read(ctypes.byref(rows_args(**over)), None)
    assert read(v=FAKE + (7 << 32) + 64) == ALIAS  # k and v share rows
    assert read(k=FAKE + (5 << 32)) == ALIAS and read(v=FAKE + (6 << 32)) == ALIAS and read(v=FAKE + (4 << 32)) == ALIAS
    assert read(ldk=200, ldv=240, v=FAKE + (7 << 32), v_off=128) == ALIAS  # other strides over one range


@no_device
@pytest.mark.parametrize("status,over", [
    (INVALID, dict(H=0)), (INVALID, dict(H=3)), (INVALID, dict(H=-2)), (UNSUPPORTED, dict(H=1 << 17)), (INVALID, dict(causal=2)),
    (INVALID, dict(scale=float("nan"))), (INVALID, dict(scale=float("inf"))), (INVALID, dict(max_len=-1)), (INVALID, dict(q=None)), (INVALID, dict(o=None)),
    (INVALID, dict(ldq=255)), (INVALID, dict(ldo=255)), (INVALID, dict(q_off=-1)), (INVALID, dict(o_off=1 << 40)), (ALIAS, dict(o=FAKE + (7 << 32))),
    (ALIAS, dict(o=FAKE + (1 << 32))), (ALIAS, dict(o=FAKE + (5 << 32))), (INVALID, dict(struct_size=0)), (INVALID, dict(dtype=0)),
    (INVALID, dict(q=FAKE + (7 << 32) + 1)),
])
def test_refusals_of_attention(status, over):
    lib = _lib.load()
    args = attn_args(**over)
    assert lib.sa_kv_attention(ctypes.byref(args), None) == status
    assert lib.sa_kv_attention_workspace_bytes(ctypes.byref(args)) == status
    r, s = ctypes.c_int32(), ctypes.c_int32()
    assert lib.sa_kv_attention_shape(ctypes.byref(args), ctypes.byref(r), ctypes.byref(s)) == status


@no_device
@pytest.mark.parametrize("scale", [3e38, -3e38])
def test_scales_whose_log2_units_overflow_are_refused(scale):
    """The kernels hold scores in log2 units: scale * log2(e) has to be a float32 number too."""
    assert _lib.load().sa_kv_attention(ctypes.byref(attn_args(scale=scale)), None) == INVALID


@no_device
def test_refusals_of_the_workspace():
    """A call that splits its keys needs one: large enough, aligned, apart from everything else."""
    lib = _lib.load()
    long = seqs(B=1, T=1, max_rows=1, max_blocks=400)
    args = attn_args(s=long)
    need = _lib.kv_attention_workspace_bytes(args)
    assert need > 0 and _lib.kv_attention_shape(args)[1] > 1
    ws = FAKE + (9 << 32)
    for status, kw in ((INVALID, {}), (INVALID, dict(workspace=ws, workspace_bytes=need - 1)), (INVALID, dict(workspace=ws + 4, workspace_bytes=need)),
                       (ALIAS, dict(workspace=FAKE + (7 << 32), workspace_bytes=need)), (ALIAS, dict(workspace=FAKE + (8 << 32), workspace_bytes=need)),
                       (ALIAS, dict(workspace=FAKE, workspace_bytes=need)), (ALIAS, dict(workspace=FAKE + (6 << 32), workspace_bytes=need))):
        assert lib.sa_kv_attention(ctypes.byref(attn_args(s=long, **kw)), None) == status, kw
    for none in (dict(B=0), dict(T=0), dict(max_rows=0)):
        assert _lib.kv_attention_workspace_bytes(attn_args(s=seqs(**none))) == 0


@no_device
@pytest.mark.parametrize("status,over", [
    (INVALID, dict(struct_size=1)), (INVALID, dict(dtype=0)), (UNSUPPORTED, dict(dtype=_lib.SA_DT["I32"])), (INVALID, dict(T=-1)), (INVALID, dict(H=-1)),
    (INVALID, dict(Hkv=-1)), (INVALID, dict(D=63)), (INVALID, dict(D=0)), (UNSUPPORTED, dict(D=514)), (UNSUPPORTED, dict(H=1 << 17)),
    (INVALID, dict(rotary_dim=63)), (INVALID, dict(rotary_dim=66)), (INVALID, dict(rotary_dim=-2)), (INVALID, dict(pairs=2)), (INVALID, dict(norm=2)),
    (INVALID, dict(eps=-1.0)), (INVALID, dict(eps=float("nan"))), (INVALID, dict(rope_scale=float("inf"))), (INVALID, dict(inv_freq=None)),
    (INVALID, dict(positions=None)), (INVALID, dict(inv_freq=FAKE + 4)), (INVALID, dict(positions=FAKE + 2)), (INVALID, dict(q_weight=FAKE + 1)),
    (INVALID, dict(q=None)), (INVALID, dict(k_out=None)), (INVALID, dict(q=FAKE + 1)), (INVALID, dict(ldq=255)), (INVALID, dict(ldko=100)),
    (INVALID, dict(q_off=-1)), (INVALID, dict(ko_off=1 << 40)),
    (ALIAS, dict(q_out=FAKE + 2)), (ALIAS, dict(k_out=FAKE)), (ALIAS, dict(k_out=FAKE + (2 << 32))), (ALIAS, dict(q_out=FAKE, ldqo=300)),
    (ALIAS, dict(q_out=FAKE + (4 << 32))), (ALIAS, dict(k_out=FAKE + (5 << 32))), (ALIAS, dict(q_weight=FAKE + (2 << 32) + 4)),
])
def test_refusals_of_norm_rope(status, over):
    lib = _lib.load()
    assert lib.sa_qk_norm_rope(ctypes.byref(rope_args(**over)), None) == status and lib.sa_last_error()


@no_device
def test_calls_that_one_launch_cannot_hold():
    lib = _lib.load()
    huge = dict(B=1 << 20, T=1 << 30, max_rows=1 << 10, max_blocks=1 << 10)
    apart = dict(k=FAKE + (1 << 44), v=FAKE + (1 << 45))
    assert lib.sa_kv_write(ctypes.byref(rows_args(s=seqs(**huge), **apart)), None) == UNSUPPORTED
    assert lib.sa_kv_read(ctypes.byref(rows_args(s=seqs(**huge), **apart)), None) == UNSUPPORTED
    args = attn_args(s=seqs(**huge), q=FAKE + (1 << 44), o=FAKE + (1 << 45), H=64)
    assert lib.sa_kv_attention(ctypes.byref(args), None) == UNSUPPORTED
    far = {n: FAKE + ((i + 1) << 44) for i, n in enumerate(("q", "k", "q_out", "k_out"))}
    assert lib.sa_qk_norm_rope(ctypes.byref(rope_args(T=(1 << 31) - 1, **far)), None) == UNSUPPORTED


def test_calls_with_nothing_to_do():
    lib = _lib.load()
    for none in (dict(B=0), dict(T=0), dict(max_rows=0)):
        empty = seqs(seq_len=None, block_table=None, row_start=None, **none)
        for fn, args in ((lib.sa_kv_write, rows_args(s=empty)), (lib.sa_kv_read, rows_args(s=empty)), (lib.sa_kv_attention, attn_args(s=empty))):
            assert fn(ctypes.byref(args), None) == 0 and lib.sa_last_error() == b""
    for none in (dict(T=0), dict(H=0, Hkv=0)):
        assert lib.sa_qk_norm_rope(ctypes.byref(rope_args(q=None, k=None, q_out=None, k_out=None, **none)), None) == 0
    for fn in (lib.sa_kv_write, lib.sa_kv_read, lib.sa_kv_attention, lib.sa_qk_norm_rope):
        assert fn(None, None) == INVALID


def test_cache_bytes():
    assert _lib.kv_cache_bytes(7, 3, 128) == 7 * 3 * 32 * 128
    assert _lib.kv_cache_bytes(1 << 20, 4096, 256) == (1 << 20) * 4096 * 32 * 256
    lib = _lib.load()
    assert lib.sa_kv_cache_bytes(0, 1, 64) == INVALID and lib.sa_kv_cache_bytes(1, 1, 80) == UNSUPPORTED and lib.sa_kv_cache_bytes(1, 5000, 64) == UNSUPPORTED


def test_splits_follow_rows_and_keys():
    """Few rows over long caches are split, at eight pages at least to a share; many rows are not; and the workspace is
    a record of each group of 16 or 32 rows for each share."""
    for H, Hkv, D, B, n, keys in ((32, 8, 128, 1, 1, 777), (32, 8, 128, 64, 1, 8191), (4, 4, 64, 2, 3, 131072), (8, 1, 256, 1, 2048, 4096), (2, 1, 64, 1, 1, 32)):
        s = seqs(B=B, T=B * n, max_rows=n, max_blocks=-(-keys // 32))
        a = attn_args(cache(Hkv=Hkv, D=D, pages=1 << 10, v=FAKE + (1 << 36), k_scale=FAKE + (2 << 36), v_scale=FAKE + (3 << 36)), s, H=H,
                      q=FAKE + (4 << 36), o=FAKE + (5 << 36))
        rows, splits = _lib.kv_attention_shape(a)
        assert rows in (16, 32, 128)
        record = min(rows, 32)
        groups = -(-n * (H // Hkv) // record)
        assert splits == 1 or splits * 8 <= -(-keys // 32) + 7
        assert _lib.kv_attention_workspace_bytes(a) == (0 if splits == 1 else B * Hkv * groups * splits * record * (D + 1) * 4)


def test_oracle_codes_are_torch_codes():
    import torch

    rng = np.random.default_rng(0)
    x = np.clip(rng.standard_normal(200_000) * np.exp2(rng.integers(-14, 8, 200_000)), -448, 448).astype(np.float32)
    mids = ((ok.E4M3[:126] + ok.E4M3[1:127]) / 2).astype(np.float32)
    x = np.concatenate([x, ok.E4M3[:127].astype(np.float32), mids, -mids])
    np.testing.assert_array_equal(ok.encode(x.astype(np.float64)), torch.from_numpy(x).to(torch.float8_e4m3fn).view(torch.uint8).numpy())


def test_oracle_attention_is_softmax():
    """Against torch's own attention in float64 (grouped heads repeated), full and causal."""
    import torch

    rng = np.random.default_rng(3)
    c = ok.Cache(3, 2, 64, rng)
    c.codes &= 0xBF
    c.exp[:] = 126
    s = ok.Seqs([70], [[2, 0, 1]], 5, 5)
    q = rng.standard_normal((5, 4, 64))
    k, v, _ = c.read(ok.Seqs([70], [[2, 0, 1]], 70, 70), 70)
    rep = lambda x: torch.from_numpy(x).transpose(0, 1).repeat_interleave(2, 0)
    for causal in (False, True):
        mask = torch.ones(5, 70, dtype=torch.bool).tril(65) if causal else None
        want = torch.nn.functional.scaled_dot_product_attention(torch.from_numpy(q).transpose(0, 1), rep(k), rep(v), attn_mask=mask, scale=0.3)
        got = c.attention(s, q, 0.3, causal)[0]
        np.testing.assert_allclose(got, want.transpose(0, 1).numpy(), rtol=1e-12, atol=1e-13)


def test_oracle_rotation_is_complex_multiplication():
    rng = np.random.default_rng(4)
    x, pos = rng.standard_normal((6, 2, 16)), np.array([0, 1, 5, 1000, 123456, -3])
    f = 10000.0 ** (-np.arange(0, 8, 2) / 8)
    turn = np.exp(1j * pos[:, None] * f)[:, None]
    for near in (False, True):
        y, _ = ok.norm_rope(x, None, 0.0, 0, pos, f, 8, near)
        a, b = (slice(0, 8, 2), slice(1, 8, 2)) if near else (slice(0, 4), slice(4, 8))
        z = (x[..., a] + 1j * x[..., b]) * turn
        np.testing.assert_allclose(y[..., a], z.real, atol=1e-12)
        np.testing.assert_allclose(y[..., b], z.imag, atol=1e-12)
        np.testing.assert_array_equal(y[..., 8:], x[..., 8:])
