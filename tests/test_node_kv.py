"""The 8-bit cache through the Node.js binding: the shim's mapping and refusals on the CPU, parity on the GPU."""

from __future__ import annotations

import json
import os
import shutil
import subprocess

import numpy as np
import pytest

from oracle import kv as ok

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")

pytestmark = pytest.mark.skipif(NODE is None, reason="node is not installed")


def test_shim_on_cpu():
    res = subprocess.run([NODE, os.path.join(ROOT, "tests", "node", "kv_cpu.js")], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    assert "all 6 checks passed" in res.stdout


@pytest.mark.gpu
def test_cache_through_node(tmp_path):
    rng = np.random.default_rng(31)
    d = str(tmp_path)
    save = lambda name, a: np.ascontiguousarray(a, np.float32).tofile(os.path.join(d, name))
    load = lambda name, *shape: np.fromfile(os.path.join(d, name), np.float32).astype(np.float64).reshape(shape)
    H, Hkv, D, lens, blocks = 6, 2, 64, [45, 70], [[3, 0], [1, 4, 2]]
    T, W = sum(lens), (H + 2 * Hkv) * D
    qkv = rng.standard_normal((T, W)).astype(np.float32)
    wq, wk = ((1 + 0.2 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    pos = np.concatenate([np.arange(n) for n in lens])
    save("qkv.bin", qkv)
    save("wq.bin", wq)
    save("wk.bin", wk)
    dit = [77, 1, 32]
    kv = [rng.standard_normal((n, 1152)).astype(np.float32) for n in dit]
    q = rng.standard_normal((3 * 256, 576)).astype(np.float32)
    save("q.bin", q)
    for b, x in enumerate(kv):
        save(f"kv{b}.bin", x)
    with open(os.path.join(d, "manifest.json"), "w") as f:
        json.dump(dict(prompts=dict(T=T, H=H, Hkv=Hkv, D=D, lens=lens, blocks=blocks, pages=5, positions=pos.tolist()), dit=dict(lens=dit)), f)
    res = subprocess.run([NODE, os.path.join(ROOT, "tests", "node", "kv_gpu.js"), d], capture_output=True, text=True, timeout=120)
    assert res.returncode == 0, res.stdout + res.stderr
    result = json.load(open(os.path.join(d, "result.json")))
    assert result["refused"] == ["SA_ERR_INVALID", "SA_ERR_INVALID", "SA_ERR_ALIAS", "SA_ERR_ALIAS"]
    assert {"qkNormRope", "kv.write", "kv.read", "kv.attention"} <= set(result["names"])

    rot = load("rotated.bin", T, W)
    freq = 10000.0 ** (-np.arange(0, D, 2) / D)
    for at, n, w in ((0, H, wq), (H * D, Hkv, wk)):
        want, size = ok.norm_rope(qkv[:, at:at + n * D].astype(np.float64).reshape(T, n, D), w, 1e-6, 1, pos, freq, D, False)
        assert (np.abs(rot[:, at:at + n * D].reshape(T, n, D) - want) <= ok.rope_tolerance(want, size, D, "F32")).all()
    np.testing.assert_array_equal(rot[:, (H + Hkv) * D:], qkv[:, (H + Hkv) * D:])
    table = np.full((2, 3), -1)
    table[0, :2], table[1] = blocks[0], blocks[1]
    starts = np.concatenate(([0], np.cumsum(lens)))
    seqs, cache = ok.Seqs(lens, table, T, max(lens), starts), ok.Cache(5, Hkv, D)
    cache.write(seqs, rot[:, H * D:(H + Hkv) * D].reshape(T, Hkv, D), rot[:, (H + Hkv) * D:].reshape(T, Hkv, D))
    k, v, _ = cache.read(seqs, T)
    np.testing.assert_array_equal(load("k.bin", T, Hkv, D), k)
    np.testing.assert_array_equal(load("v.bin", T, Hkv, D), v)
    o, size, reach, count, _ = cache.attention(seqs, rot[:, :H * D].reshape(T, H, D), D ** -0.5, True)
    assert (np.abs(load("o.bin", T, H, D) - o) <= ok.attention_tolerance(o, size, reach, count, D, "F32")).all()

    table = np.array([[0, 1, 2], [3, -1, -1], [4, -1, -1]])
    written, cache = ok.Seqs(dit, table, sum(dit), max(dit), np.concatenate(([0], np.cumsum(dit)))), ok.Cache(5, 9, 64)
    rows = np.concatenate(kv).astype(np.float64)
    cache.write(written, rows[:, :576].reshape(-1, 9, 64), rows[:, 576:].reshape(-1, 9, 64))
    some = np.concatenate([np.arange(b * 256, b * 256 + 256, 37) for b in range(3)])  # rows of each sample
    per = len(some) // 3
    o, size, reach, count, _ = cache.attention(ok.Seqs(dit, table, len(some), per), q[some].astype(np.float64).reshape(-1, 9, 64), 0.125, False)
    x = load("x.bin", 768, 9, 64)[some]
    assert (np.abs(x - o) <= ok.attention_tolerance(o, size, reach, count, 64, "F32")).all()
