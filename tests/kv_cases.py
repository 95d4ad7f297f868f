"""Staging for the cached-attention tests: device copies of an oracle cache and of a call's sequences."""

from __future__ import annotations

import numpy as np

from oracle import kv as ok
from supra_attn import _lib

NP_OF = {"F32": np.float32, "F16": np.float16, "BF16": np.uint16}
GUARD = 0xAB


class Cached:
    """Device buffers of an oracle cache."""

    def __init__(self, dev, cache: ok.Cache):
        self.dev, self.oracle = dev, cache
        self.bufs = [dev.from_array(a) for a in cache.device_arrays()]
        self.desc = _lib.KvCache(pages=cache.pages, Hkv=cache.Hkv, D=cache.D, k=self.bufs[0].ptr, v=self.bufs[1].ptr,
                                 k_scale=self.bufs[2].ptr, v_scale=self.bufs[3].ptr)

    def now(self) -> ok.Cache:
        return self.oracle.from_device(*(b.read() for b in self.bufs))

    def release(self):
        for b in self.bufs:
            b.release()


class Sequences:
    """Device copies of an oracle's sequences, and the call's description of them."""

    def __init__(self, dev, seqs: ok.Seqs):
        self.oracle = seqs
        self.bufs = [dev.from_array(seqs.seq_len), dev.from_array(seqs.table)]
        start = None
        if seqs.row_start is not None:
            self.bufs.append(dev.from_array(seqs.row_start))
            start = self.bufs[2].ptr
        self.desc = _lib.KvSeqs(B=len(seqs.seq_len), T=seqs.T, max_rows=seqs.max_rows, max_blocks=seqs.table.shape[1], row_start=start,
                                seq_len=self.bufs[0].ptr, block_table=self.bufs[1].ptr)

    def release(self):
        for b in self.bufs:
            b.release()


class Rows:
    """[T, width] rows of a type inside a guarded buffer: `off` elements before them, a row stride of `ld`."""

    def __init__(self, dev, T, width, dtype, off=0, ld=0, data=None):
        self.T, self.width, self.dtype, self.off, self.ld = T, width, dtype, off, ld or width
        n = off + max(T, 1) * self.ld + 16
        host = np.full(n * np.dtype(NP_OF[dtype]).itemsize, GUARD, np.uint8).view(NP_OF[dtype])
        if data is not None:
            self.view(host)[:] = np.asarray(data).reshape(T, width)
        self.host = host
        self.buf = dev.from_array(host)

    def view(self, host):
        return np.lib.stride_tricks.as_strided(host[self.off:], (self.T, self.width), (self.ld * host.itemsize, host.itemsize))

    def read(self, shape):
        """The rows' float64 values; fails if anything outside them changed."""
        got = self.buf.read()
        rows = self.view(got).copy()
        self.view(got)[:] = self.view(self.host)
        np.testing.assert_array_equal(got.view(np.uint8), self.host.view(np.uint8), err_msg="wrote outside the rows")
        self.raw = rows
        return ok.values(rows, self.dtype).reshape(shape)

    def untouched(self, rows):
        """Whether those rows of the last read still hold the guard bytes."""
        return (np.ascontiguousarray(self.raw[rows]).view(np.uint8) == GUARD).all()

    def release(self):
        self.buf.release()


def scattered_table(rng, lens, pages, extra=1):
    """A block table with every sequence's pages at random places and -1 behind them."""
    blocks = [-(-max(n, 0) // ok.BLOCK) for n in lens]
    ids = rng.permutation(pages)[:sum(blocks)]
    t = np.full((len(lens), max(blocks + [0]) + extra), -1, np.int32)
    at = 0
    for b, n in enumerate(blocks):
        t[b, :n] = ids[at:at + n]
        at += n
    return t


def starts(rows):
    return np.concatenate(([0], np.cumsum(rows))).astype(np.int32)


def attend(dev, cached, seqs, q, H, dtype, scale, causal, max_len=0, off=0, ld=0, o_off=0, ldo=0):
    """One sa_kv_attention call: (the rows' values [T, H, D], its Rows, splits)."""
    D, T = cached.oracle.D, seqs.oracle.T
    rq = Rows(dev, T, H * D, dtype, off, ld, q)
    ro = Rows(dev, T, H * D, dtype, o_off, ldo)
    a = _lib.KvAttnArgs(dtype=_lib.SA_DT[dtype], cache=cached.desc, seqs=seqs.desc, H=H, causal=int(causal), scale=scale, max_len=max_len,
                        q=rq.buf.ptr, o=ro.buf.ptr, q_off=off, o_off=o_off, ldq=ld, ldo=ldo)
    need, ws = _lib.kv_attention_workspace_bytes(a), None
    if need:
        ws = dev.empty([need], np.uint8).fill_bytes(0xFF)  # NaN patterns: what a call has not written it must not use
        a.workspace, a.workspace_bytes = ws.ptr, need
    _lib.kv_attention(a, dev.stream)
    got = ro.read((T, H, D))
    if ws:
        ws.release()
    rq.release()
    return got, ro, _lib.kv_attention_shape(a)[1]
