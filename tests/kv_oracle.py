"""Paged k/v caches on the host, from their definition and in 64 bits, and the
batches that the tests run: shared by the k/v tests."""
from __future__ import annotations

import numpy as np

from midge_amd import DevBuf
from midge_amd.kv import KV_F16, KV_MXFP4, KVBatch, KVCache, KVRows

LEVELS = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def encode(x):
    """f32 x[..., hd] -> (codes uint8 [..., hd / 2], exponent bytes [..., hd / 32])."""
    b = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    fine = np.isfinite(b).all(-1)
    a = np.where(fine[..., None], np.abs(b), 0).astype(np.float64)
    exps = np.arange(-13, 14)
    e = exps[np.minimum((a.max(-1, keepdims=True) > 7.0 * 2.0 ** exps).sum(-1), 26)]
    far = np.abs((a / 2.0 ** e[..., None])[..., None] - LEVELS)
    near = far == far.min(-1, keepdims=True)
    # the nearest code, of two the even one
    code = np.where(near.sum(-1) > 1, (near & (np.arange(8) % 2 == 0)).argmax(-1), near.argmax(-1)).astype(np.uint8)
    code = (code | (np.signbit(b).astype(np.uint8) << 3)).reshape(x.shape)
    return code[..., 0::2] | (code[..., 1::2] << 4), np.where(fine, e + 127, 255).astype(np.uint8)


def decode(codes, exps):
    lut = np.concatenate((LEVELS, -LEVELS))
    x = np.stack((lut[codes & 15], lut[codes >> 4]), -1).reshape(*codes.shape[:-1], -1)
    s = np.where(exps == 255, np.nan, 2.0 ** (exps.astype(np.float64) - 127))
    return (x.reshape(*x.shape[:-1], -1, 32) * s[..., None]).reshape(x.shape)


def f16(x):
    """wk_to_f16 (engine/mkern.h:261-273)."""
    with np.errstate(over="ignore"):
        h = x.astype(np.float32).astype(np.float16)
    return np.where(np.abs(x) < 2.0 ** -14, np.copysign(np.float32(0), x.astype(np.float32)).astype(np.float16), h)


class Pages:
    """A cache on the host (k, v [n_pages][nkv][page][...]) and on the device."""

    def __init__(self, dt, nkv, hd, page, n_pages, rng, junk=True):
        self.dt, self.nkv, self.hd, self.page, self.n_pages = dt, nkv, hd, page, n_pages
        shape = (n_pages, nkv, page)
        if dt == KV_F16:
            # what was there before: every kind of value
            self.arr = [(rng.integers(0, 65536, shape + (hd,)).astype(np.uint16) if junk else np.zeros(shape + (hd,), np.uint16)) for _ in "kv"]
        else:
            self.arr = [rng.integers(0, 256, shape + (hd // 2,)).astype(np.uint8) for _ in "kv"]
            self.arr += [(rng.integers(0, 256, shape + (hd // 32,)).astype(np.uint8) if junk else np.full(shape + (hd // 32,), 127, np.uint8))
                         for _ in "kv"]
        self.bufs = [DevBuf.from_array(a) for a in self.arr]
        self.cache = KVCache(dt, nkv, hd, page, n_pages, *self.bufs)

    def put(self, seq_pages, t, which, x):
        """Token t of a sequence gets f32 x[nkv][hd] as its k (0) or v (1), on the host."""
        at = (seq_pages[t // self.page], slice(None), t % self.page)
        if self.dt == KV_F16:
            self.arr[which][at] = f16(x).view(np.uint16)
        else:
            self.arr[which][at], self.arr[which + 2][at] = encode(x)

    def fill(self, seq_pages, n, rng, std=1.0):
        """n tokens of normal values (host)."""
        for t0 in range(0, n, self.page):
            m = min(self.page, n - t0)
            for w in (0, 1):
                x = (rng.standard_normal((self.nkv, m, self.hd)) * std).astype(np.float32)
                at = (seq_pages[t0 // self.page], slice(None), slice(0, m))
                if self.dt == KV_F16:
                    self.arr[w][at] = f16(x).view(np.uint16)
                else:
                    self.arr[w][at], self.arr[w + 2][at] = encode(x)

    def upload(self):
        for b, a in zip(self.bufs, self.arr):
            b.upload(a)

    def download(self):
        return [b.download(a.dtype, a.shape) for b, a in zip(self.bufs, self.arr)]

    def tokens(self, seq_pages, n, which, arr=None):
        """f64 [nkv][n][hd] of a sequence's first n tokens."""
        arr = arr or self.arr
        if n == 0:
            return np.zeros((self.nkv, 0, self.hd))
        at = np.asarray(seq_pages[:-(-n // self.page)] if n else [], np.int64)
        x = arr[which][at].view(np.float16).astype(np.float64) if self.dt == KV_F16 else decode(arr[which][at], arr[which + 2][at])
        return np.moveaxis(x, 0, 1).reshape(self.nkv, -1, self.hd)[:, :n]

    def free(self):
        for b in self.bufs:
            b.free()


class Batch:
    """seqs: [(len, rows)]; random disjoint pages, -1 behind a sequence's last."""

    def __init__(self, seqs, page, rng, extra_rows=0, n_pages=None, max_pages=None, one=False, extra_pages=3):
        self.seqs = seqs
        need = [-(-n // page) for n, _ in seqs]
        self.n_pages = n_pages or sum(need) + extra_pages
        self.max_pages = max_pages or max(max(need), 1)
        order = rng.permutation(self.n_pages)
        self.pages = np.full((len(seqs), self.max_pages), -1, np.int32)
        at = 0
        for i, m in enumerate(need):
            self.pages[i, :m] = order[at:at + m]
            at += m
        self.row0 = np.concatenate(([0], np.cumsum([r for _, r in seqs]))).astype(np.int32)
        self.len = np.array([n for n, _ in seqs], np.int32)
        self.n_rows = int(self.row0[-1]) + extra_rows
        self.max_rows = max(max(r for _, r in seqs), 1)
        self.bufs = [DevBuf.from_array(a) for a in (self.row0, self.len, self.pages)]
        self.batch = KVBatch(len(seqs), self.n_rows, self.max_rows, self.max_pages, 0 if one else self.bufs[0], *self.bufs[1:])

    def upload(self):
        for b, a in zip(self.bufs, (self.row0, self.len, self.pages)):
            b.upload(a)

    def host(self):
        """The batch with its arrays in host memory (for check())."""
        return KVBatch(len(self.seqs), self.n_rows, self.max_rows, self.max_pages, self.row0.ctypes.data, self.len.ctypes.data,
                       self.pages.ctypes.data)

    def rows(self):
        """(row, sequence, position) of every row of a sequence."""
        for s, (n, r) in enumerate(self.seqs):
            for i in range(r):
                yield int(self.row0[s]) + i, s, n - r + i

    def free(self):
        for b in self.bufs:
            b.free()


def prepared(x, bias, norm, eps, cos, sin):
    """One row's heads x[heads][hd] (f64): bias, norm, rotation by tables at its position."""
    x = x.astype(np.float64)
    if bias is not None:
        x = x + bias.astype(np.float64).reshape(x.shape)
    if norm is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + np.float64(np.float32(eps))) * norm.astype(np.float64)
    if cos is not None:
        h = x.shape[-1] // 2
        a, b, c, s = x[:, :h], x[:, h:], cos.astype(np.float64), sin.astype(np.float64)
        x = np.concatenate((a * c - b * s, b * c + a * s), -1)
    return x


def attention(q, k, v, scale, sink):
    """One row: q[nh][hd], its visible k, v [nkv][n][hd] (f64), sink[nh] or None -> (out[nh][hd], bound of the
    scores' magnitude sum)."""
    nh, hd = q.shape
    nkv = k.shape[0]
    g = nh // nkv
    if k.shape[1] == 0:
        return np.zeros((nh, hd)), 0.0
    qq = q.astype(np.float64).reshape(nkv, g, hd)
    s = scale * (qq @ k.transpose(0, 2, 1))
    mag = abs(scale) * (np.abs(qq) @ np.abs(k).transpose(0, 2, 1)).max()
    m = s.max(-1, keepdims=True)
    if sink is not None:
        sk = sink.astype(np.float64).reshape(nkv, g, 1)
        m = np.maximum(m, sk)
    e = np.exp(s - m)
    den = e.sum(-1, keepdims=True)
    if sink is not None:
        den = den + np.exp(sk - m)
    return (e @ v / den).reshape(nh, hd), float(mag)


__all__ = ["KV_F16", "KV_MXFP4", "KVBatch", "KVCache", "KVRows", "Pages", "Batch", "encode", "decode", "f16", "prepared", "attention"]
